// attention_op_delta.cu -- the row sums that the attention operator's backward pass
// subtracts,
//   delta_i = sum_j P_ij dP_ij = sum_d dO_id O_id.
//
// The right side reads both arrays once and is bound by memory, but takes O as the
// forward left it, rounded to 16 bits: delta is off by up to half a step of sum
// |dO O|, which dQ and dK of rows with few keys show. Against a 32-bit pass rounded
// once the gradients' error is 1.7 times at 2 keys, 1.5 at 9, 1.45 at 16, 1.43 from
// 32 on; with the left side, in f32, 1.4 throughout. So a row gets the left side if
// its sequence has SHORT tokens at most, its window is NARROW at most or it sees FEW
// keys at most, whatever else the call holds; otherwise it gets the right side, if
// its call does not have the left one at hand.
//
// Inside the dQ pass, whose warps are few, delta took a third of an item's time at
// 175-180 tokens (64 of them, 12 heads: dQ 80 -> 47 us without it, delta 8.6).
#include "attention_op.cuh"

namespace laya {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int ROWS = 4;                    // of eight lanes, all loads under way at once
constexpr int PAIRS = ROWS * THREADS / 8;  // (token, head) pairs of a block, heads fastest
constexpr int TILE = 16;                   // rows of an mma.sync tile
constexpr int KEYS = 32;                   // that such a tile looks at
static_assert(SHORT <= KEYS && TILE + 2 * NARROW <= KEYS, "a tile sees all of its rows' keys");

// The sum over eight lanes, in each of them.
__device__ __forceinline__ float sum8(float x) {
#pragma unroll
    for (int k = 1; k < 8; k *= 2) x += __shfl_xor_sync(0xffffffffu, x, k);
    return x;
}

// A quarter of a row of a head, 16 elements: what a lane feeds to the products.
// Which of the 64 a product's 16 are does not matter, as long as both operands
// agree; so a lane takes them in two loads instead of sixteen.
struct Quarter {
    uint32_t x[8];
    template <typename T>
    __device__ __forceinline__ void load(const AttnRows& r, long long row, int head, int quarter, bool ok) {
        uint4 u = make_uint4(0, 0, 0, 0), w = u;
        if (ok) {
            u = piece<T>(r, row, head, quarter * 16);
            w = piece<T>(r, row, head, quarter * 16 + 8);
        }
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
        x[4] = w.x, x[5] = w.y, x[6] = w.z, x[7] = w.w;
    }
};

// c (16 x 8) = rows of two quarters each . the eight rows of b, over the head
template <typename T>
__device__ __forceinline__ void product(float (&c)[4], const Quarter& r0, const Quarter& r1, const Quarter& b) {
    c[0] = c[1] = c[2] = c[3] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const uint32_t a[4] = {r0.x[k], r1.x[k], r0.x[k + 1], r1.x[k + 1]};
        mma<T>(c, a, b.x[k], b.x[k + 1]);
    }
}

// Does row i see more than FEW keys? A thread's look at those around it, which
// nearly always has the answer; false: perhaps not.
__device__ __forceinline__ bool sees_more(const AttnArgs& a, const SeqTile& t, int i) {
    int lo, hi, count = 0;
    span(a, t, i, &lo, &hi);
    const int near = max(lo, min(i - 8, hi - 15));
#pragma unroll
    for (int x = 0; x < 16; x++)
        if (near + x <= hi) count += present(a, t, near + x);
    return count > FEW;
}

// delta from P dP of rows row0 .. row0 + 15 of a sequence and one head, whose keys
// are all among the KEYS from key0 on (which may lie before the sequence): a warp,
// with 8 * AHEAD keys on their way at once.
template <typename T, int AHEAD>
__device__ __forceinline__ void tile_from_keys(const AttnArgs& a, const SeqTile& t, int head, int row0, int key0,
                                               float* delta, int lane) {
    const int g = lane >> 2, c = lane & 3, hk = head / a.group;
    const int i0 = row0 + g, i1 = i0 + 8;
    const bool p0 = present(a, t, i0), p1 = present(a, t, i1);
    const long long at = (long long)head * a.n_tokens + t.start;
    Quarter q0, q1, d0, d1;
    q0.load<T>(a.io.q, t.start + i0, head, c, p0);
    q1.load<T>(a.io.q, t.start + i1, head, c, p1);
    d0.load<T>(a.io.dout, t.start + i0, head, c, p0);
    d1.load<T>(a.io.dout, t.start + i1, head, c, p1);
    const float sl2 = a.scale * LOG2E;
    const float e0 = p0 ? a.io.lse[at + i0] * LOG2E : 0.f, e1 = p1 ? a.io.lse[at + i1] * LOG2E : 0.f;
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int n0 = 0; n0 < KEYS; n0 += 8 * AHEAD) {
        Quarter k[AHEAD], v[AHEAD];
        uint32_t keys[AHEAD];  // four lanes to a key
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int key = key0 + n0 + 8 * u + g;
            const bool ok = present(a, t, key);
            keys[u] = __ballot_sync(0xffffffffu, ok);
            k[u].template load<T>(a.io.k, t.start + key, hk, c, ok);
            v[u].template load<T>(a.io.v, t.start + key, hk, c, ok);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            float s[4], dp[4];
            product<T>(s, q0, q1, k[u]);
            product<T>(dp, d0, d1, v[u]);
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int x = 2 * c + e, j = key0 + n0 + 8 * u + x;
                const bool there = keys[u] >> (4 * x) & 1;
                if (there && (a.window < 0 || abs(i0 - j) <= a.window))
                    sum0 = fmaf(ex2_approx(fmaf(s[e], sl2, -e0)), dp[e], sum0);
                if (there && (a.window < 0 || abs(i1 - j) <= a.window))
                    sum1 = fmaf(ex2_approx(fmaf(s[2 + e], sl2, -e1)), dp[2 + e], sum1);
            }
        }
    }
#pragma unroll
    for (int x = 1; x < 4; x *= 2) {
        sum0 += __shfl_xor_sync(0xffffffffu, sum0, x);
        sum1 += __shfl_xor_sync(0xffffffffu, sum1, x);
    }
    if (c == 0 && p0) delta[at + i0] = sum0;
    if (c == 0 && p1) delta[at + i1] = sum1;
}

// delta of row i of a sequence, all heads, from its keys among lo .. hi, wherever
// they are: the whole warp, eight lanes to a head, two keys' loads under way at once.
template <typename T>
__device__ __forceinline__ void from_keys(const AttnArgs& a, const SeqTile& t, int i, int heads, int lo, int hi,
                                          int lane) {
    const int c = (lane & 7) * 8;
    const float sl2 = a.scale * LOG2E;
    const long long row = t.start + i;
    for (int g = 0; g < heads; g += 4) {
        const int h = min(g + (lane >> 3), heads - 1), hk = h / a.group;  // a head too many: the last one again
        const uint4 q = piece<T>(a.io.q, row, h, c), d = piece<T>(a.io.dout, row, h, c);
        const float e = a.io.lse[(long long)h * a.n_tokens + row] * LOG2E;
        float sum = 0.f;
        for (int j = lo; j <= hi; j += 32) {
            uint32_t keys = __ballot_sync(0xffffffffu, j + lane <= hi && present(a, t, j + lane));
            while (keys) {
                uint4 k[2], v[2];
                const int n = min(__popc(keys), 2);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u >= n) break;
                    const long long at = t.start + j + __ffs(keys) - 1;
                    keys &= keys - 1;
                    k[u] = piece<T>(a.io.k, at, hk, c);
                    v[u] = piece<T>(a.io.v, at, hk, c);
                }
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u >= n) break;
                    const float s = sum8(dot8<T>(q, k[u])), dp = sum8(dot8<T>(d, v[u]));
                    sum = fmaf(ex2_approx(fmaf(s, sl2, -e)), dp, sum);
                }
            }
        }
        if (c == 0 && g + (lane >> 3) < heads) a.io.delta[(long long)h * a.n_tokens + row] = sum;
    }
}

// All of a short sequence, by the warps of a block.
template <typename T>
__device__ __forceinline__ void short_sequence(const AttnArgs& a, const SeqTile& t, int heads, int warp, int lane) {
    const int tiles = (t.len + TILE - 1) / TILE;
    for (int u = warp; u < heads * tiles; u += WARPS)
        tile_from_keys<T, 1>(a, t, u / tiles, u % tiles * TILE, 0, a.io.delta_short, lane);
}

__device__ __forceinline__ void open(const AttnArgs& a) {
    griddep_launch();
    if (blockIdx.x == 0 && threadIdx.x < 2) a.io.tickets[threadIdx.x] = 0;  // for the passes that follow
}

// The first blocks take the short sequences, a block to a sequence, into
// a.io.delta_short; the others 128 (token, head) pairs each, eight lanes to a row,
// without a look at the table: what they leave for rows of short sequences is not
// used.
template <typename T>
__global__ void __launch_bounds__(THREADS, 4)
    attention_delta_kernel(const __grid_constant__ AttnArgs a, int heads, int seq_blocks) {
    open(a);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = (threadIdx.x & 7) * 8;
    if ((int)blockIdx.x < seq_blocks) {
        for (long long s = blockIdx.x; s < a.n_seqs; s += seq_blocks) {
            const int start = a.cu[s], end = a.cu[s + 1];
            if (!run_ok(start, end, a.n_tokens, a.max_len)) continue;
            const SeqTile t{start, end - start, 0};
            if (t.len <= SHORT) short_sequence<T>(a, t, heads, warp, lane);
        }
        return;
    }
    // tokens times heads: below 2^32 with the last block's surplus
    const unsigned first = (blockIdx.x - seq_blocks) * PAIRS;
    const int begin = max(a.cu[0], 0), end = min(a.cu[a.n_seqs], a.n_tokens);  // rows past either are not the call's
    uint4 o[ROWS], d[ROWS];
    long long to[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const unsigned at = first + i * (THREADS / 8) + threadIdx.x / 8;
        const int t = (int)(at / (unsigned)heads), h = (int)(at - (unsigned)t * heads);
        to[i] = -1;
        o[i] = d[i] = make_uint4(0, 0, 0, 0);
        if (t >= begin && t < end) {
            to[i] = (long long)h * a.n_tokens + t;
            o[i] = piece<T>(a.io.out, t, h, c);
            d[i] = piece<T>(a.io.dout, t, h, c);
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float sum = sum8(dot8<T>(o[i], d[i]));
        if (to[i] >= 0 && c == 0) a.io.delta[to[i]] = sum;
    }
}

// The same where tokens may be absent: a block to a tile of a sequence's rows, of
// which it first finds out, a thread to a row, which may see few keys. (128 x 1-512
// tokens, a fifth of them absent, 12 heads over 4: the backward pass 294 us, 287 with
// the kernel above, which does not ask; with 32 rows to a block 296, with 16 305.)
constexpr int MASKED_ROWS = 64;
enum : uint8_t { ABSENT, FROM_OUT, PERHAPS };

template <typename T>
__global__ void __launch_bounds__(THREADS, 4)
    attention_masked_delta_kernel(const __grid_constant__ AttnArgs a, int heads) {
    __shared__ uint8_t source[MASKED_ROWS];
    open(a);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = (threadIdx.x & 7) * 8;
    SeqTile t;
    if (!find_tile(a.cu, a.n_seqs, a.n_tokens, a.max_len, MASKED_ROWS, blockIdx.x, lane, &t)) return;
    if (t.len <= SHORT) return short_sequence<T>(a, t, heads, warp, lane);
    const int rows = min(MASKED_ROWS, t.len - t.row0);
    bool more = false;
    if (threadIdx.x < rows) {
        const int i = t.row0 + threadIdx.x;
        uint8_t from = ABSENT;
        if (present(a, t, i)) {
            more = !sees_more(a, t, i);
            from = more ? PERHAPS : FROM_OUT;
        }
        source[threadIdx.x] = from;
    }
    more = __syncthreads_or(more);
    for (int p = threadIdx.x / 8; p - (int)threadIdx.x / 8 < rows * heads; p += PAIRS) {
        uint4 o[ROWS], d[ROWS];
        long long to[ROWS];
#pragma unroll
        for (int x = 0; x < ROWS; x++) {
            const int at = p + x * (THREADS / 8), i = at / heads, h = at - i * heads;
            to[x] = -1;
            o[x] = d[x] = make_uint4(0, 0, 0, 0);
            if (i < rows && source[i] != ABSENT) {
                const int row = t.start + t.row0 + i;
                to[x] = (long long)h * a.n_tokens + row;
                o[x] = piece<T>(a.io.out, row, h, c);
                d[x] = piece<T>(a.io.dout, row, h, c);
            }
        }
#pragma unroll
        for (int x = 0; x < ROWS; x++) {
            const float sum = sum8(dot8<T>(o[x], d[x]));
            if (to[x] >= 0 && c == 0) a.io.delta[to[x]] = sum;
        }
    }
    if (!more) return;
    __syncthreads();  // what follows overwrites some of it
    for (int r = warp; r < rows; r += WARPS) {
        if (source[r] != PERHAPS) continue;
        int lo, hi, count = 0;
        span(a, t, t.row0 + r, &lo, &hi);
        for (int j = lo + lane; j - lane <= hi && count <= FEW; j += 32)
            count += __popc(__ballot_sync(0xffffffffu, j <= hi && present(a, t, j)));
        if (count <= FEW) from_keys<T>(a, t, t.row0 + r, heads, lo, hi, lane);
    }
}

// Narrow windows: every row from its keys, a block to a tile of 16 rows, whose warps
// take a head each. (A warp to a token, a dot product at a time: the backward pass of
// 64 x 180 tokens, 12 heads, window 4, 108 us instead of 91.)
constexpr int NARROW_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(NARROW_THREADS) attention_narrow_delta_kernel(const __grid_constant__ AttnArgs a, int heads) {
    open(a);
    const int lane = threadIdx.x & 31;
    SeqTile t;
    if (!find_tile(a.cu, a.n_seqs, a.n_tokens, a.max_len, TILE, blockIdx.x, lane, &t)) return;
    for (int h = threadIdx.x >> 5; h < heads; h += NARROW_THREADS / 32)
        tile_from_keys<T, 2>(a, t, h, t.row0, t.row0 - a.window, a.io.delta, lane);
}

template <typename T>
void launch(int heads, const AttnArgs& a, cudaStream_t stream) {
    if (narrow(a.window)) {
        const unsigned tiles = (unsigned)seq_tiles(a.n_tokens, a.n_seqs, TILE);
        attention_narrow_delta_kernel<T><<<tiles, NARROW_THREADS, 0, stream>>>(a, heads);
    } else if (a.mask) {
        const unsigned tiles = (unsigned)seq_tiles(a.n_tokens, a.n_seqs, MASKED_ROWS);
        attention_masked_delta_kernel<T><<<tiles, THREADS, 0, stream>>>(a, heads);
    } else {
        const int seq_blocks = a.n_seqs < 2 * 148 ? a.n_seqs : 2 * 148;
        const unsigned blocks = (unsigned)(((unsigned long long)a.n_tokens * heads + PAIRS - 1) / PAIRS);
        attention_delta_kernel<T><<<seq_blocks + blocks, THREADS, 0, stream>>>(a, heads, seq_blocks);
    }
}

}  // namespace

cudaError_t launch_attention_delta(bool bf16, int n_heads, const AttnArgs& a, cudaStream_t stream) {
    if (bf16) launch<__nv_bfloat16>(n_heads, a, stream);
    else launch<__half>(n_heads, a, stream);
    return cudaGetLastError();
}

}  // namespace laya
