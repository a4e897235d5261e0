// attention_op.cu -- packed attention as an operator: the forward with its
// statistics and the backward pass, on mma.sync tiles of 64 x 64.
//
// Forward, per query row: the online softmax (running maximum and sum, one
// pass over the keys), out = O / l and lse = m + log l.
//
// Backward, with the probabilities recomputed as P = exp(S - lse):
//   delta_i = sum_d dO_id O_id            (= sum_j P_ij dP_ij, which rows with few
//                                          keys take: attention_op_delta.cu)
//   dP = dO V^T,  dS = P (dP - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// One launch, without atomics: a block per query tile walks the keys for dQ, a
// block per key tile walks the queries of every head of its group for dK and
// dV. S, dP and delta are computed in both, seven products instead of five,
// which is what a fixed order of the sums costs here.
// P and dS are rounded to 16 bits as operands of the products that follow;
// statistics, sums and accumulators are f32.
//
// These kernels serve calls that a few waves of blocks finish, where what
// counts is the chain of dependent steps in one block (find the sequence, load,
// two to five products of 16 x 8 x 16 instructions, exponentials, store), not
// a rate. One sequence of 64 tokens, 12 heads, bf16: forward 3.7 us, backward
// 4.3 us (a short kernel on its own takes 1.8 there). Backward in one launch
// instead of a dQ launch followed by a dK/dV launch that reads its delta: half the
// time there; delta is recomputed from O, which a row's tile costs little.
//
// Sequences of 64 tokens at most have kernels of their own below (the backward
// pass of a few of more than 32 tokens does without, see one_block_each), because a
// 128-row tcgen05 item or a search for each of them costs more than its work: forward
// and backward of 512 sequences of 16 / 32 / 64 tokens, 12 heads, 265 / 230 / 235 us
// on tcgen05, 72 / 102 / 153 here (139 / 277 / 553 MB: 3.6 TB/s for the last).
//
// Rows outside their sequence and absent tokens are filled with zeros on
// their way into shared memory (cp.async with a source size of 0), so nothing
// they hold enters a product: zero rows of Q and dO add nothing to dK and dV,
// zero rows of K nothing to dQ, and the scores of such keys are masked where
// the softmax sums them.
#include <type_traits>

#include "attention_op.cuh"

namespace laya {
namespace {

constexpr int TB = 64;  // rows per tile
constexpr int THREADS = 128;
constexpr int TILE = TB * 64;  // elements
constexpr int SMALL_LEN = 512;  // tokens of the longest sequence of a small call

// element offset of (row, col) in a 64 x 64 16-bit tile whose 16-byte chunks
// are XORed by row: ldmatrix row fetches never share a bank
__device__ __forceinline__ int swz(int r, int c) { return r * 64 + (((c >> 3) ^ (r & 7)) << 3) + (c & 7); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p)));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_u32(p)));
}

// Rows row0 .. row0 + 63 of the sequence (the first n times 16 of them), 64
// elements each, into a tile.
template <typename T>
__device__ __forceinline__ void load_tile(T* s, const AttnRows& rows, int head, const AttnArgs& a, const SeqTile& t,
                                          int row0, int n = TB / 16) {
    const T* g = static_cast<const T*>(rows.p) + head * 64;
    static_assert(THREADS / 8 == 16, "a round of the loop takes 16 rows");
#pragma unroll
    for (int i = 0; i < TILE / 8 / THREADS; i++) {
        if (i >= n) break;
        const int idx = threadIdx.x + i * THREADS, r = idx >> 3, c = (idx & 7) * 8;
        const bool ok = present(a, t, row0 + r);
        const long long row = t.start + (ok ? row0 + r : 0);
        copy16(s + swz(r, c), g + row * rows.ld + c, ok);
    }
}

// Bits of the tile's 64 keys that are there.
__device__ __forceinline__ void key_bits(uint32_t* bits, const AttnArgs& a, const SeqTile& t, int row0) {
    const int w = threadIdx.x >> 5;
    if (w < 2) {
        const uint32_t b = __ballot_sync(0xffffffffu, present(a, t, row0 + (int)threadIdx.x));
        if ((threadIdx.x & 31) == 0) bits[w] = b;
    }
}

// A fragments (16 rows x 64) of a warp's rows of a tile.
template <typename T>
__device__ __forceinline__ void load_a(uint32_t (&f)[4][4], const T* s, int warp, int lane) {
#pragma unroll
    for (int ks = 0; ks < 4; ks++) ldsm4(f[ks], s + swz(warp * 16 + (lane & 15), ks * 16 + (lane >> 4) * 8));
}

template <int N>
__device__ __forceinline__ void clear(float (&c)[N][4]) {
#pragma unroll
    for (int j = 0; j < N; j++) c[j][0] = c[j][1] = c[j][2] = c[j][3] = 0.f;
}

// c[16 x 64 tile rows] = a (16 x 64) . tile^T, of the tile's first n times 16
// rows (0 for the others)
template <typename T>
__device__ __forceinline__ void mma_nt(float (&c)[8][4], const uint32_t (&a)[4][4], const T* tile, int lane,
                                       int n = 4) {
    clear(c);
#pragma unroll
    for (int ks = 0; ks < 4; ks++)
#pragma unroll
        for (int np = 0; np < 4; np++) {
            if (np >= n) break;
            uint32_t b[4];
            ldsm4(b, tile + swz(np * 16 + (lane & 7) + (lane >> 4) * 8, ks * 16 + ((lane >> 3) & 1) * 8));
            mma<T>(c[2 * np], a[ks], b[0], b[1]);
            mma<T>(c[2 * np + 1], a[ks], b[2], b[3]);
        }
}

// c[16 x 64] += a (16 x 16) . rows 16 kk .. 16 kk + 15 of the tile
template <typename T>
__device__ __forceinline__ void mma_step(float (&c)[8][4], const uint32_t (&a)[4], const T* tile, int kk, int lane) {
#pragma unroll
    for (int dp = 0; dp < 4; dp++) {
        uint32_t b[4];
        ldsm4_t(b, tile + swz(kk * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, dp * 16 + (lane >> 4) * 8));
        mma<T>(c[2 * dp], a, b[0], b[1]);
        mma<T>(c[2 * dp + 1], a, b[2], b[3]);
    }
}

// c[16 x 64] += p (16 x the tile's first n times 16 rows, as accumulators) . tile
template <typename T>
__device__ __forceinline__ void mma_nn(float (&c)[8][4], const float (&p)[8][4], const T* tile, int lane, int n = 4) {
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
        if (kk >= n) break;
        uint32_t a[4];
        a[0] = pack2<T>(p[2 * kk][0], p[2 * kk][1]);
        a[1] = pack2<T>(p[2 * kk][2], p[2 * kk][3]);
        a[2] = pack2<T>(p[2 * kk + 1][0], p[2 * kk + 1][1]);
        a[3] = pack2<T>(p[2 * kk + 1][2], p[2 * kk + 1][3]);
        mma_step<T>(c, a, tile, kk, lane);
    }
}

// c[16 x 64] += the transpose of x's columns 16 warp .. 16 warp + 15, over the
// first n times 16 rows of x and of the tile
template <typename T>
__device__ __forceinline__ void mma_tn(float (&c)[8][4], const T* x, const T* tile, int warp, int lane, int n) {
#pragma unroll
    for (int kk = 0; kk < 4; kk++) {
        if (kk >= n) break;
        uint32_t a[4];
        ldsm4_t(a, x + swz(kk * 16 + (lane & 7) + (lane >> 4) * 8, warp * 16 + ((lane >> 3) & 1) * 8));
        mma_step<T>(c, a, tile, kk, lane);
    }
}

// A warp's 16 x 64 accumulators, times two row factors, into its rows of a
// tile as 16-bit values; 0 for the factor 0, whatever the accumulator holds.
template <typename T>
__device__ __forceinline__ void put_rows(T* s, const float (&c)[8][4], int warp, int lane, float f0 = 1.f,
                                         float f1 = 1.f) {
    const int r = warp * 16 + (lane >> 2), k = 2 * (lane & 3);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        *reinterpret_cast<uint32_t*>(s + swz(r, 8 * j + k)) = f0 == 0.f ? 0u : pack2<T>(c[j][0] * f0, c[j][1] * f0);
        *reinterpret_cast<uint32_t*>(s + swz(r + 8, 8 * j + k)) = f1 == 0.f ? 0u : pack2<T>(c[j][2] * f1, c[j][3] * f1);
    }
}

// The same to the sequence's rows r0 + 16 warp .. in global memory, those past
// its end left alone; by way of the warp's rows of tile s, which nobody needs
// any more: whole rows of 128 bytes an instruction instead of 16 bytes each.
template <typename T>
__device__ __forceinline__ void store_rows(T* s, const AttnRows& rows, int head, const SeqTile& t, int r0, int warp,
                                           int lane, const float (&c)[8][4], float f0, float f1) {
    __syncwarp();
    put_rows<T>(s, c, warp, lane, f0, f1);
    __syncwarp();
    T* g = static_cast<T*>(rows.p) + head * 64 + (lane & 7) * 8;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = warp * 16 + i * 4 + (lane >> 3);
        const uint4 u = *reinterpret_cast<const uint4*>(s + swz(r, (lane & 7) * 8));
        if (r0 + r < t.len) *reinterpret_cast<uint4*>(g + (t.start + r0 + r) * rows.ld) = u;
    }
}

__device__ __forceinline__ bool block_tile(const AttnArgs& a, SeqTile* t) {
    if (threadIdx.x == 0 && blockIdx.y == 0)  // the grid has a block for every entry
        check_table(a.cu, a.n_seqs, a.n_tokens, a.max_len, blockIdx.x, a.status);
    return find_tile(a.cu, a.n_seqs, a.n_tokens, a.max_len, TB, blockIdx.x, threadIdx.x & 31, t);
}

// ------------------------------------------------------------------ forward
constexpr int FWD_SMEM = 5 * TILE * 2;

template <typename T>
__global__ void __launch_bounds__(THREADS, 3) attention_fwd_kernel(const AttnArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    T* sq = reinterpret_cast<T*>(smem);
    T* sk = sq + TILE;
    T* sv = sk + 2 * TILE;
    __shared__ uint32_t bits[2][2];
    SeqTile t;
    griddep_begin();
    if (!block_tile(a, &t)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y, hk = h / a.group;
    int kt0, kt1;
    visible_tiles(a, t, TB, TB, &kt0, &kt1);
    load_tile(sq, a.io.q, h, a, t, t.row0);
    load_tile(sk, a.io.k, hk, a, t, kt0 * TB);
    load_tile(sv, a.io.v, hk, a, t, kt0 * TB);
    key_bits(bits[0], a, t, kt0 * TB);
    copy_commit();

    const float sl2 = a.scale * LOG2E;
    const int i0 = t.row0 + warp * 16 + (lane >> 2), i1 = i0 + 8;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float o[8][4];
    clear(o);
    uint32_t qa[4][4];
    for (int kt = kt0; kt < kt1; kt++) {
        const int b = (kt - kt0) & 1;
        if (kt + 1 < kt1) {
            load_tile(sk + (b ^ 1) * TILE, a.io.k, hk, a, t, (kt + 1) * TB);
            load_tile(sv + (b ^ 1) * TILE, a.io.v, hk, a, t, (kt + 1) * TB);
            key_bits(bits[b ^ 1], a, t, (kt + 1) * TB);
        }
        copy_commit();
        copy_wait<1>();
        __syncthreads();
        if (kt == kt0) load_a(qa, sq, warp, lane);
        float s[8][4];
        mma_nt<T>(s, qa, sk + b * TILE, lane);
        const uint64_t there = bits[b][0] | (uint64_t)bits[b][1] << 32;
        if (there != ~0ull || edge(a.window, t.row0, TB, kt * TB, TB)) {
            // element (j, e) of this thread is key kt * 64 + 8 j + 2 (lane & 3) + e
            const int c0 = 2 * (lane & 3), k0 = kt * TB + c0;
            const uint64_t w = there >> c0;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const bool ok = (w >> (8 * j + e)) & 1;
                    const int key = k0 + 8 * j + e;
                    if (!ok || (a.window >= 0 && abs(i0 - key) > a.window)) s[j][e] = -INFINITY;
                    if (!ok || (a.window >= 0 && abs(i1 - key) > a.window)) s[j][2 + e] = -INFINITY;
                }
        }
        float x0 = s[0][0], x1 = s[0][2];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x0 = fmaxf(x0, fmaxf(s[j][0], s[j][1]));
            x1 = fmaxf(x1, fmaxf(s[j][2], s[j][3]));
        }
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
        x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
        x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float u0 = n0 == -INFINITY ? 0.f : n0 * sl2, u1 = n1 == -INFINITY ? 0.f : n1 * sl2;
        const float a0 = ex2_approx(m0 * sl2 - u0), a1 = ex2_approx(m1 * sl2 - u1);
        m0 = n0;
        m1 = n1;
        float r0 = 0.f, r1 = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            s[j][0] = ex2_approx(fmaf(s[j][0], sl2, -u0));
            s[j][1] = ex2_approx(fmaf(s[j][1], sl2, -u0));
            s[j][2] = ex2_approx(fmaf(s[j][2], sl2, -u1));
            s[j][3] = ex2_approx(fmaf(s[j][3], sl2, -u1));
            r0 += s[j][0] + s[j][1];
            r1 += s[j][2] + s[j][3];
            o[j][0] *= a0;
            o[j][1] *= a0;
            o[j][2] *= a1;
            o[j][3] *= a1;
        }
        l0 = l0 * a0 + r0;
        l1 = l1 * a1 + r1;
        mma_nn<T>(o, s, sv + b * TILE, lane);
        __syncthreads();  // every warp is done with this buffer before it is refilled
    }
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    const bool p0 = present(a, t, i0), p1 = present(a, t, i1);
    store_rows<T>(sq, a.io.out, h, t, t.row0, warp, lane, o, p0 ? 1.f / l0 : 0.f, p1 ? 1.f / l1 : 0.f);
    if (a.io.lse && (lane & 3) == 0) {
        float* g = a.io.lse + (long long)h * a.n_tokens + t.start;
        if (i0 < t.len) g[i0] = p0 ? m0 * a.scale + logf(l0) : -INFINITY;
        if (i1 < t.len) g[i1] = p1 ? m1 * a.scale + logf(l1) : -INFINITY;
    }
}

// ------------------------------------------------------------------ backward

// delta of 64 rows from their tiles of O and dO: two threads to a row.
template <typename T>
__device__ __forceinline__ void tile_delta(float* sdelta, const T* so, const T* sdo) {
    const int r = threadIdx.x >> 1, c0 = (threadIdx.x & 1) * 32;
    float acc = 0.f;
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint4 o = *reinterpret_cast<const uint4*>(so + swz(r, c0 + 8 * c));
        const uint4 d = *reinterpret_cast<const uint4*>(sdo + swz(r, c0 + 8 * c));
        const T* x = reinterpret_cast<const T*>(&o);
        const T* y = reinterpret_cast<const T*>(&d);
#pragma unroll
        for (int e = 0; e < 8; e++) acc = fmaf(to_float(x[e]), to_float(y[e]), acc);
    }
    acc += __shfl_xor_sync(0xffffffffu, acc, 1);
    if ((threadIdx.x & 1) == 0) sdelta[r] = acc;
}

// Which rows of a small call's sequence are there and which of them see FEW keys at
// most (absent tokens can leave them so few), a bit each.
struct RowBits {
    uint32_t there[SMALL_LEN / 32], few[SMALL_LEN / 32];
};

// few is to be read behind another barrier.
__device__ __forceinline__ void find_few(RowBits* bits, const AttnArgs& a, const SeqTile& t) {
    for (int i = threadIdx.x; i - (int)threadIdx.x < t.len; i += THREADS) {
        const uint32_t b = __ballot_sync(0xffffffffu, present(a, t, i));
        if ((threadIdx.x & 31) == 0) bits->there[i >> 5] = b;
    }
    __syncthreads();
    for (int i = threadIdx.x; i - (int)threadIdx.x < t.len; i += THREADS) {
        bool f = bits->there[i >> 5] >> (i & 31) & 1;
        if (f) {
            int lo, hi, count = 0;
            span(a, t, i, &lo, &hi);
            for (int w = lo >> 5; w <= hi >> 5 && count <= FEW; w++) {
                uint32_t keys = bits->there[w];
                if (w == lo >> 5) keys &= ~0u << (lo & 31);
                if (w == hi >> 5) keys &= ~0u >> (31 - (hi & 31));
                count += __popc(keys);
            }
            f = count <= FEW;
        }
        const uint32_t b = __ballot_sync(0xffffffffu, f);
        if ((threadIdx.x & 31) == 0) bits->few[i >> 5] = b;
    }
}
__device__ __forceinline__ bool any_few(const RowBits* bits, int row0) {
    return (bits->few[row0 >> 5] | bits->few[(row0 >> 5) + 1]) != 0;
}

// Their delta, of rows row0 .. row0 + 63 and one head, from P dP: eight lanes to a row.
template <typename T>
__device__ __forceinline__ void few_delta(float* sdelta, const RowBits* bits, const AttnArgs& a, const SeqTile& t,
                                          int h, int row0) {
    const int lane = threadIdx.x & 31, l = lane & 7, c = l * 8, hk = h / a.group;
    const uint32_t group = 0xffu << (lane & 24);
    for (int r = threadIdx.x >> 3; r < TB; r += THREADS / 8) {
        const int i = row0 + r;
        if (!(bits->few[i >> 5] >> (i & 31) & 1)) continue;
        const uint4 q = piece<T>(a.io.q, t.start + i, h, c), d = piece<T>(a.io.dout, t.start + i, h, c);
        const float e = a.io.lse[(long long)h * a.n_tokens + t.start + i] * LOG2E;
        float sum = 0.f;
        int lo, hi;
        span(a, t, i, &lo, &hi);
        for (int j = lo; j <= hi; j += 8) {
            uint32_t keys = __ballot_sync(group, j + l <= hi && present(a, t, j + l)) >> (lane & 24);
            for (; keys; keys &= keys - 1) {
                const long long at = t.start + j + __ffs(keys) - 1;
                float s = dot8<T>(q, piece<T>(a.io.k, at, hk, c)), dp = dot8<T>(d, piece<T>(a.io.v, at, hk, c));
#pragma unroll
                for (int x = 1; x < 8; x *= 2) {
                    s += __shfl_xor_sync(group, s, x);
                    dp += __shfl_xor_sync(group, dp, x);
                }
                sum = fmaf(ex2_approx(fmaf(s, a.scale * LOG2E, -e)), dp, sum);
            }
        }
        if (l == 0) sdelta[r] = sum;
    }
}

template <typename T, bool MASKED>
__device__ __forceinline__ void dq_block(const AttnArgs& a, const SeqTile& t, int h, uint8_t* smem, RowBits* rows) {
    T* sq = reinterpret_cast<T*>(smem);
    T* sdo = sq + TILE;
    T* sk = sdo + TILE;
    T* sv = sk + 2 * TILE;
    T* so = sv + 2 * TILE;
    float* sdelta = reinterpret_cast<float*>(so + TILE);
    __shared__ uint32_t bits[2][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = h / a.group;
    int kt0, kt1;
    visible_tiles(a, t, TB, TB, &kt0, &kt1);
    load_tile(sq, a.io.q, h, a, t, t.row0);
    load_tile(sdo, a.io.dout, h, a, t, t.row0);
    load_tile(so, a.io.out, h, a, t, t.row0);
    load_tile(sk, a.io.k, hk, a, t, kt0 * TB);
    load_tile(sv, a.io.v, hk, a, t, kt0 * TB);
    key_bits(bits[0], a, t, kt0 * TB);
    copy_commit();
    if (MASKED) find_few(rows, a, t);
    copy_wait<0>();
    __syncthreads();
    tile_delta(sdelta, so, sdo);
    __syncthreads();
    if (MASKED && any_few(rows, t.row0)) {
        few_delta<T>(sdelta, rows, a, t, h, t.row0);
        __syncthreads();
    }
    const float sl2 = a.scale * LOG2E;
    const int i0 = t.row0 + warp * 16 + (lane >> 2), i1 = i0 + 8;
    const bool p0 = present(a, t, i0), p1 = present(a, t, i1);
    const float* lse = a.io.lse + (long long)h * a.n_tokens + t.start;
    // absent rows have q = dO = 0: any finite lse gives them dS = 0
    const float e0 = p0 ? lse[i0] * LOG2E : 0.f, e1 = p1 ? lse[i1] * LOG2E : 0.f;
    const float d0 = sdelta[warp * 16 + (lane >> 2)], d1 = sdelta[warp * 16 + (lane >> 2) + 8];
    uint32_t qa[4][4], da[4][4];
    load_a(qa, sq, warp, lane);
    load_a(da, sdo, warp, lane);
    float dq[8][4];
    clear(dq);
    for (int kt = kt0; kt < kt1; kt++) {
        const int b = (kt - kt0) & 1;
        if (kt + 1 < kt1) {
            load_tile(sk + (b ^ 1) * TILE, a.io.k, hk, a, t, (kt + 1) * TB);
            load_tile(sv + (b ^ 1) * TILE, a.io.v, hk, a, t, (kt + 1) * TB);
            key_bits(bits[b ^ 1], a, t, (kt + 1) * TB);
        }
        copy_commit();
        copy_wait<1>();
        __syncthreads();
        float s[8][4], dp[8][4];
        mma_nt<T>(s, qa, sk + b * TILE, lane);
        mma_nt<T>(dp, da, sv + b * TILE, lane);
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                s[j][e] = ex2_approx(fmaf(s[j][e], sl2, -e0)) * (dp[j][e] - d0);
                s[j][2 + e] = ex2_approx(fmaf(s[j][2 + e], sl2, -e1)) * (dp[j][2 + e] - d1);
            }
        const uint64_t there = bits[b][0] | (uint64_t)bits[b][1] << 32;
        if (there != ~0ull || edge(a.window, t.row0, TB, kt * TB, TB)) {
            const int c0 = 2 * (lane & 3), k0 = kt * TB + c0;
            const uint64_t w = there >> c0;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const bool ok = (w >> (8 * j + e)) & 1;
                    const int key = k0 + 8 * j + e;
                    if (!ok || (a.window >= 0 && abs(i0 - key) > a.window)) s[j][e] = 0.f;
                    if (!ok || (a.window >= 0 && abs(i1 - key) > a.window)) s[j][2 + e] = 0.f;
                }
        }
        mma_nn<T>(dq, s, sk + b * TILE, lane);
        __syncthreads();
    }
    store_rows<T>(sq, a.io.dq, h, t, t.row0, warp, lane, dq, p0 ? a.scale : 0.f, p1 ? a.scale : 0.f);
}

template <typename T, bool MASKED>
__device__ __forceinline__ void dkv_block(const AttnArgs& a, const SeqTile& t, int hk, uint8_t* smem, RowBits* rows) {
    T* sk = reinterpret_cast<T*>(smem);
    T* sv = sk + TILE;
    T* sq = sv + TILE;
    T* sdo = sq + 2 * TILE;
    T* so = sdo + 2 * TILE;
    float* sdelta = reinterpret_cast<float*>(so + 2 * TILE);
    float* slse = sdelta + TB;  // [2][64]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int qt0, qt1;
    visible_tiles(a, t, TB, TB, &qt0, &qt1);
    const int nqt = qt1 - qt0, total = nqt * a.group;
    auto load_q = [&](int it, int b) {
        const int h = hk * a.group + it / nqt, row0 = (qt0 + it % nqt) * TB;
        load_tile(sq + b * TILE, a.io.q, h, a, t, row0);
        load_tile(sdo + b * TILE, a.io.dout, h, a, t, row0);
        load_tile(so + b * TILE, a.io.out, h, a, t, row0);
        if (threadIdx.x < TB) {
            const int r = threadIdx.x;
            const bool ok = present(a, t, row0 + r);
            const long long at = (long long)h * a.n_tokens + t.start + (ok ? row0 + r : 0);
            copy4(slse + b * TB + r, a.io.lse + at, ok);
        }
    };
    load_tile(sk, a.io.k, hk, a, t, t.row0);
    load_tile(sv, a.io.v, hk, a, t, t.row0);
    load_q(0, 0);
    copy_commit();
    if (MASKED) find_few(rows, a, t);  // read behind the loop's first barrier
    const float sl2 = a.scale * LOG2E;
    const int j0 = t.row0 + warp * 16 + (lane >> 2), j1 = j0 + 8;
    uint32_t ka[4][4], va[4][4];
    float dk[8][4], dv[8][4];
    clear(dk);
    clear(dv);
    for (int it = 0; it < total; it++) {
        const int b = it & 1;
        if (it + 1 < total) load_q(it + 1, b ^ 1);
        copy_commit();
        copy_wait<1>();
        __syncthreads();
        if (it == 0) {
            load_a(ka, sk, warp, lane);
            load_a(va, sv, warp, lane);
        }
        tile_delta(sdelta, so + b * TILE, sdo + b * TILE);  // read behind the barrier below
        const int row0 = (qt0 + it % nqt) * TB;
        if (MASKED && any_few(rows, row0)) {
            __syncthreads();
            few_delta<T>(sdelta, rows, a, t, hk * a.group + it / nqt, row0);
        }
        // transposed: rows are keys, columns queries
        float s[8][4], dp[8][4];
        mma_nt<T>(s, ka, sq + b * TILE, lane);
        const int c0 = 2 * (lane & 3);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float2 e = *reinterpret_cast<const float2*>(slse + b * TB + 8 * j + c0);
            s[j][0] = ex2_approx(fmaf(s[j][0], sl2, -e.x * LOG2E));
            s[j][1] = ex2_approx(fmaf(s[j][1], sl2, -e.y * LOG2E));
            s[j][2] = ex2_approx(fmaf(s[j][2], sl2, -e.x * LOG2E));
            s[j][3] = ex2_approx(fmaf(s[j][3], sl2, -e.y * LOG2E));
        }
        if (edge(a.window, row0, TB, t.row0, TB)) {
            const int q0 = row0 + c0;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if (abs(q0 + 8 * j + e - j0) > a.window) s[j][e] = 0.f;
                    if (abs(q0 + 8 * j + e - j1) > a.window) s[j][2 + e] = 0.f;
                }
        }
        mma_nn<T>(dv, s, sdo + b * TILE, lane);
        mma_nt<T>(dp, va, sdo + b * TILE, lane);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float2 d = *reinterpret_cast<const float2*>(sdelta + 8 * j + c0);
            s[j][0] *= dp[j][0] - d.x;
            s[j][1] *= dp[j][1] - d.y;
            s[j][2] *= dp[j][2] - d.x;
            s[j][3] *= dp[j][3] - d.y;
        }
        mma_nn<T>(dk, s, sq + b * TILE, lane);
        __syncthreads();
    }
    const bool p0 = present(a, t, j0), p1 = present(a, t, j1);
    store_rows<T>(sk, a.io.dk, hk, t, t.row0, warp, lane, dk, p0 ? a.scale : 0.f, p1 ? a.scale : 0.f);
    store_rows<T>(sv, a.io.dv, hk, t, t.row0, warp, lane, dv, p0 ? 1.f : 0.f, p1 ? 1.f : 0.f);
}

// ------------------------------------------------------------------ short sequences
// Of 64 tokens at most: one tile, so no search, no running maximum, and no
// second look at anything. Warps and steps of 16 rows that the sequence does
// not reach are left out.

// Sequence seq, if it has tokens.
__device__ __forceinline__ bool one_sequence(const AttnArgs& a, long long seq, SeqTile* t) {
    const int start = a.cu[seq], end = a.cu[seq + 1];
    *t = SeqTile{start, end - start, 0};
    if (run_ok(start, end, a.n_tokens, a.max_len)) return start < end;
    if (blockIdx.y == 0 && threadIdx.x == 0) atomicOr(a.status, ERR_BAD_INDEX);
    return false;
}

// What a thread holds of rows i0 and i1 becomes `gone` at keys (bits of
// `there`) that its row does not see.
__device__ __forceinline__ void hide(float (&s)[8][4], uint64_t there, int window, int i0, int i1, int lane, float gone) {
    if (there == ~0ull && !edge(window, 0, TB, 0, TB)) return;
    const int c0 = 2 * (lane & 3);
    const uint64_t w = there >> c0;
#pragma unroll
    for (int j = 0; j < 8; j++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const bool ok = (w >> (8 * j + e)) & 1;
            const int key = c0 + 8 * j + e;
            if (!ok || (window >= 0 && abs(i0 - key) > window)) s[j][e] = gone;
            if (!ok || (window >= 0 && abs(i1 - key) > window)) s[j][2 + e] = gone;
        }
}

constexpr int FWD_ONE_SMEM = 3 * TILE * 2;

template <typename T>
__global__ void __launch_bounds__(THREADS, 6) attention_fwd_one_kernel(const AttnArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    T* sq = reinterpret_cast<T*>(smem);
    T* sk = sq + TILE;
    T* sv = sk + TILE;
    __shared__ uint32_t bits[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y, hk = h / a.group;
    const float sl2 = a.scale * LOG2E;
    griddep_begin();
    for (long long seq = blockIdx.x; seq < a.n_seqs; seq += gridDim.x) {
        SeqTile t;
        if (!one_sequence(a, seq, &t)) continue;
        const int n = (t.len + 15) >> 4;
        load_tile(sq, a.io.q, h, a, t, 0, n);
        load_tile(sk, a.io.k, hk, a, t, 0, n);
        load_tile(sv, a.io.v, hk, a, t, 0, n);
        key_bits(bits, a, t, 0);
        copy_commit();
        const int i0 = warp * 16 + (lane >> 2), i1 = i0 + 8;
        const bool p0 = present(a, t, i0), p1 = present(a, t, i1);
        copy_wait<0>();
        __syncthreads();
        if (warp < n) {
            uint32_t f[4][4];
            float s[8][4], o[8][4];
            load_a(f, sq, warp, lane);
            mma_nt<T>(s, f, sk, lane, n);
            hide(s, bits[0] | (uint64_t)bits[1] << 32, a.window, i0, i1, lane, -INFINITY);
            float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    m0 = fmaxf(m0, s[j][e]);
                    m1 = fmaxf(m1, s[j][2 + e]);
                }
#pragma unroll
            for (int x = 1; x < 4; x *= 2) {
                m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
            }
            const float u0 = m0 == -INFINITY ? 0.f : m0 * sl2, u1 = m1 == -INFINITY ? 0.f : m1 * sl2;
            float l0 = 0.f, l1 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    s[j][e] = ex2_approx(fmaf(s[j][e], sl2, -u0));
                    s[j][2 + e] = ex2_approx(fmaf(s[j][2 + e], sl2, -u1));
                    l0 += s[j][e];
                    l1 += s[j][2 + e];
                }
#pragma unroll
            for (int x = 1; x < 4; x *= 2) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, x);
                l1 += __shfl_xor_sync(0xffffffffu, l1, x);
            }
            clear(o);
            mma_nn<T>(o, s, sv, lane, n);
            store_rows<T>(sq, a.io.out, h, t, 0, warp, lane, o, p0 ? 1.f / l0 : 0.f, p1 ? 1.f / l1 : 0.f);
            if (a.io.lse && (lane & 3) == 0) {
                float* g = a.io.lse + (long long)h * a.n_tokens + t.start;
                if (i0 < t.len) g[i0] = p0 ? m0 * a.scale + logf(l0) : -INFINITY;
                if (i1 < t.len) g[i1] = p1 ? m1 * a.scale + logf(l1) : -INFINITY;
            }
        }
        __syncthreads();  // the tiles are free for the next sequence
    }
}

// The backward pass, all of a sequence and key head in one block.
// S and dP are computed once, five products instead of seven; delta is the sum
// over P dP, which is all there, in f32 (attention_op_delta.cu says what that is
// worth).
template <bool SHARED>
constexpr int ONE_SMEM = (SHARED ? 7 : 6) * TILE * 2;

// SHARED: several query heads to a key head, whose dK and dV are then held
// while the next one's scores are computed: fewer blocks to an SM.
template <typename T, bool SHARED>
__device__ __forceinline__ void one_block(const AttnArgs& a, const SeqTile& t, int hk, uint8_t* smem) {
    T* sk = reinterpret_cast<T*>(smem);
    T* sv = sk + TILE;
    T* sq = sv + TILE;
    T* sdo = sq + TILE;
    T* sp = sdo + TILE;
    T* sds = sp + TILE;
    T* sdq = SHARED ? sds + TILE : sv;  // V is not needed again when it has one query head
    __shared__ uint32_t bits[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float sl2 = a.scale * LOG2E;
    const int n = (t.len + 15) >> 4;
    const int i0 = warp * 16 + (lane >> 2), i1 = i0 + 8;  // this thread's queries, then keys
    const bool p0 = present(a, t, i0), p1 = present(a, t, i1);
    load_tile(sk, a.io.k, hk, a, t, 0, n);
    load_tile(sv, a.io.v, hk, a, t, 0, n);
    key_bits(bits, a, t, 0);
    float dk[8][4], dv[8][4];
    if (SHARED) {
        clear(dk);
        clear(dv);
    }
    int h = hk * a.group;
    do {
        load_tile(sq, a.io.q, h, a, t, 0, n);
        load_tile(sdo, a.io.dout, h, a, t, 0, n);
        copy_commit();
        const float* lse = a.io.lse + (long long)h * a.n_tokens + t.start;
        const float e0 = p0 ? lse[i0] * LOG2E : 0.f, e1 = p1 ? lse[i1] * LOG2E : 0.f;
        copy_wait<0>();
        __syncthreads();
        float dp[8][4];  // later dQ
        if (warp < n) {
            uint32_t f[4][4];
            float s[8][4];
            load_a(f, sq, warp, lane);
            mma_nt<T>(s, f, sk, lane, n);
            load_a(f, sdo, warp, lane);
            mma_nt<T>(dp, f, sv, lane, n);
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    s[j][e] = ex2_approx(fmaf(s[j][e], sl2, -e0));
                    s[j][2 + e] = ex2_approx(fmaf(s[j][2 + e], sl2, -e1));
                }
            hide(s, bits[0] | (uint64_t)bits[1] << 32, a.window, i0, i1, lane, 0.f);
            float d0 = 0.f, d1 = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    d0 = fmaf(s[j][e], dp[j][e], d0);
                    d1 = fmaf(s[j][2 + e], dp[j][2 + e], d1);
                }
            put_rows<T>(sp, s, warp, lane);
#pragma unroll
            for (int x = 1; x < 4; x *= 2) {
                d0 += __shfl_xor_sync(0xffffffffu, d0, x);
                d1 += __shfl_xor_sync(0xffffffffu, d1, x);
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    s[j][e] *= dp[j][e] - d0;
                    s[j][2 + e] *= dp[j][2 + e] - d1;
                }
            put_rows<T>(sds, s, warp, lane);
            clear(dp);
            mma_nn<T>(dp, s, sk, lane, n);
        }
        __syncthreads();
        if (warp < n) store_rows<T>(sdq, a.io.dq, h, t, 0, warp, lane, dp, p0 ? a.scale : 0.f, p1 ? a.scale : 0.f);
        if (!SHARED) {
            clear(dk);
            clear(dv);
        }
        if (warp < n) {
            mma_tn<T>(dv, sp, sdo, warp, lane, n);
            mma_tn<T>(dk, sds, sq, warp, lane, n);
        }
        __syncthreads();
    } while (SHARED && ++h < (hk + 1) * a.group);
    if (warp < n) {
        store_rows<T>(sds, a.io.dk, hk, t, 0, warp, lane, dk, p0 ? a.scale : 0.f, p1 ? a.scale : 0.f);
        store_rows<T>(sp, a.io.dv, hk, t, 0, warp, lane, dv, p0 ? 1.f : 0.f, p1 ? 1.f : 0.f);
    }
}

template <typename T, bool SHARED>
__global__ void __launch_bounds__(THREADS, SHARED ? 3 : 4) attention_bwd_one_kernel(const AttnArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    griddep_begin();
    for (long long seq = blockIdx.x; seq < a.n_seqs; seq += gridDim.x) {
        SeqTile t;
        if (one_sequence(a, seq, &t)) one_block<T, SHARED>(a, t, blockIdx.y, smem);
    }
}

// ------------------------------------------------------------------ backward of a little work
constexpr int BWD_SMEM = 8 * TILE * 2 + 3 * TB * 4;
static_assert(BWD_SMEM >= ONE_SMEM<true>, "a short sequence's block");

// (inlined it would take registers from the longer ones' code)
template <typename T>
__device__ __noinline__ void short_sequence(const AttnArgs& a, const SeqTile& t, int hk, uint8_t* smem) {
    one_block<T, true>(a, t, hk, smem);
}

template <typename T, bool MASKED>
__global__ void __launch_bounds__(THREADS, 2)
    attention_bwd_kernel(const __grid_constant__ AttnArgs a, int n_heads) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ typename std::conditional<MASKED, RowBits, int>::type bits;
    RowBits* rows = reinterpret_cast<RowBits*>(&bits);
    SeqTile t;
    griddep_begin();
    if (!block_tile(a, &t)) return;
    const int y = blockIdx.y;
    if (t.len <= SHORT) {  // delta from P dP, whatever the call holds besides
        if (y >= n_heads) short_sequence<T>(a, t, y - n_heads, smem);
    } else if (y < n_heads) {
        dq_block<T, MASKED>(a, t, y, smem, rows);
    } else {
        dkv_block<T, MASKED>(a, t, y - n_heads, smem, rows);
    }
}

AttnArgs make_args(const laya_attention& a, const AttnIO& io) {
    AttnArgs g;
    g.cu = a.cu_seqlens;
    g.mask = a.token_mask;
    g.status = a.status;
    g.n_seqs = (int)a.n_seqs;
    g.n_tokens = (int)a.n_tokens;
    g.max_len = (int)(a.max_len < a.n_tokens ? a.max_len : a.n_tokens);
    g.group = (int)(a.n_heads / a.n_kv_heads);
    g.window = a.window;
    g.scale = a.scale;
    g.io = io;
    if (a.token_mask || narrow(a.window)) g.io.delta_short = io.delta;  // one kernel deals with all rows there
    return g;
}

}  // namespace

// Which kernels a call gets. Sequences of 64 tokens at most: a block to a
// sequence and head; otherwise 64-row mma.sync blocks for a little work (rows
// of all heads times keys, at most 2^20 x 3, in at most 64 sequences, of at
// most 512 tokens, because every entry of the table costs blocks), and tcgen05
// for the rest. Forward and backward of bf16, 12 heads, us by mma.sync /
// tcgen05: 1 x 256 tokens 17.1 / 27.0, 16 x 128 29.3 / 35.9; at the limit 1 x
// 512 36.3 / 36.1; beyond it 8 x 256 47.1 / 34.2, 64 x 100 99.8 / 66.1.
static bool small_call(const laya_attention& a) {
    return a.max_len <= SMALL_LEN && a.n_seqs <= 64 && a.n_heads <= 1024 &&
           (uint64_t)a.n_tokens * a.n_heads * a.max_len <= 3u << 20;
}

// Does the backward pass of short sequences take a block to a sequence and key
// head? Up to 32 tokens always: they take delta from P dP, which is there (1 x 16
// tokens, 12 heads 5.3 us, 5.2 in blocks of their own for dQ and for dK and dV); up to
// 64 in a narrow window for the same reason (1 x 64, window 2, 6.3 us, 19.8 with
// delta's own launch). Otherwise up to 64 when there are more than 96 of them: before
// that most SMs idle and the blocks of their own end sooner (12 heads over 12, blocks of
// their own / a block each: 1 x 64 4.3 / 5.9, 8 x 64 8.0 / 7.1, 32 x 64 17.3 / 11.4).
// Heads that share a key head lengthen a block: 12 over 4, 1 x 64 7.6 / 14.1, 24 x 64
// 16.5 / 20.1; 12 over 1, 64 x 64 42 / 69, and from 65 sequences to 96, where it is no
// longer a small call, 31-36 on tcgen05.
static bool one_block_each(const laya_attention& a) {
    return a.max_len <= SHORT ||
           (a.max_len <= TB && (narrow(a.window) || (uint64_t)a.n_seqs * a.n_kv_heads > 96));
}

// A few times the blocks that the GPU holds at once: a block takes every
// gridDim.x-th sequence.
static cudaError_t launch_one(void (*kernel)(AttnArgs), int smem, unsigned heads, const AttnArgs& g, cudaStream_t stream) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const unsigned most = (148 * 16 + heads - 1) / heads;
    return launch_k(kernel, dim3((unsigned)g.n_seqs < most ? g.n_seqs : most, heads), dim3(THREADS), smem, stream, g);
}

cudaError_t launch_attention_fwd(const laya_attention& a, const AttnIO& io, cudaStream_t stream) {
    const bool bf16 = a.elem_dtype == LAYA_DT_BF16;
    const AttnArgs g = make_args(a, io);
    if (a.max_len <= TB)
        return launch_one(bf16 ? attention_fwd_one_kernel<__nv_bfloat16> : attention_fwd_one_kernel<__half>, FWD_ONE_SMEM,
                          a.n_heads, g, stream);
    if (!small_call(a)) return launch_attention_fwd_tc(bf16, (int)a.n_heads, g, stream);
    auto kernel = bf16 ? attention_fwd_kernel<__nv_bfloat16> : attention_fwd_kernel<__half>;
    const dim3 grid((unsigned)seq_tiles(g.n_tokens, g.n_seqs, TB), a.n_heads);
    return launch_k(kernel, grid, dim3(THREADS), FWD_SMEM, stream, g);
}

cudaError_t launch_attention_bwd(const laya_attention& a, const AttnIO& io, cudaStream_t stream) {
    const bool bf16 = a.elem_dtype == LAYA_DT_BF16;
    const AttnArgs g = make_args(a, io);
    if (one_block_each(a)) {
        if (g.group > 1)
            return launch_one(bf16 ? attention_bwd_one_kernel<__nv_bfloat16, true> : attention_bwd_one_kernel<__half, true>,
                              ONE_SMEM<true>, a.n_kv_heads, g, stream);
        return launch_one(bf16 ? attention_bwd_one_kernel<__nv_bfloat16, false> : attention_bwd_one_kernel<__half, false>,
                          ONE_SMEM<false>, a.n_kv_heads, g, stream);
    }
    if (!small_call(a) || narrow(a.window))
        return launch_attention_bwd_tc(bf16, (int)a.n_heads, (int)a.n_kv_heads, g, stream);
    auto kernel = a.token_mask ? (bf16 ? attention_bwd_kernel<__nv_bfloat16, true> : attention_bwd_kernel<__half, true>)
                               : (bf16 ? attention_bwd_kernel<__nv_bfloat16, false> : attention_bwd_kernel<__half, false>);
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BWD_SMEM);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)seq_tiles(g.n_tokens, g.n_seqs, TB), a.n_heads + a.n_kv_heads);
    return launch_k(kernel, grid, dim3(THREADS), BWD_SMEM, stream, g, (int)a.n_heads);
}

}  // namespace laya
