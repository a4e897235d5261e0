// attention_op_tc.cu -- the attention operator on tcgen05: forward, dQ, and
// dK with dV (the formulas are in attention_op.cu).
//
// One CTA takes 128 rows (queries, or keys for dK and dV) of one head, one to
// a TMEM lane, and walks the other side in tiles of 64:
//
//   warps 0-3  the softmax's arithmetic: thread t owns row t, reads its 64
//              scores from TMEM, and writes P or dS back as 16-bit pairs over
//              the scores it has read. A lane's columns are its thread's
//              alone, so that needs no barrier among the threads, and the
//              next product takes P or dS from TMEM as its A operand.
//   warp 4     loads: TMA boxes of 64 rows x 128 bytes into a ring of STAGES
//              tile pairs. A box of the packed rows also brings the rows of
//              absent tokens and of the next sequence; in tiles that have
//              such rows the warp overwrites them with zeros once the box has
//              landed, while the next one is on its way, before it hands the
//              stage over. (The 128-row tile needs none of that: its rows
//              are the MMA's M index, and nothing crosses from one to another.)
//   warp 5     owns TMEM and issues the MMAs.
//
// TMEM holds 256 columns a CTA (two S tiles, or S and dP; one or two 64-wide
// accumulators), so two CTAs share an SM: while one waits for a product the
// other has the SFU, which bounds all three kernels (a 128 x 64 tile costs
// 512 cycles of ex2 an SM sub-partition, its products 320 to 640).
//
// TMEM is only overwritten by a product after the barrier that says its last
// reader is done: MMAs to different accumulators are not taken to be ordered.
// Every wait is bounded (common.cuh); a CTA that gives up records it, waits
// for its own copies and MMAs, frees TMEM and leaves.
#include <type_traits>

#include "attention_op.cuh"
#include "gemm.cuh"

namespace laya {
namespace {

constexpr int ROWS = 128;  // rows per CTA, one TMEM lane each
constexpr int STEP = 64;   // rows of the other side per tile
constexpr int STAGES = 3;
constexpr int THREADS = 192;
constexpr int BIG = ROWS * 64 * 2;    // 16 KB
constexpr int SMALL = STEP * 64 * 2;  // 8 KB
constexpr uint32_t COLS = 256;

struct Bars {
    uint64_t full[STAGES], empty[STAGES], landed[STAGES];
    uint64_t s_full[2], dp_full;  // products ready for the softmax warps
    uint64_t p_full, ds_full;     // operands ready for the MMA warp
    uint64_t done[2];             // the products that read them are complete
    uint64_t all_done;
    uint32_t tmem;
    int abort;
};

// Per stage: two words of presence bits (keys), or 64 values each of -lse *
// log2 e and delta (queries).
struct Extra {
    float lse[STAGES][STEP], delta[STAGES][STEP];
    uint32_t bits[STAGES][2];
};

constexpr int smem_bytes(int big_tiles) {
    return big_tiles * BIG + STAGES * 2 * SMALL + (int)sizeof(Bars) + (int)sizeof(Extra) + 16 + 1024;
}

struct Frame {
    uint8_t* smem;  // big tiles, then the ring
    uint8_t* ring;
    Bars* bar;
    Extra* extra;
    uint32_t tmem;
};

__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity, int* err) {
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity))
        if (globaltimer() - t0 > WAIT_LIMIT_NS) {
            atomicOr(err, ERR_WAIT_TIMEOUT);
            return;
        }
}

// ------------------------------------------------------------------ loads

// Presence bits of N * 32 rows of the sequence from row0.
template <int N>
__device__ __forceinline__ void row_bits(uint32_t (&bits)[N], const AttnArgs& a, const SeqTile& t, int row0, int lane) {
#pragma unroll
    for (int i = 0; i < N; i++) bits[i] = __ballot_sync(0xffffffffu, present(a, t, row0 + i * 32 + lane));
}

// The loading warp's side of the ring. A stage is full when its boxes have
// landed, zeroed where they must be, and every lane has arrived (32 lanes, and
// lane 0 once more: with the bytes it expects, or for them).
struct Ring {
    const Frame& f;
    const AttnArgs& a;
    const CUtensorMap *m0, *m1;
    int lane;
    int issued = 0;
    int patch = -1;  // the stage that waits for its zeros
    uint32_t patch_bits[2] = {0, 0};
    uint32_t landed_parity = 0;  // one bit a stage

    __device__ __forceinline__ void fill() {
        if (patch < 0) return;
        Bars* bar = f.bar;
        const bool ok = mbar_wait(&bar->landed[patch], landed_parity >> patch & 1, a.status, &bar->abort);
        landed_parity ^= 1u << patch;
        if (ok) {
            uint8_t* s = f.ring + patch * 2 * SMALL;
            const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < 2; w++)
                for (uint32_t gone = ~patch_bits[w]; gone; gone &= gone - 1) {
                    const int r = w * 32 + __ffs(gone) - 1;  // 16 lanes a row: both tiles
                    if (lane < 16) *reinterpret_cast<uint4*>(s + (lane >> 3) * SMALL + r * 128 + (lane & 7) * 16) = zero;
                }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->full[patch]);
        mbar_arrive(&bar->full[patch]);
        patch = -1;
    }
    // Room for the next stage; a warp that has to wait first hands over what it holds.
    __device__ __forceinline__ bool room() {
        const int s = issued % STAGES;
        const uint32_t parity = ((issued / STAGES) & 1) ^ 1;
        if (__all_sync(0xffffffffu, mbar_try_wait(&f.bar->empty[s], parity))) return true;
        fill();
        return __all_sync(0xffffffffu, mbar_wait(&f.bar->empty[s], parity, a.status, &f.bar->abort));
    }
    // Rows `row` of both arrays (columns `col0`, `col1`) into the next stage;
    // with the first go `big` tiles of rows `big_row` (columns `big0`, `big1`).
    __device__ __forceinline__ void load(int col0, int col1, int row, const uint32_t (&bits)[2], const CUtensorMap* big0,
                                         const CUtensorMap* big1, int big_col, int big_row) {
        Bars* bar = f.bar;
        const int s = issued % STAGES;
        const bool whole = (bits[0] & bits[1]) == ~0u;
        if (lane == 0) {
            uint64_t* b = whole ? &bar->full[s] : &bar->landed[s];
            const bool first = issued == 0;
            mbar_arrive_expect_tx(b, 2 * SMALL + (first ? (big1 ? 2 : 1) * BIG : 0));
            if (first) {
                for (int i = 0; i < 2; i++) {
                    tma_load_2d(f.smem + i * SMALL, big0, b, big_col, big_row + i * STEP);
                    if (big1) tma_load_2d(f.smem + BIG + i * SMALL, big1, b, big_col, big_row + i * STEP);
                }
            }
            tma_load_2d(f.ring + 2 * s * SMALL, m0, b, col0, row);
            tma_load_2d(f.ring + (2 * s + 1) * SMALL, m1, b, col1, row);
        }
        issued++;
        fill();
        if (whole) {
            mbar_arrive(&bar->full[s]);
        } else {
            patch = s;
            patch_bits[0] = bits[0];
            patch_bits[1] = bits[1];
        }
    }
    // Every box has landed before shared memory goes away.
    __device__ __forceinline__ void finish() {
        fill();
        for (int j = max(0, issued - STAGES); j < issued; j++) drain(&f.bar->full[j % STAGES], (j / STAGES) & 1, a.status);
    }
};

// ------------------------------------------------------------------ TMEM rows

__device__ __forceinline__ void load64(uint32_t taddr, float (&v)[64]) {
    tmem_ld32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
    tmem_ld32(taddr + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
    tc_wait_ld();
}

// 32 values as 16-bit pairs into 16 columns.
template <typename T>
__device__ __forceinline__ void store_pairs(uint32_t taddr, const float* v) {
    uint32_t p[16];
#pragma unroll
    for (int i = 0; i < 16; i++) p[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    tmem_st16(taddr, p);
}

// A thread's accumulator row (64 columns), times f (0: zeros), to global memory.
template <typename T>
__device__ __forceinline__ void store_row(uint32_t taddr, T* dst, bool write, float f) {
    float v[64];
    load64(taddr, v);
    if (!write) return;
    uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll
    for (int c = 0; c < 8; c++) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (f != 0.f) {
            u.x = pack2<T>(v[8 * c] * f, v[8 * c + 1] * f);
            u.y = pack2<T>(v[8 * c + 2] * f, v[8 * c + 3] * f);
            u.z = pack2<T>(v[8 * c + 4] * f, v[8 * c + 5] * f);
            u.w = pack2<T>(v[8 * c + 6] * f, v[8 * c + 7] * f);
        }
        d[c] = u;
    }
}

// v[i] = to where key col0 + i is not there or lies outside row's window.
__device__ __forceinline__ void mask_row(float (&v)[64], const uint32_t (&bits)[2], int window, int row, int col0,
                                         float to) {
    const unsigned span = window >= 0 ? 2u * (unsigned)window : 0xffffffffu;
    const unsigned d = (unsigned)(col0 - row) + (window >= 0 ? (unsigned)window : 0u);
#pragma unroll
    for (int i = 0; i < 64; i++)
        if (!(bits[i / 32] >> (i & 31) & 1) || (window >= 0 && d + i > span)) v[i] = to;
}

// ------------------------------------------------------------------ MMAs

template <typename T>
constexpr uint32_t IDESC = idesc_f16(ROWS, STEP, std::is_same<T, __nv_bfloat16>::value);
constexpr uint32_t B_MN = 1u << 16;  // B is MN-major (its rows are the sum's index)

// D (128 x 64) = A . B^T, both K-major in shared memory, over the head.
template <typename T>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b) {
#pragma unroll
    for (int ks = 0; ks < 4; ks++)
        tc_mma_f16(d, sw128_desc(a) + 2 * ks, sw128_desc(b) + 2 * ks, IDESC<T>, ks != 0);
}

// D (128 x 64) += P . B, P (128 x 64, 16-bit pairs) in TMEM, B's 64 rows summed over.
template <typename T>
__device__ __forceinline__ void mma_sum(uint32_t d, uint32_t p, uint32_t b, bool accumulate) {
#pragma unroll
    for (int ks = 0; ks < 4; ks++)
        tc_mma_f16_ts(d, p + 8 * ks, sw128_desc(b + ks * 2048), IDESC<T> | B_MN, accumulate || ks != 0);
}

// ------------------------------------------------------------------ CTA frame

template <int BIG_TILES>
__device__ __forceinline__ Frame open_frame(uint8_t* raw, int warp) {
    Frame f;
    f.smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    f.ring = f.smem + BIG_TILES * BIG;
    f.bar = reinterpret_cast<Bars*>(f.ring + STAGES * 2 * SMALL);
    f.extra = reinterpret_cast<Extra*>(
        (reinterpret_cast<uintptr_t>(f.bar) + sizeof(Bars) + 15) & ~uintptr_t(15));
    if (threadIdx.x == 0) {
        Bars* b = f.bar;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&b->full[s], 33);
            mbar_init(&b->empty[s], 1);
            mbar_init(&b->landed[s], 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(&b->s_full[s], 1);
            mbar_init(&b->done[s], 1);
        }
        mbar_init(&b->dp_full, 1);
        mbar_init(&b->p_full, ROWS);
        mbar_init(&b->ds_full, ROWS);
        mbar_init(&b->all_done, 1);
        b->abort = 0;
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == 5) {
        tmem_alloc(&f.bar->tmem, COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    f.tmem = f.bar->tmem;
    return f;
}

__device__ __forceinline__ void close_frame(const Frame& f, int warp) {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 5) tmem_dealloc(f.tmem, COLS);
}

__device__ __forceinline__ bool block_tile(const AttnArgs& a, SeqTile* t) {
    if (threadIdx.x == 0 && blockIdx.y == 0)
        check_table(a.cu, a.n_seqs, a.n_tokens, a.max_len, blockIdx.x, a.status);
    return find_tile(a.cu, a.n_seqs, a.n_tokens, a.max_len, ROWS, blockIdx.x, threadIdx.x & 31, t);
}

// Warp-wide wait of the softmax warps.
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, const AttnArgs& a, Bars* b) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, a.status, &b->abort));
}

// ------------------------------------------------------------------ forward
constexpr int FWD_SMEM = smem_bytes(1);

template <typename T>
__global__ void __launch_bounds__(THREADS, 2)
    attention_fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                            const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap,
                            const AttnArgs a) {
    extern __shared__ uint8_t raw[];
    SeqTile t;
    if (!block_tile(a, &t)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y, hk = h / a.group;
    int kt0, kt1;
    visible_tiles(a, t, ROWS, STEP, &kt0, &kt1);
    const int n = kt1 - kt0;
    const Frame f = open_frame<1>(raw, warp);
    Bars* bar = f.bar;
    // TMEM: S 0, 1 at columns 0, 64 (P over them); O at 128

    if (warp == 4) {
        Ring ring{f, a, &mk, &mv, lane};
        for (int j = 0; j < n; j++) {
            uint32_t bits[2];
            row_bits(bits, a, t, (kt0 + j) * STEP, lane);
            if (!ring.room()) break;
            if (lane < 2) f.extra->bits[j % STAGES][lane] = lane ? bits[1] : bits[0];
            ring.load(hk * 64, hk * 64, t.start + (kt0 + j) * STEP, bits, &mq, nullptr, h * 64, t.start + t.row0);
        }
        ring.finish();
    } else if (warp == 5) {
        if (lane == 0) {
            const uint32_t q = smem_u32(f.smem), kv = smem_u32(f.ring);
            bool ok = true;
            auto scores = [&](int j) {
                const int s = j % STAGES;
                ok = mbar_wait(&bar->full[s], (j / STAGES) & 1, a.status, &bar->abort);
                if (!ok) return;
                tc_fence_after();
                mma_rows<T>(f.tmem + (j & 1) * 64, q, kv + 2 * s * SMALL);
                tc_commit(&bar->s_full[j & 1]);
            };
            scores(0);
            if (ok && n > 1) scores(1);
            for (int j = 0; j < n && ok; j++) {
                const int s = j % STAGES;
                ok = mbar_wait(&bar->p_full, j & 1, a.status, &bar->abort);
                if (!ok) break;
                tc_fence_after();
                mma_sum<T>(f.tmem + 128, f.tmem + (j & 1) * 64, kv + (2 * s + 1) * SMALL, j != 0);
                tc_commit(&bar->empty[s]);
                tc_commit(&bar->done[0]);
                if (j + 2 < n) {
                    ok = mbar_wait(&bar->done[0], j & 1, a.status, &bar->abort);
                    if (ok) scores(j + 2);
                }
            }
            tc_commit(&bar->all_done);
            drain(&bar->all_done, 0, a.status);
        }
        __syncwarp();
    } else {
        const int i = t.row0 + threadIdx.x;  // query
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const uint32_t t_o = f.tmem + lanes + 128;
        const float sl2 = a.scale * LOG2E;
        constexpr float RESCALE = 8.0f;  // exponent growth that moves the reference point
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        for (int j = 0; j < n; j++) {
            const uint32_t t_s = f.tmem + lanes + (j & 1) * 64;
            const int s = j % STAGES;
            ok = wait_all(&bar->full[s], (j / STAGES) & 1, a, bar) && wait_all(&bar->s_full[j & 1], (j >> 1) & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
            float v[64];
            load64(t_s, v);
            const uint32_t bits[2] = {f.extra->bits[s][0], f.extra->bits[s][1]};
            if ((bits[0] & bits[1]) != ~0u || edge(a.window, t.row0, ROWS, (kt0 + j) * STEP, STEP))
                mask_row(v, bits, a.window, i, (kt0 + j) * STEP, -INFINITY);
            float mx[8];
#pragma unroll
            for (int c = 0; c < 8; c++) mx[c] = fmaxf(v[c], v[c + 8]);
#pragma unroll
            for (int c = 16; c < 64; c++) mx[c & 7] = fmaxf(mx[c & 7], v[c]);
            const float top =
                fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
            // The reference point moves when the maximum has grown by more
            // than 2^8 (p stays below 2^8 otherwise): then O and l shrink.
            float alpha = 1.f;
            const bool move = j == 0 || (top - m) * sl2 > RESCALE;
            if (move) {
                alpha = ex2_approx((m - top) * sl2);  // m = -inf: 0 (NaN if top is -inf too, of an l and O of 0)
                alpha = m == -INFINITY ? 0.f : alpha;
                m = top;
                l *= alpha;
            }
            const float u = m == -INFINITY ? 0.f : m * sl2;
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 64; c++) {
                v[c] = ex2_approx(fmaf(v[c], sl2, -u));
                sum[c & 3] += v[c];
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            store_pairs<T>(t_s, v);
            store_pairs<T>(t_s + 16, v + 32);
            if (j > 0) {
                ok = wait_all(&bar->done[0], (j - 1) & 1, a, bar);
                if (!ok) break;
                if (__any_sync(0xffffffffu, move)) {
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        uint32_t r[32];
                        tmem_ld32(t_o + c, r);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; e++) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
                        tmem_st32(t_o + c, r);
                    }
                }
            }
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&bar->p_full);
        }
        if (ok) ok = wait_all(&bar->all_done, 0, a, bar);
        if (ok) {
            tc_fence_after();
            const bool there = present(a, t, i), write = i < t.len;
            T* out = static_cast<T*>(a.io.out.p) + ((long long)t.start + (write ? i : 0)) * a.io.out.ld + h * 64;
            store_row<T>(t_o, out, write, there ? 1.f / l : 0.f);
            if (a.io.lse && write)
                a.io.lse[(long long)h * a.n_tokens + t.start + i] = there ? m * a.scale + logf(l) : -INFINITY;
        }
    }
    close_frame(f, warp);
}

// ------------------------------------------------------------------ dQ (and delta)
constexpr int DQ_SMEM = smem_bytes(2);

template <typename T>
__global__ void __launch_bounds__(THREADS, 2)
    attention_dq_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                           const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                           const AttnArgs a) {
    extern __shared__ uint8_t raw[];
    SeqTile t;
    if (!block_tile(a, &t)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.y, hk = h / a.group;
    int kt0, kt1;
    visible_tiles(a, t, ROWS, STEP, &kt0, &kt1);
    const int n = kt1 - kt0;
    const Frame f = open_frame<2>(raw, warp);
    Bars* bar = f.bar;
    // TMEM: S 0, 1 at columns 0, 64 (dS over them); dP at 128; dQ at 192

    if (warp == 4) {
        Ring ring{f, a, &mk, &mv, lane};
        for (int j = 0; j < n; j++) {
            uint32_t bits[2];
            row_bits(bits, a, t, (kt0 + j) * STEP, lane);
            if (!ring.room()) break;
            if (lane < 2) f.extra->bits[j % STAGES][lane] = lane ? bits[1] : bits[0];
            ring.load(hk * 64, hk * 64, t.start + (kt0 + j) * STEP, bits, &mq, &mdo, h * 64, t.start + t.row0);
        }
        ring.finish();
    } else if (warp == 5) {
        if (lane == 0) {
            const uint32_t q = smem_u32(f.smem), dout = q + BIG, kv = smem_u32(f.ring);
            bool ok = true;
            auto scores = [&](int j) {
                const int s = j % STAGES;
                ok = mbar_wait(&bar->full[s], (j / STAGES) & 1, a.status, &bar->abort);
                if (!ok) return;
                tc_fence_after();
                mma_rows<T>(f.tmem + (j & 1) * 64, q, kv + 2 * s * SMALL);
                tc_commit(&bar->s_full[j & 1]);
            };
            auto dp = [&](int j) {
                mma_rows<T>(f.tmem + 128, dout, kv + (2 * (j % STAGES) + 1) * SMALL);
                tc_commit(&bar->dp_full);
            };
            scores(0);
            if (ok) dp(0);
            if (ok && n > 1) scores(1);
            for (int j = 0; j < n && ok; j++) {
                const int s = j % STAGES;
                ok = mbar_wait(&bar->ds_full, j & 1, a.status, &bar->abort);
                if (!ok) break;
                tc_fence_after();
                if (j + 1 < n) dp(j + 1);  // dP(j) has been read
                mma_sum<T>(f.tmem + 192, f.tmem + (j & 1) * 64, kv + 2 * s * SMALL, j != 0);
                tc_commit(&bar->empty[s]);
                tc_commit(&bar->done[0]);
                if (j + 2 < n) {
                    ok = mbar_wait(&bar->done[0], j & 1, a.status, &bar->abort);
                    if (ok) scores(j + 2);
                }
            }
            tc_commit(&bar->all_done);
            drain(&bar->all_done, 0, a.status);
        }
        __syncwarp();
    } else {
        const int r = threadIdx.x, i = t.row0 + r;  // query
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const float sl2 = a.scale * LOG2E;
        const bool there = present(a, t, i);
        const long long at = (long long)h * a.n_tokens + t.start + i;
        // absent rows have q = dO = 0: any finite lse gives them dS = 0
        const float e = there ? a.io.lse[at] * LOG2E : 0.f;
        uint4 o[8];
        if (there) {
            const uint4* g = reinterpret_cast<const uint4*>(static_cast<const T*>(a.io.out.p) +
                                                            ((long long)t.start + i) * a.io.out.ld + h * 64);
#pragma unroll
            for (int c = 0; c < 8; c++) o[c] = g[c];
        }
        bool ok = wait_all(&bar->full[0], 0, a, bar);  // dO came with the first keys
        float delta = 0.f;
        if (ok) {
            if (there) {
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const uint4 d = *reinterpret_cast<const uint4*>(f.smem + BIG + r * 128 + ((c ^ (r & 7)) << 4));
                    const T* x = reinterpret_cast<const T*>(&o[c]);
                    const T* y = reinterpret_cast<const T*>(&d);
#pragma unroll
                    for (int k = 0; k < 8; k++) delta = fmaf(to_float(x[k]), to_float(y[k]), delta);
                }
            }
            if (i < t.len) a.io.delta[at] = delta;
        }
        for (int j = 0; j < n && ok; j++) {
            const uint32_t t_s = f.tmem + lanes + (j & 1) * 64;
            const int s = j % STAGES;
            ok = wait_all(&bar->full[s], (j / STAGES) & 1, a, bar) && wait_all(&bar->s_full[j & 1], (j >> 1) & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
            float v[64];
            load64(t_s, v);
#pragma unroll
            for (int c = 0; c < 64; c++) v[c] = ex2_approx(fmaf(v[c], sl2, -e));
            const uint32_t bits[2] = {f.extra->bits[s][0], f.extra->bits[s][1]};
            if ((bits[0] & bits[1]) != ~0u || edge(a.window, t.row0, ROWS, (kt0 + j) * STEP, STEP))
                mask_row(v, bits, a.window, i, (kt0 + j) * STEP, 0.f);
            ok = wait_all(&bar->dp_full, j & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float d[32];
                tmem_ld32(f.tmem + lanes + 128 + half * 32, *reinterpret_cast<uint32_t(*)[32]>(&d[0]));
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 32; c++) d[c] = v[half * 32 + c] * (d[c] - delta);
                store_pairs<T>(t_s + half * 16, d);
            }
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&bar->ds_full);
        }
        if (ok) ok = wait_all(&bar->all_done, 0, a, bar);
        if (ok) {
            tc_fence_after();
            const bool write = i < t.len;
            T* dq = static_cast<T*>(a.io.dq.p) + ((long long)t.start + (write ? i : 0)) * a.io.dq.ld + h * 64;
            store_row<T>(f.tmem + lanes + 192, dq, write, there ? a.scale : 0.f);
        }
    }
    close_frame(f, warp);
}

// ------------------------------------------------------------------ dK, dV
constexpr int DKV_SMEM = smem_bytes(2);

template <typename T>
__global__ void __launch_bounds__(THREADS, 2)
    attention_dkv_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                           const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                           const AttnArgs a) {
    extern __shared__ uint8_t raw[];
    SeqTile t;
    if (!block_tile(a, &t)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hk = blockIdx.y;
    int qt0, qt1;
    visible_tiles(a, t, ROWS, STEP, &qt0, &qt1);
    const int nq = qt1 - qt0, n = nq * a.group;  // the query tiles of every head of the group
    const Frame f = open_frame<2>(raw, warp);
    Bars* bar = f.bar;
    // TMEM: S^T at column 0 (P^T over it); dP^T at 64 (dS^T over it); dV at 128; dK at 192

    if (warp == 4) {
        Ring ring{f, a, &mq, &mdo, lane};
        for (int j = 0; j < n; j++) {
            const int h = hk * a.group + j / nq, row0 = (qt0 + j % nq) * STEP;
            uint32_t bits[2];
            row_bits(bits, a, t, row0, lane);
            // statistics of rows lane and lane + 32 (0 for rows that are not there: q = dO = 0)
            const long long g = (long long)h * a.n_tokens + t.start + row0 + lane;
            const bool b0 = bits[0] >> lane & 1, b1 = bits[1] >> lane & 1;
            const float l0 = b0 ? a.io.lse[g] : 0.f, l1 = b1 ? a.io.lse[g + 32] : 0.f;
            const float d0 = b0 ? a.io.delta[g] : 0.f, d1 = b1 ? a.io.delta[g + 32] : 0.f;
            if (!ring.room()) break;
            const int s = j % STAGES;
            f.extra->lse[s][lane] = -LOG2E * l0;
            f.extra->lse[s][lane + 32] = -LOG2E * l1;
            f.extra->delta[s][lane] = d0;
            f.extra->delta[s][lane + 32] = d1;
            ring.load(h * 64, h * 64, t.start + row0, bits, &mk, &mv, hk * 64, t.start + t.row0);
        }
        ring.finish();
    } else if (warp == 5) {
        if (lane == 0) {
            const uint32_t k = smem_u32(f.smem), v = k + BIG, qd = smem_u32(f.ring);
            bool ok = mbar_wait(&bar->full[0], 0, a.status, &bar->abort);
            if (ok) {
                tc_fence_after();
                mma_rows<T>(f.tmem, k, qd);
                tc_commit(&bar->s_full[0]);
                mma_rows<T>(f.tmem + 64, v, qd + SMALL);
                tc_commit(&bar->dp_full);
            }
            for (int j = 0; j < n && ok; j++) {
                const int s = j % STAGES, s1 = (j + 1) % STAGES;
                ok = mbar_wait(&bar->p_full, j & 1, a.status, &bar->abort);
                if (!ok) break;
                tc_fence_after();
                mma_sum<T>(f.tmem + 128, f.tmem, qd + (2 * s + 1) * SMALL, j != 0);
                tc_commit(&bar->done[0]);
                if (j + 1 < n) {
                    ok = mbar_wait(&bar->full[s1], ((j + 1) / STAGES) & 1, a.status, &bar->abort) &&
                         mbar_wait(&bar->done[0], j & 1, a.status, &bar->abort);
                    if (!ok) break;
                    tc_fence_after();
                    mma_rows<T>(f.tmem, k, qd + 2 * s1 * SMALL);
                    tc_commit(&bar->s_full[0]);
                }
                ok = mbar_wait(&bar->ds_full, j & 1, a.status, &bar->abort);
                if (!ok) break;
                tc_fence_after();
                mma_sum<T>(f.tmem + 192, f.tmem + 64, qd + 2 * s * SMALL, j != 0);
                tc_commit(&bar->empty[s]);
                tc_commit(&bar->done[1]);
                if (j + 1 < n) {
                    ok = mbar_wait(&bar->done[1], j & 1, a.status, &bar->abort);
                    if (!ok) break;
                    tc_fence_after();
                    mma_rows<T>(f.tmem + 64, v, qd + (2 * s1 + 1) * SMALL);
                    tc_commit(&bar->dp_full);
                }
            }
            tc_commit(&bar->all_done);
            drain(&bar->all_done, 0, a.status);
        }
        __syncwarp();
    } else {
        const int i = t.row0 + threadIdx.x;  // key
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const uint32_t t_s = f.tmem + lanes, t_dp = t_s + 64;
        const float sl2 = a.scale * LOG2E;
        bool ok = true;
        for (int j = 0; j < n; j++) {
            const int s = j % STAGES;
            ok = wait_all(&bar->full[s], (j / STAGES) & 1, a, bar) && wait_all(&bar->s_full[0], j & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
            float v[64];
            load64(t_s, v);
            const float4* lse = reinterpret_cast<const float4*>(f.extra->lse[s]);
#pragma unroll
            for (int c = 0; c < 16; c++) {
                const float4 e = lse[c];
                v[4 * c] = ex2_approx(fmaf(v[4 * c], sl2, e.x));
                v[4 * c + 1] = ex2_approx(fmaf(v[4 * c + 1], sl2, e.y));
                v[4 * c + 2] = ex2_approx(fmaf(v[4 * c + 2], sl2, e.z));
                v[4 * c + 3] = ex2_approx(fmaf(v[4 * c + 3], sl2, e.w));
            }
            const int row0 = (qt0 + j % nq) * STEP;
            if (edge(a.window, row0, STEP, t.row0, ROWS)) {
                const uint32_t all[2] = {~0u, ~0u};
                mask_row(v, all, a.window, i, row0, 0.f);
            }
            store_pairs<T>(t_s, v);
            store_pairs<T>(t_s + 16, v + 32);
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&bar->p_full);
            ok = wait_all(&bar->dp_full, j & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
            const float4* delta = reinterpret_cast<const float4*>(f.extra->delta[s]);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                float d[32];
                tmem_ld32(t_dp + half * 32, *reinterpret_cast<uint32_t(*)[32]>(&d[0]));
                tc_wait_ld();
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const float4 e = delta[half * 8 + c];
                    const float* p = &v[half * 32 + 4 * c];
                    d[4 * c] = p[0] * (d[4 * c] - e.x);
                    d[4 * c + 1] = p[1] * (d[4 * c + 1] - e.y);
                    d[4 * c + 2] = p[2] * (d[4 * c + 2] - e.z);
                    d[4 * c + 3] = p[3] * (d[4 * c + 3] - e.w);
                }
                store_pairs<T>(t_dp + half * 16, d);
            }
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&bar->ds_full);
        }
        if (ok) ok = wait_all(&bar->all_done, 0, a, bar);
        if (ok) {
            tc_fence_after();
            const bool there = present(a, t, i), write = i < t.len;
            const long long row = (long long)t.start + (write ? i : 0);
            store_row<T>(t_s + 192, static_cast<T*>(a.io.dk.p) + row * a.io.dk.ld + hk * 64, write,
                         there ? a.scale : 0.f);
            store_row<T>(t_s + 128, static_cast<T*>(a.io.dv.p) + row * a.io.dv.ld + hk * 64, write, there ? 1.f : 0.f);
        }
    }
    close_frame(f, warp);
}

using Kernel = void (*)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, AttnArgs);

struct Maps {
    CUtensorMap q, k, v, dout;
};

bool map_rows(CUtensorMap* m, const AttnRows& r, int heads, const AttnArgs& a, bool bf16) {
    return make_tmap_rows(m, r.p, (uint64_t)heads * 64, (uint64_t)a.n_tokens, (uint64_t)r.ld, STEP, bf16) == CUDA_SUCCESS;
}

cudaError_t launch(Kernel kernel, unsigned heads, int smem, const Maps& m, const AttnArgs& a, cudaStream_t stream) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((unsigned)seq_tiles(a.n_tokens, a.n_seqs, ROWS), heads);
    kernel<<<grid, THREADS, smem, stream>>>(m.q, m.k, m.v, m.dout, a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_attention_fwd_tc(bool bf16, int n_heads, const AttnArgs& a, cudaStream_t stream) {
    Maps m;
    const int kv = n_heads / a.group;
    if (!map_rows(&m.q, a.io.q, n_heads, a, bf16) || !map_rows(&m.k, a.io.k, kv, a, bf16) ||
        !map_rows(&m.v, a.io.v, kv, a, bf16))
        return cudaErrorInvalidValue;
    m.dout = m.q;  // not used
    return launch(bf16 ? attention_fwd_tc_kernel<__nv_bfloat16> : attention_fwd_tc_kernel<__half>, n_heads, FWD_SMEM,
                  m, a, stream);
}

cudaError_t launch_attention_bwd_tc(bool bf16, int n_heads, int n_kv_heads, const AttnArgs& a, cudaStream_t stream) {
    Maps m;
    if (!map_rows(&m.q, a.io.q, n_heads, a, bf16) || !map_rows(&m.k, a.io.k, n_kv_heads, a, bf16) ||
        !map_rows(&m.v, a.io.v, n_kv_heads, a, bf16) || !map_rows(&m.dout, a.io.dout, n_heads, a, bf16))
        return cudaErrorInvalidValue;
    cudaError_t e = launch(bf16 ? attention_dq_tc_kernel<__nv_bfloat16> : attention_dq_tc_kernel<__half>, n_heads,
                           DQ_SMEM, m, a, stream);
    if (e == cudaSuccess)
        e = launch(bf16 ? attention_dkv_tc_kernel<__nv_bfloat16> : attention_dkv_tc_kernel<__half>, n_kv_heads,
                   DKV_SMEM, m, a, stream);
    return e;
}

}  // namespace laya
