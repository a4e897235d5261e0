// attention_op_tc.cu -- the attention operator on tcgen05: forward, dQ, and
// dK with dV (the formulas are in attention_op.cu).
//
// Two CTAs to an SM walk over the call's items, an item being 128 rows
// (queries, or keys for dK and dV) of one head, one row to a TMEM lane, which
// go through the other side in tiles of 64:
//
//   warps 0-7  the softmax's arithmetic, in two groups of four warps: thread t
//              of either owns row t, of which group g reads columns 32 g .. 32
//              g + 31 of the tile's scores from TMEM and writes P or dS back
//              as 16-bit pairs into the columns it has read. A lane's columns
//              of a group are its thread's alone, so that needs no barrier
//              among the threads, and the next product takes P or dS from
//              TMEM as its A operand. (In the forward each group has its own
//              maximum, sum and O over its half of the keys; they are joined
//              at the item's end.)
//   warp 8     finds the items and loads: TMA boxes of 64 rows x 128 bytes
//              into a ring of STAGES tile pairs. A box of the packed rows also
//              brings the rows of absent tokens and of the next sequence; in
//              tiles that have such rows the warp overwrites them with zeros
//              once the box has landed, while the next one is on its way,
//              before it hands the stage over. (The 128-row tile needs none
//              of that: its rows are the MMA's M index, and nothing crosses
//              from one to another.)
//   warp 9     owns TMEM and issues the MMAs.
//
// The next item is found and loaded while the present one is computed: at
// 175-180 tokens an item has three tiles, and finding it, setting up and the
// first loads took a third of a CTA's time when every item had its own.
//
// TMEM holds 256 columns a CTA: two buffers for scores, so that a tile's are
// there when the tile before has been dealt with, and the accumulators. With
// the registers (20 warps of 96) that allows two CTAs, four softmax warps to a
// sub-partition, and what bounds the kernels is the latency of these warps'
// dependent steps (TMEM load, ex2, pack, TMEM store, barrier) more than any
// unit: on one sequence of 8,192 tokens, 12 heads, the SFU is busy 64 % of the
// forward's time (512 cycles of ex2 for a 128 x 64 tile) and 51 % of the backward's,
// the tensor cores 32 and 45 %, and issue slots 54 % at most.
// There the forward takes 345 us (597 TFLOP/s) and the backward 800 (644 over
// the five products needed, 901 over the seven that it does); 64 sequences of
// 175-180 tokens 31 and 73 us, where an item has three tiles: of an item's 10,500
// cycles in dK/dV these take 6,000, waiting for the accumulators 800, storing them
// 2,500 and the next item's beginning 600 (forward: 6,200, of them 3,500 in tiles);
// 2 of 16,000 with a window of 64 (forward) 71 us. The mma.sync kernels took 3,619
// us for both passes of the first and 197 of the second.
//
// Measured and not kept: the groups on tiles of their own, three CTAs of one
// group, four ring stages, 1 KB of staging (no faster); an item's last sums
// followed at once by the next item's scores (111 -> 119 us for 64 x 175-180: the
// scores are there in time as it is, and every tile pays for keeping track of both
// items).
//
// TMEM is only overwritten by a product after the barrier that says its last
// reader is done: MMAs to different accumulators are not taken to be ordered.
// Every wait is bounded; a CTA that gives up records it, waits for its own
// copies and MMAs, frees TMEM and leaves.
#include <type_traits>

#include "attention_op.cuh"
#include "attention_op_loader.cuh"
#include "gemm.cuh"

namespace laya {
namespace {

template <typename C>
constexpr int smem_bytes() {
    return C::BIGS * BIG + STAGES * 2 * SMALL + 8 * STAGE_BYTES + C::EXTRA * 4 + C::PASSES * (int)sizeof(Bars) +
           (int)sizeof(Slots) + 1024;
}

// ------------------------------------------------------------------ items and loads

// Presence of 64 rows of the sequence, two a lane: read for a tile while the
// one before is dealt with, made bits of when its turn comes.
struct Presence {
    uint32_t v0, v1;
    __device__ __forceinline__ void read(const AttnArgs& a, const SeqTile& t, int row0, int lane) {
        const int i0 = row0 + lane, i1 = i0 + 32;
        v0 = i0 < t.len;
        v1 = i1 < t.len;
        if (a.mask) {
            if (v0) v0 = a.mask[t.start + i0];
            if (v1) v1 = a.mask[t.start + i1];
        }
    }
    __device__ __forceinline__ void bits(uint32_t (&b)[2]) const {
        b[0] = __ballot_sync(0xffffffffu, v0 != 0);
        b[1] = __ballot_sync(0xffffffffu, v1 != 0);
    }
};

// The loading warp's walk over the call's items: tile slot x of the call (see
// seq_tiles) for one head after the other. A CTA begins with item blockIdx.x
// and then takes every gridDim.x-th or, with a counter in global memory, the
// next that nobody has: sequences of different lengths make items of different
// cost (128 sequences of 1-512 tokens: dK and dV 214 us by turns, 187 by tickets).
struct Walk {
    const AttnArgs& a;
    int heads, lane;
    unsigned long long* tickets;
    unsigned long long ahead;  // the next candidate
    int x;                     // the candidate's slot
    int head;
    int pivot;  // key of entry lane * step: the search's first round
    int step;
    int end = -1;  // no slot from here on has a tile (-1: not looked up yet)
    SeqTile t;     // the item found
    bool found;

    // Finds the first item (in the forward, before the frame is open: the look
    // at the offsets passes while the other warps set the CTA up).
    __device__ __forceinline__ Walk(const AttnArgs& a_, int heads_, int lane_, bool mine, unsigned long long* tickets_)
        : a(a_), heads(heads_), lane(lane_), tickets(tickets_) {
        found = false;
        if (!mine) return;
        ahead = blockIdx.x;
        step = (a.n_seqs + 31) / 32;
        pivot = lane * step < a.n_seqs ? key(a.cu[lane * step], lane * step) : 0;
        next();
    }
    __device__ __forceinline__ static int key(int start, int s) { return max(start, 0) / ROWS + s; }
    __device__ __forceinline__ void next() {
        for (found = false; !found;) {
            const unsigned long long item = __shfl_sync(0xffffffffu, ahead, 0);
            x = (int)(item / heads);
            head = (int)(item - (unsigned long long)x * heads);
            if (x >= (end < 0 ? a.n_tokens / ROWS + a.n_seqs : end)) return;
            if (!tickets)
                ahead = item + gridDim.x;
            else if (lane == 0)
                ahead = atomicAdd(tickets, 1ull) + gridDim.x;  // not looked at before the item after this one
            t.len = 0;
            found = find();
            if (!found && t.len == 0 && end < 0) end = slots();
        }
    }
    // A table with room for more sequences than it holds ends in many that
    // start where the last one ends: the slots before those. (3 sequences of
    // 180 tokens in a table of 1,024, forward and backward: 107 us without it,
    // 29 with it; 26 in a table of 3.)
    __device__ __forceinline__ int slots() const {
        const int* cu = a.cu;
        const int last = min(max(cu[a.n_seqs], 0), a.n_tokens);
        const int used = warp_search(a.n_seqs, lane, [&](int i) { return (long long)cu[i]; }, (long long)last - 1) + 1;
        return last / ROWS + used;
    }
    // The whole table, by the loading warps of all CTAs of one kernel of a call.
    __device__ __forceinline__ void check() const {
        for (long long s = (long long)blockIdx.x * 32 + lane; s < a.n_seqs; s += (long long)gridDim.x * 32)
            check_table(a.cu, a.n_seqs, a.n_tokens, a.max_len, s, a.status);
    }
    // find_tile for slot x, with one look at the table for up to 1,024 sequences.
    __device__ __forceinline__ bool find() {
        const int n = a.n_seqs;
        if (n > 1024) return find_tile(a.cu, n, a.n_tokens, a.max_len, ROWS, x, lane, &t);
        const int c = __popc(__ballot_sync(0xffffffffu, lane * step < n && pivot <= x));
        if (c == 0) return false;
        const int lo = (c - 1) * step, m = min(step, n - lo);
        const int at = a.cu[min(lo + lane, n)];
        const int c1 = __popc(__ballot_sync(0xffffffffu, lane < m && key(at, lo + lane) <= x));
        if (c1 == 0) return false;
        const int s = lo + c1 - 1, start = __shfl_sync(0xffffffffu, at, c1 - 1);
        const int end = c1 < 32 ? __shfl_sync(0xffffffffu, at, c1 & 31) : a.cu[s + 1];
        if (!run_ok(start, end, a.n_tokens, a.max_len)) return false;
        const int tile = x - key(start, s);
        t = SeqTile{start, end - start, 0};
        if (tile < 0 || (long long)tile * ROWS >= t.len) return false;
        t.row0 = tile * ROWS;
        return true;
    }
};

// The k-th item, for every other warp: its slot, until it arrives on item_empty.
__device__ __forceinline__ bool next_item(const Frame& f, const AttnArgs& a, int k) {
    Bars* b = f.bar;
    return wait_one(&b->item_full[k & 1], (k >> 1) & 1, a.status, &b->abort) && f.slots->item[k & 1].n >= 0;
}

// The softmax warps' place in the score buffers and in the ring, from the
// number of tiles they have gone through, of all items.
struct Turn {
    unsigned tile = 0;
    __device__ __forceinline__ int buffer() const { return tile & 1; }
    __device__ __forceinline__ uint32_t own() const { return (tile >> 1) & 1; }  // parity of the buffer's barriers
    __device__ __forceinline__ int stage() const { return tile % STAGES; }
};

// ------------------------------------------------------------------ TMEM rows

__device__ __forceinline__ void load64(uint32_t taddr, float (&v)[64]) {
    tmem_ld32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
    tmem_ld32(taddr + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
    tc_wait_ld();
}
__device__ __forceinline__ void load32(uint32_t taddr, float (&v)[32]) {
    tmem_ld32(taddr, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
    tc_wait_ld();
}

// Two f32 operations an instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)),
          "l"(*reinterpret_cast<uint64_t*>(&c)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(d)
        : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// A warp's 32 rows of 32 accumulators, times f (a row's own; 0: zeros), to
// global memory by way of 2 KB of shared memory: 64 bytes to a row and 8 rows
// to an instruction instead of 16 bytes to each of 32. g is the first row's
// address; rows at `rows` and past it are not written.
template <typename T>
__device__ __forceinline__ void store_rows(uint8_t* stage, const float* v, float f, T* g, long long ld, int rows,
                                           int lane) {
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 4; c++) {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 x = mul2(make_float2(v[8 * c + 2 * e], v[8 * c + 2 * e + 1]), make_float2(f, f));
            u[e] = f == 0.f ? 0u : pack2<T>(x.x, x.y);  // whatever the accumulator holds
        }
        *reinterpret_cast<uint4*>(stage + lane * 64 + ((c ^ (lane >> 1 & 3)) << 4)) =
            make_uint4(u[0], u[1], u[2], u[3]);
    }
    __syncwarp();
    const int c = lane & 3, r0 = lane >> 2;  // r0 >> 1 & 3 is the same for r0 + 8 i
    const uint8_t* from = stage + r0 * 64 + ((c ^ (r0 >> 1 & 3)) << 4);
    T* to = g + r0 * ld + c * 8;
#pragma unroll
    for (int i = 0; i < 4; i++, to += 8 * ld) {
        const uint4 u = *reinterpret_cast<const uint4*>(from + i * 512);
        if (r0 + i * 8 < rows) *reinterpret_cast<uint4*>(to) = u;
    }
}

// v[i] = -inf where column col0 + i is not there or lies outside row's window.
__device__ __forceinline__ void mask_row(float (&v)[32], uint32_t bits, int window, int row, int col0) {
    if (bits != ~0u) {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = bits & 1u << i ? v[i] : -INFINITY;
    }
    if (window >= 0) {  // col0 + i - (row - window) in [0, 2 window], as one unsigned comparison
        const unsigned span = 2u * (unsigned)window, d = (unsigned)(col0 - row) + (unsigned)window;
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = d + i <= span ? v[i] : -INFINITY;
    }
}

// ------------------------------------------------------------------ MMAs

// One lane of the warp, chosen by the hardware. Code under it keeps the MMAs'
// operands in uniform registers; under `lane == 0` four MMAs and two commits
// took 530 cycles to issue instead of 180.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

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

// D (128 x 64) += P . B over N x 16 of B's rows; P: 16 rows' 16-bit pairs
// every `step` columns of TMEM.
template <typename T, int N>
__device__ __forceinline__ void mma_sum(uint32_t d, uint32_t p, int step, uint32_t b, bool accumulate) {
#pragma unroll
    for (int ks = 0; ks < N; ks++)
        tc_mma_f16_ts(d, p + step * ks, sw128_desc(b + ks * 2048), IDESC<T> | B_MN, accumulate || ks != 0);
}

// ------------------------------------------------------------------ CTA frame

template <typename C>
__device__ __forceinline__ Frame open_frame(uint8_t* raw, int warp) {
    Frame f;
    f.big = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    f.ring = f.big + C::BIGS * BIG;
    f.stage = f.ring + STAGES * 2 * SMALL;
    f.extra = reinterpret_cast<float*>(f.stage + 8 * STAGE_BYTES);
    f.bar = reinterpret_cast<Bars*>(f.extra + C::EXTRA);
    f.slots = reinterpret_cast<Slots*>(f.bar + C::PASSES);
    f.stage += (warp & 7) * STAGE_BYTES;
    if (threadIdx.x == 0) {
        for (Bars* b = f.bar; b < f.bar + C::PASSES; b++) {
            for (int s = 0; s < STAGES; s++) {
                mbar_init(&b->full[s], 33);
                mbar_init(&b->empty[s], 1);
                mbar_init(&b->landed[s], 1);
            }
            mbar_init(&b->big_full, 1);
            mbar_init(&b->big_empty, 1);
            for (int s = 0; s < 2; s++) {
                mbar_init(&b->item_full[s], 32);
                mbar_init(&b->item_empty[s], SOFTMAX + 1);
                mbar_init(&b->s_full[s], 2);  // the product, and the MMA lane on what the stage holds besides
                mbar_init(&b->dp_full[s], 1);
                mbar_init(&b->s_read[s], SOFTMAX);
                mbar_init(&b->p_full[s], SOFTMAX);
                mbar_init(&b->done[s], 1);
                mbar_init(&b->acc_full[s], 1);
                mbar_init(&b->acc_free[s], SOFTMAX);
            }
            mbar_init(&b->sync, SOFTMAX);
            mbar_init(&b->drained, 1);
            b->abort = 0;
        }
        fence_barrier_init();
        fence_proxy_async();
    }
    if (warp == MMA) {
        tmem_alloc(&f.bar->tmem, COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    f.tmem = f.bar->tmem;
    return f;
}

template <typename C>
__device__ __forceinline__ void close_frame(const Frame& f, int warp) {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == MMA) tmem_dealloc(f.tmem, COLS);
}

// From one pass to the next: its copies and MMAs are complete, and everyone is
// done with shared memory and TMEM. False in a CTA that gave up.
__device__ __forceinline__ bool next_pass(Frame& f) {
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*(volatile int*)&f.bar->abort) return false;
    f.bar++;
    return true;
}

// The MMA lane's waits.
struct Waits {
    int* err;
    int* abort;
    __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t parity) const {
        const bool ok = wait_one(bar, parity, err, abort);
        tc_fence_after();
        return ok;
    }
};

// Warp-wide wait of the softmax warps.
__device__ __forceinline__ bool wait_all(uint64_t* bar, uint32_t parity, const AttnArgs& a, Bars* b) {
    return __all_sync(0xffffffffu, wait_one(bar, parity, a.status, &b->abort));
}

// ------------------------------------------------------------------ forward
// TMEM: S at columns 0, 64 (P over it, a group's 16 columns at the start of its
// 32); O of group 0, 1 at 128, 192. extra: maximum and sum of the rows of either
// group, of two items in turn.
using Fwd = Shape<1, 8 * ROWS>;

template <typename T, typename C>
__global__ void __launch_bounds__(THREADS, CTAS)
    attention_fwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                            const __grid_constant__ CUtensorMap mv, const AttnArgs a, int heads) {
    extern __shared__ uint8_t raw[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == LOADER * 32) {
        prefetch_tmap(&mq);
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
    }
    Walk walk(a, heads, lane, warp == LOADER, nullptr);
    const Frame f = open_frame<C>(raw, warp);
    Bars* bar = f.bar;

    if (warp == LOADER) {
        Loader<C> ld{f, a, lane};
        bool ok = true;
        while (walk.found && ok) {
            const SeqTile t = walk.t;
            const int h = walk.head;
            int kt0, kt1;
            visible_tiles(a, t, ROWS, STEP, &kt0, &kt1);
            Presence rows;
            rows.read(a, t, kt0 * STEP, lane);
            ok = ld.item(Item{t.start, t.len, t.row0, h, kt0, kt1 - kt0}, &mq, nullptr);
            for (int j = kt0; j < kt1 && ok; j++) {
                uint32_t bits[2];
                rows.bits(bits);
                if (j + 1 < kt1) rows.read(a, t, (j + 1) * STEP, lane);
                ok = ld.room();
                if (!ok) break;
                if (lane < 2) f.slots->bits[ld.issued % STAGES][lane] = lane ? bits[1] : bits[0];
                ld.tile(&mk, &mv, h / a.group * 64, t.start + j * STEP, bits);
            }
            walk.next();  // while the last boxes are on their way
            ld.fill();
        }
        const int big = ld.items;
        if (ok) ld.item(Item{0, 0, 0, 0, 0, -1}, &mq, nullptr);
        ld.finish(big);
        walk.check();
    } else if (warp == MMA) {
        if (elect_one()) {
            const uint32_t q = smem_u32(f.big), kv = smem_u32(f.ring);
            const Waits wait{a.status, &bar->abort};
            int c = 0;  // tiles of the items before
            auto scores = [&](int j) {
                if (!wait(&bar->full[j % STAGES], (j / STAGES) & 1) || (j > 1 && !wait(&bar->done[j & 1], ((j >> 1) - 1) & 1)))
                    return false;
                mma_rows<T>(f.tmem + (j & 1) * 64, q, kv + 2 * (j % STAGES) * SMALL);
                tc_commit(&bar->s_full[j & 1]);
                mbar_arrive(&bar->s_full[j & 1]);
                return true;
            };
            // S runs two tiles ahead of P V: of the tile before P V's buffer is free
            for (int k = 0; next_item(f, a, k); k++) {
                const int n = f.slots->item[k & 1].n;
                mbar_arrive(&bar->item_empty[k & 1]);
                if (!wait(&bar->big_full, k & 1) || !scores(c) || (n > 1 && !scores(c + 1))) break;
                if (n <= 2) tc_commit(&bar->big_empty);
                int i = 0;
                for (; i < n; i++) {
                    const int j = c + i, s = j % STAGES;
                    const uint32_t p = f.tmem + (j & 1) * 64, v = kv + (2 * s + 1) * SMALL;
                    if (!wait(&bar->p_full[j & 1], (j >> 1) & 1)) break;
                    if (i == 0 && k > 0 && !wait(&bar->acc_free[0], (k - 1) & 1)) break;
                    mma_sum<T, 2>(f.tmem + 128, p, 8, v, i > 0);
                    mma_sum<T, 2>(f.tmem + 192, p + 32, 8, v + 2 * 2048, i > 0);
                    tc_commit(&bar->empty[s]);
                    tc_commit(&bar->done[j & 1]);
                    if (i + 2 < n) {
                        if (!scores(j + 2)) break;
                        if (i + 3 == n) tc_commit(&bar->big_empty);
                    }
                }
                if (i < n) break;
                tc_commit(&bar->acc_full[0]);
                c += n;
            }
            tc_commit(&bar->drained);
            drain(&bar->drained, 0, a.status, &bar->abort);
        }
        __syncwarp();
    } else {
        const int g = warp >> 2, r = threadIdx.x & (ROWS - 1);
        const uint32_t lanes = f.tmem + ((uint32_t)((warp & 3) * 32) << 16), t_o = lanes + 128 + g * 64;
        const float sl2 = a.scale * LOG2E;
        constexpr float RESCALE = 8.0f;  // exponent growth that moves the reference point
        Turn turn;
        bool ok = true;
        for (int k = 0; ok; k++) {
            if (!__all_sync(0xffffffffu, next_item(f, a, k))) break;
            const Item& it = f.slots->item[k & 1];
            const int n = it.n, row0 = it.row0;
            int col0 = it.t0 * STEP + g * 32;
            float m = -INFINITY, l = 0.f;
            for (int j = 0; j < n; j++, col0 += STEP, turn.tile++) {
                const uint32_t t_s = lanes + turn.buffer() * 64 + g * 32;
                ok = wait_all(&bar->s_full[turn.buffer()], turn.own(), a, bar);
                if (!ok) break;
                tc_fence_after();
                float v[32];
                load32(t_s, v);
                const uint32_t bits = f.slots->bits[turn.stage()][g];
                if (bits != ~0u || edge(a.window, row0, ROWS, col0, 32)) mask_row(v, bits, a.window, row0 + r, col0);
                float mx[4];
#pragma unroll
                for (int e = 0; e < 4; e++) mx[e] = v[e];
#pragma unroll
                for (int e = 4; e < 28; e += 8)
#pragma unroll
                    for (int x = 0; x < 4; x++) mx[x] = max3(mx[x], v[e + x], v[e + 4 + x]);
                const float top = fmaxf(max3(max3(mx[0], v[28], v[29]), mx[1], mx[2]), max3(mx[3], v[30], v[31]));
                // The reference point moves when the maximum has grown by more
                // than 2^8 (p stays below 2^8 otherwise): then O and l shrink.
                float alpha = 1.f;
                const bool move = j == 0 || (top - m) * sl2 > RESCALE;
                if (move) {
                    alpha = m == -INFINITY ? 0.f : ex2_approx((m - top) * sl2);
                    m = top;
                    l *= alpha;
                }
                if (j > 0 && __any_sync(0xffffffffu, move)) {
                    // once P V of the tile before is complete, O is at rest
                    ok = wait_all(&bar->done[turn.buffer() ^ 1], ((turn.tile - 1) >> 1) & 1, a, bar);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int e = 0; e < 64; e += 16) {
                        uint32_t o[16];
                        tmem_ld16(t_o + e, o);
                        tc_wait_ld();
#pragma unroll
                        for (int x = 0; x < 16; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                        tmem_st16(t_o + e, o);
                    }
                }
                const float u = m == -INFINITY ? 0.f : m * sl2;
                float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t p[16];
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const float2 y = fma2(make_float2(v[2 * x], v[2 * x + 1]), make_float2(sl2, sl2), make_float2(-u, -u));
                    const float2 q = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                    sum[x & 1] = add2(sum[x & 1], q);
                    p[x] = pack2<T>(q.x, q.y);
                }
                tmem_st16(t_s, p);
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&bar->p_full[turn.buffer()]);
            }
            // The groups' halves of the row are joined: each takes 32 columns
            // of both (the two threads of a row share its TMEM lane).
            float2* ml = reinterpret_cast<float2*>(f.extra) + (k & 1) * 2 * ROWS + r;
            if (ok) {
                ml[g * ROWS] = make_float2(m, l);
                mbar_arrive(&bar->sync);
            }
            ok = ok && wait_all(&bar->sync, k & 1, a, bar) && wait_all(&bar->acc_full[0], k & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
            float o[32], o1[32];
            tmem_ld32(lanes + 128 + g * 64 + g * 32, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
            tmem_ld32(lanes + 128 + (1 - g) * 64 + g * 32, *reinterpret_cast<uint32_t(*)[32]>(&o1[0]));
            tc_wait_ld();
            tc_fence_before();
            mbar_arrive(&bar->acc_free[0]);
            const float2 other = ml[(1 - g) * ROWS];
            const float top = fmaxf(m, other.x);
            const float u = top == -INFINITY ? 0.f : top;
            const float f0 = ex2_approx((m - u) * sl2), f1 = ex2_approx((other.x - u) * sl2);
            const float sum = l * f0 + other.y * f1;
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const float2 x = fma2(make_float2(o[e], o[e + 1]), make_float2(f0, f0),
                                      mul2(make_float2(o1[e], o1[e + 1]), make_float2(f1, f1)));
                o[e] = x.x;
                o[e + 1] = x.y;
            }
            const SeqTile t{it.start, it.len, row0};
            const bool there = present(a, t, row0 + r);
            const int row = row0 + (warp & 3) * 32;  // the warp's first
            store_rows<T>(f.stage, o, there ? rcp_approx(sum) : 0.f,
                          static_cast<T*>(a.io.out.p) + ((long long)t.start + row) * a.io.out.ld + it.head * 64 + g * 32,
                          a.io.out.ld, t.len - row, lane);
            if (a.io.lse && g == 0 && row0 + r < t.len)
                a.io.lse[(long long)it.head * a.n_tokens + t.start + row0 + r] =
                    there ? top * a.scale + logf(sum) : -INFINITY;
            mbar_arrive(&bar->item_empty[k & 1]);
        }
    }
    close_frame<C>(f, warp);
}

// The MMA lane of either backward kernel: S = A0 . R0^T, dP = A1 . R1^T (A:
// 128-row tiles, R: the ring's), then the sums over the tile's rows.
template <typename T, int ACCS, typename Sum>
__device__ __forceinline__ void backward_mmas(const Frame& f, const AttnArgs& a, Sum sums) {
    Bars* bar = f.bar;
    const uint32_t big0 = smem_u32(f.big), big1 = big0 + BIG, ring = smem_u32(f.ring);
    const Waits wait{a.status, &bar->abort};
    int c = 0;  // tiles of the items before
    auto scores = [&](int j) {
        if (!wait(&bar->full[j % STAGES], (j / STAGES) & 1) || (j > 1 && !wait(&bar->done[j & 1], ((j >> 1) - 1) & 1)))
            return false;
        mma_rows<T>(f.tmem + (j & 1) * 64, big0, ring + 2 * (j % STAGES) * SMALL);
        tc_commit(&bar->s_full[j & 1]);
        mbar_arrive(&bar->s_full[j & 1]);
        return true;
    };
    auto dp = [&](int j) {
        if (!wait(&bar->s_read[j & 1], (j >> 1) & 1)) return false;
        mma_rows<T>(f.tmem + (j & 1) * 64, big1, ring + (2 * (j % STAGES) + 1) * SMALL);
        tc_commit(&bar->dp_full[j & 1]);
        return true;
    };
    // In the order in which the softmax warps come to them: the sums of a
    // tile, the next one's dP (its scores are read right after), the scores of
    // the tile after that. An accumulator gets its tiles in their order.
    for (int k = 0; next_item(f, a, k); k++) {
        const int n = f.slots->item[k & 1].n, acc = k % ACCS;
        mbar_arrive(&bar->item_empty[k & 1]);
        if (!wait(&bar->big_full, k & 1) || !scores(c) || (n > 1 && !scores(c + 1)) || !dp(c)) break;
        if (n == 1) tc_commit(&bar->big_empty);
        int i = 0;
        for (; i < n; i++) {
            const int j = c + i;
            if (!wait(&bar->p_full[j & 1], (j >> 1) & 1)) break;
            if (i == 0 && k >= ACCS && !wait(&bar->acc_free[acc], (k / ACCS - 1) & 1)) break;
            sums(f.tmem + (j & 1) * 64, ring + 2 * (j % STAGES) * SMALL, acc, i > 0);
            tc_commit(&bar->empty[j % STAGES]);
            tc_commit(&bar->done[j & 1]);
            if (i + 1 < n) {
                if (!dp(j + 1)) break;
                if (i + 2 == n) tc_commit(&bar->big_empty);
            }
            if (i + 2 < n && !scores(j + 2)) break;
        }
        if (i < n) break;
        tc_commit(&bar->acc_full[acc]);
        c += n;
    }
    tc_commit(&bar->drained);
    drain(&bar->drained, 0, a.status, &bar->abort);
}

// ------------------------------------------------------------------ dQ
// TMEM: S at columns 0, 64 (dP over it, dS over that, 8 columns of every 16);
// dQ at 128, the next item's at 192. extra: -lse * log2 e and -delta of the rows
// of two items in turn.
template <typename T, typename C>
__device__ __forceinline__ void dq_pass(const Frame& f, const CUtensorMap& mq, const CUtensorMap& mk,
                                        const CUtensorMap& mv, const CUtensorMap& mdo, const AttnArgs& a, int heads) {
    static_assert(C::EXTRA >= 4 * ROWS, "the rows' statistics");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Walk walk(a, heads, lane, warp == LOADER, a.io.tickets);
    Bars* bar = f.bar;

    if (warp == LOADER) {
        Loader<C> ld{f, a, lane};
        bool ok = true;
        while (walk.found && ok) {
            const SeqTile t = walk.t;
            const int h = walk.head;
            int kt0, kt1;
            visible_tiles(a, t, ROWS, STEP, &kt0, &kt1);
            Presence rows;
            rows.read(a, t, kt0 * STEP, lane);
            // the rows' statistics (absent rows are not stored: 0 will do)
            float* stat = f.extra + (ld.items & 1) * 2 * ROWS + lane;
            float lse[4], delta[4];
            const float* deltas = t.len <= SHORT ? a.io.delta_short : a.io.delta;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const int i = t.row0 + x * 32 + lane;
                const bool there = present(a, t, i);
                const long long at = (long long)h * a.n_tokens + t.start + i;
                lse[x] = there ? a.io.lse[at] : 0.f;
                delta[x] = there ? deltas[at] : 0.f;
            }
            ok = ld.slot();
            if (!ok) break;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                stat[x * 32] = -LOG2E * lse[x];
                stat[ROWS + x * 32] = -delta[x];
            }
            ok = ld.item(Item{t.start, t.len, t.row0, h, kt0, kt1 - kt0}, &mq, &mdo);
            for (int j = kt0; j < kt1 && ok; j++) {
                uint32_t bits[2];
                rows.bits(bits);
                if (j + 1 < kt1) rows.read(a, t, (j + 1) * STEP, lane);
                ok = ld.room();
                if (!ok) break;
                if (lane < 2) f.slots->bits[ld.issued % STAGES][lane] = lane ? bits[1] : bits[0];
                ld.tile(&mk, &mv, h / a.group * 64, t.start + j * STEP, bits);
            }
            walk.next();  // while the last boxes are on their way
            ld.fill();
        }
        const int big = ld.items;
        if (ok) ld.item(Item{0, 0, 0, 0, 0, -1}, &mq, &mdo);
        ld.finish(big);
    } else if (warp == MMA) {
        if (elect_one())
            backward_mmas<T, 2>(f, a, [&](uint32_t p, uint32_t kv, int acc, bool more) {
                mma_sum<T, 4>(f.tmem + 128 + acc * 64, p, 16, kv, more);
            });
        __syncwarp();
    } else {
        const int g = warp >> 2, r = threadIdx.x & (ROWS - 1);
        const uint32_t lanes = f.tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const float sl2 = a.scale * LOG2E;
        Turn turn;
        bool ok = true;
        for (int k = 0; ok; k++) {
            if (!__all_sync(0xffffffffu, next_item(f, a, k))) break;
            const Item& it = f.slots->item[k & 1];
            const int n = it.n, i = it.row0 + r;  // query
            int col0 = it.t0 * STEP + g * 32;
            const SeqTile t{it.start, it.len, it.row0};
            const bool there = present(a, t, i);
            const float* stat = f.extra + (k & 1) * 2 * ROWS + r;
            const float e = stat[0], delta = stat[ROWS];
            for (int j = 0; j < n; j++, col0 += STEP, turn.tile++) {
                const uint32_t t_s = lanes + turn.buffer() * 64 + g * 32;
                ok = wait_all(&bar->s_full[turn.buffer()], turn.own(), a, bar);
                if (!ok) break;
                tc_fence_after();
                float v[32];
                load32(t_s, v);
                tc_fence_before();
                mbar_arrive(&bar->s_read[turn.buffer()]);
                const uint32_t bits = f.slots->bits[turn.stage()][g];
                if (bits != ~0u || edge(a.window, i - r, ROWS, col0, 32)) mask_row(v, bits, a.window, i, col0);
#pragma unroll
                for (int x = 0; x < 32; x += 2) {
                    const float2 y = fma2(make_float2(v[x], v[x + 1]), make_float2(sl2, sl2), make_float2(e, e));
                    v[x] = ex2_approx(y.x);
                    v[x + 1] = ex2_approx(y.y);
                }
                ok = wait_all(&bar->dp_full[turn.buffer()], turn.own(), a, bar);
                if (!ok) break;
                tc_fence_after();
                float d[32];
                load32(t_s, d);
#pragma unroll
                for (int x = 0; x < 32; x += 16) {
                    uint32_t ds[8];
#pragma unroll
                    for (int z = 0; z < 8; z++) {
                        const int c = x + 2 * z;
                        const float2 y = mul2(make_float2(v[c], v[c + 1]),
                                              add2(make_float2(d[c], d[c + 1]), make_float2(delta, delta)));
                        ds[z] = pack2<T>(y.x, y.y);
                    }
                    tmem_st8(t_s + x, ds);
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&bar->p_full[turn.buffer()]);
            }
            if (ok) ok = wait_all(&bar->acc_full[k & 1], (k >> 1) & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
            float d[32];
            load32(lanes + 128 + (k & 1) * 64 + g * 32, d);
            tc_fence_before();
            mbar_arrive(&bar->acc_free[k & 1]);
            const int row = it.row0 + (warp & 3) * 32;  // the warp's first
            store_rows<T>(f.stage, d, there ? a.scale : 0.f,
                          static_cast<T*>(a.io.dq.p) + ((long long)it.start + row) * a.io.dq.ld + it.head * 64 + g * 32,
                          a.io.dq.ld, it.len - row, lane);
            mbar_arrive(&bar->item_empty[k & 1]);
        }
    }
}

// ------------------------------------------------------------------ dK, dV
// TMEM: S^T at columns 0, 64 (dP^T over it, P^T and dS^T over
// that, 8 columns of each in turn); dV at 128; dK at 192. extra: -lse * log2 e
// and -delta of each stage's queries.
template <typename T, typename C>
__device__ __forceinline__ void dkv_pass(const Frame& f, const CUtensorMap& mq, const CUtensorMap& mk,
                                         const CUtensorMap& mv, const CUtensorMap& mdo, const AttnArgs& a, int heads) {
    static_assert(C::EXTRA >= 2 * STAGES * STEP, "the stages' statistics");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Walk walk(a, heads, lane, warp == LOADER, a.io.tickets + 1);
    Bars* bar = f.bar;

    if (warp == LOADER) {
        Loader<C> ld{f, a, lane};
        bool ok = true;
        while (walk.found && ok) {
            const SeqTile t = walk.t;
            const int hk = walk.head;
            int qt0, qt1;
            visible_tiles(a, t, ROWS, STEP, &qt0, &qt1);
            // the query tiles of every head of the group
            const int n = (qt1 - qt0) * a.group;
            Presence rows;
            rows.read(a, t, qt0 * STEP, lane);
            ok = ld.item(Item{t.start, t.len, t.row0, hk, qt0, n}, &mk, &mv);
            const float* deltas = t.len <= SHORT ? a.io.delta_short : a.io.delta;
            int h = hk * a.group, q = qt0;
            for (int j = 0; j < n && ok; j++) {
                uint32_t bits[2];
                rows.bits(bits);
                const int row0 = q * STEP;
                // statistics of rows lane and lane + 32 (0 for rows that are not there: q = dO = 0)
                const long long at = (long long)h * a.n_tokens + t.start + row0 + lane;
                const bool b0 = bits[0] >> lane & 1, b1 = bits[1] >> lane & 1;
                const float l0 = b0 ? a.io.lse[at] : 0.f, l1 = b1 ? a.io.lse[at + 32] : 0.f;
                const float d0 = b0 ? deltas[at] : 0.f, d1 = b1 ? deltas[at + 32] : 0.f;
                const int head = h;
                if (++q == qt1) {
                    q = qt0;
                    h++;
                }
                if (j + 1 < n) rows.read(a, t, q * STEP, lane);
                ok = ld.room();
                if (!ok) break;
                const int s = ld.issued % STAGES;
                float* stat = f.extra + s * 2 * STEP + lane;
                stat[0] = -LOG2E * l0;
                stat[32] = -LOG2E * l1;
                stat[STEP] = -d0;
                stat[STEP + 32] = -d1;
                ld.tile(&mq, &mdo, head * 64, t.start + row0, bits);
            }
            walk.next();  // while the last boxes are on their way
            ld.fill();
        }
        const int big = ld.items;
        if (ok) ld.item(Item{0, 0, 0, 0, 0, -1}, &mk, &mv);
        ld.finish(big);
        walk.check();
    } else if (warp == MMA) {
        if (elect_one())
            backward_mmas<T, 1>(f, a, [&](uint32_t p, uint32_t qd, int, bool more) {
                mma_sum<T, 4>(f.tmem + 128, p, 16, qd + SMALL, more);
                mma_sum<T, 4>(f.tmem + 192, p + 8, 16, qd, more);
            });
        __syncwarp();
    } else {
        const int g = warp >> 2, r = threadIdx.x & (ROWS - 1);
        const uint32_t lanes = f.tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const float sl2 = a.scale * LOG2E;
        Turn turn;
        bool ok = true;
        for (int k = 0; ok; k++) {
            if (!__all_sync(0xffffffffu, next_item(f, a, k))) break;
            const Item& it = f.slots->item[k & 1];
            const int n = it.n, i = it.row0 + r;  // key
            for (int j = 0; j < n; j++, turn.tile++) {
                const uint32_t t_s = lanes + turn.buffer() * 64 + g * 32;
                ok = wait_all(&bar->s_full[turn.buffer()], turn.own(), a, bar);
                if (!ok) break;
                tc_fence_after();
                float v[32];
                load32(t_s, v);
                tc_fence_before();
                mbar_arrive(&bar->s_read[turn.buffer()]);
                if (a.window >= 0) {
                    const int col0 = (it.t0 + j % (n / a.group)) * STEP + g * 32;
                    if (edge(a.window, col0, 32, i - r, ROWS)) mask_row(v, ~0u, a.window, i, col0);
                }
                const float4* lse = reinterpret_cast<const float4*>(f.extra + turn.stage() * 2 * STEP + g * 32);
                const float4* delta = lse + STEP / 4;
#pragma unroll
                for (int x = 0; x < 8; x++) {
                    const float4 e = lse[x];
                    const float2 y = fma2(make_float2(v[4 * x], v[4 * x + 1]), make_float2(sl2, sl2), make_float2(e.x, e.y));
                    const float2 z =
                        fma2(make_float2(v[4 * x + 2], v[4 * x + 3]), make_float2(sl2, sl2), make_float2(e.z, e.w));
                    v[4 * x] = ex2_approx(y.x);
                    v[4 * x + 1] = ex2_approx(y.y);
                    v[4 * x + 2] = ex2_approx(z.x);
                    v[4 * x + 3] = ex2_approx(z.y);
                }
                ok = wait_all(&bar->dp_full[turn.buffer()], turn.own(), a, bar);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < 32; x += 16) {
                    uint32_t d[16], w[16];  // 16 of dP, then 16 of P and 16 of dS in pairs
                    tmem_ld16(t_s + x, d);
                    tc_wait_ld();
#pragma unroll
                    for (int z = 0; z < 4; z++) {
                        const float4 e = delta[x / 4 + z];
                        const float2 p0 = make_float2(v[x + 4 * z], v[x + 4 * z + 1]);
                        const float2 p1 = make_float2(v[x + 4 * z + 2], v[x + 4 * z + 3]);
                        const float2 s0 = mul2(p0, add2(make_float2(__uint_as_float(d[4 * z]), __uint_as_float(d[4 * z + 1])),
                                                        make_float2(e.x, e.y)));
                        const float2 s1 =
                            mul2(p1, add2(make_float2(__uint_as_float(d[4 * z + 2]), __uint_as_float(d[4 * z + 3])),
                                          make_float2(e.z, e.w)));
                        w[2 * z] = pack2<T>(p0.x, p0.y);
                        w[2 * z + 1] = pack2<T>(p1.x, p1.y);
                        w[8 + 2 * z] = pack2<T>(s0.x, s0.y);
                        w[9 + 2 * z] = pack2<T>(s1.x, s1.y);
                    }
                    tmem_st16(t_s + x, w);
                }
                tc_wait_st();
                tc_fence_before();
                mbar_arrive(&bar->p_full[turn.buffer()]);
            }
            if (ok) ok = wait_all(&bar->acc_full[0], k & 1, a, bar);
            if (!ok) break;
            tc_fence_after();
            // group 0 stores dV, group 1 dK
            float d[64];
            load64(lanes + 128 + g * 64, d);
            tc_fence_before();
            mbar_arrive(&bar->acc_free[0]);
            const SeqTile t{it.start, it.len, it.row0};
            const float by = !present(a, t, i) ? 0.f : g ? a.scale : 1.f;
            const AttnRows& out = g ? a.io.dk : a.io.dv;
            const int row = it.row0 + (warp & 3) * 32;  // the warp's first
            T* to = static_cast<T*>(out.p) + ((long long)it.start + row) * out.ld + it.head * 64;
            store_rows<T>(f.stage, d, by, to, out.ld, it.len - row, lane);
            store_rows<T>(f.stage, d + 32, by, to + 32, out.ld, it.len - row, lane);
            mbar_arrive(&bar->item_empty[k & 1]);
        }
    }
}

// ------------------------------------------------------------------ backward
// Both passes in one launch, whose CTAs go from dK/dV's items to dQ's as they come
// free: the passes use nothing of one another, and all that they share (delta, the
// counters) is complete when the CTA's wait returns. The longer items go first: a
// key head's item goes through the queries of its whole group. (As two launches,
// the second one's CTAs in the places of the first's, dQ first unless heads are
// shared: 64 x 175-180 tokens, 12 heads 76 us instead of 72, 128 x 1-512, 12 heads
// over 4 288 instead of 284, one sequence of 8,192 760 instead of 800; but there the
// second launch has no wait of its own behind which delta is known to be complete.)
using Bwd = Shape<2, 4 * ROWS, 2>;

template <typename T, typename C>
__global__ void __launch_bounds__(THREADS, CTAS)
    attention_bwd_tc_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                            const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mdo,
                            const AttnArgs a, int heads, int kv_heads) {
    extern __shared__ uint8_t raw[];
    const int warp = threadIdx.x >> 5;
    if (threadIdx.x == LOADER * 32) {
        prefetch_tmap(&mq);
        prefetch_tmap(&mk);
        prefetch_tmap(&mv);
        prefetch_tmap(&mdo);
    }
    Frame f = open_frame<C>(raw, warp);
    griddep_wait();
    dkv_pass<T, C>(f, mq, mk, mv, mdo, a, kv_heads);
    if (next_pass(f)) dq_pass<T, C>(f, mq, mk, mv, mdo, a, heads);
    close_frame<C>(f, warp);
}


struct Maps {
    CUtensorMap q, k, v, dout;
};

bool map_rows(CUtensorMap* m, const AttnRows& r, int heads, const AttnArgs& a, bool bf16) {
    return make_tmap_rows(m, r.p, (uint64_t)heads * 64, (uint64_t)a.n_tokens, (uint64_t)r.ld, STEP, bf16) == CUDA_SUCCESS;
}

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0)
        return 148;
    return sms;
}

// CTAs to a kernel over `heads` heads.
unsigned ctas(const AttnArgs& a, int heads) {
    const long long work = seq_tiles(a.n_tokens, a.n_seqs, ROWS) * heads, most = (long long)CTAS * sm_count();
    return (unsigned)(work < most ? work : most);
}

template <typename C, typename Kernel>
cudaError_t allow_smem(Kernel kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<C>());
}

template <typename T>
cudaError_t forward(const Maps& m, const AttnArgs& a, int heads, cudaStream_t stream) {
    const auto kernel = attention_fwd_tc_kernel<T, Fwd>;
    const cudaError_t e = allow_smem<Fwd>(kernel);
    if (e != cudaSuccess) return e;
    kernel<<<ctas(a, heads), THREADS, smem_bytes<Fwd>(), stream>>>(m.q, m.k, m.v, a, heads);
    return cudaGetLastError();
}

template <typename T>
cudaError_t backward(const Maps& m, const AttnArgs& a, int heads, int kv_heads, cudaStream_t stream) {
    const auto kernel = attention_bwd_tc_kernel<T, Bwd>;
    cudaError_t e = allow_smem<Bwd>(kernel);
    if (e != cudaSuccess) return e;
    e = launch_attention_delta(std::is_same<T, __nv_bfloat16>::value, heads, a, stream);
    if (e != cudaSuccess) return e;
    return launch_k(kernel, dim3(ctas(a, heads)), THREADS, smem_bytes<Bwd>(), stream, m.q, m.k, m.v, m.dout, a, heads,
                    kv_heads);
}

}  // namespace

cudaError_t launch_attention_fwd_tc(bool bf16, int n_heads, const AttnArgs& a, cudaStream_t stream) {
    Maps m;
    const int kv = n_heads / a.group;
    if (!map_rows(&m.q, a.io.q, n_heads, a, bf16) || !map_rows(&m.k, a.io.k, kv, a, bf16) ||
        !map_rows(&m.v, a.io.v, kv, a, bf16))
        return cudaErrorInvalidValue;
    return bf16 ? forward<__nv_bfloat16>(m, a, n_heads, stream) : forward<__half>(m, a, n_heads, stream);
}

cudaError_t launch_attention_bwd_tc(bool bf16, int n_heads, int n_kv_heads, const AttnArgs& a, cudaStream_t stream) {
    Maps m;
    if (!map_rows(&m.q, a.io.q, n_heads, a, bf16) || !map_rows(&m.k, a.io.k, n_kv_heads, a, bf16) ||
        !map_rows(&m.v, a.io.v, n_kv_heads, a, bf16) || !map_rows(&m.dout, a.io.dout, n_heads, a, bf16))
        return cudaErrorInvalidValue;
    return bf16 ? backward<__nv_bfloat16>(m, a, n_heads, n_kv_heads, stream)
                : backward<__half>(m, a, n_heads, n_kv_heads, stream);
}

}  // namespace laya
