// attention_op_loader.cuh -- the barriers of the tcgen05 attention operator's
// CTAs, their bounded waits, and the loading warp's way of filling the ring.
//
// Included behind common.cuh's mbarrier and TMA operations. It has no includes of
// its own, so that a host program can compile it behind stand-ins for these and
// watch what the loading warp leaves behind when a wait runs out.
#pragma once

namespace laya {
namespace {

constexpr int ROWS = 128;  // rows per item, one TMEM lane each
constexpr int STEP = 64;   // rows of the other side per tile
constexpr int BIG = ROWS * 64 * 2;    // 16 KB
constexpr int SMALL = STEP * 64 * 2;  // 8 KB

constexpr int STAGES = 3;
constexpr int SOFTMAX = 256;  // threads of the two groups
constexpr int LOADER = 8, MMA = 9, THREADS = SOFTMAX + 64;
constexpr int CTAS = 2;  // on an SM
constexpr uint32_t COLS = 256;

constexpr int STAGE_BYTES = 2048;  // staging for a softmax warp's stores

// Of one kernel: 128-row tiles, floats besides, passes over the call's items (each
// has barriers of its own).
template <int BIGS_, int EXTRA_, int PASSES_ = 1>
struct Shape {
    static constexpr int BIGS = BIGS_, EXTRA = EXTRA_, PASSES = PASSES_;
};

// What the loading warp found; n < 0: there is no further item.
struct Item {
    int start, len, row0;  // the sequence and the item's first row in it
    int head;              // of the 128 rows
    int t0, n;             // its tiles
};

struct Bars {
    uint64_t full[STAGES], empty[STAGES], landed[STAGES];
    uint64_t item_full[2], item_empty[2];
    uint64_t big_full, big_empty;
    // one of each for each score buffer
    uint64_t s_full[2], dp_full[2];  // products to read
    uint64_t s_read[2];              // S has been read: its columns may take dP
    uint64_t p_full[2];              // P (and dS) written: operands of the next products
    uint64_t done[2];                // which are complete: the columns may take S again
    uint64_t acc_full[2], acc_free[2];  // an item's accumulators
    uint64_t sync;                   // among the softmax threads
    uint64_t drained;
    uint32_t tmem;
    int abort;
};

struct Slots {
    uint32_t bits[STAGES][2];  // presence of a stage's rows (keys)
    Item item[2];
};

struct Frame {
    uint8_t* big;    // the 128-row tiles
    uint8_t* ring;   // STAGES pairs of 64-row tiles
    uint8_t* stage;  // the warp's STAGE_BYTES
    Bars* bar;
    Slots* slots;
    float* extra;  // 16-byte aligned
    uint32_t tmem;
};

// mbar_wait (common.cuh), looking at the clock and the abort word only every
// 32 tries: reading the clock takes some hundred cycles, which a barrier that
// is about to complete would wait for.
__device__ __forceinline__ bool wait_one(uint64_t* bar, uint32_t parity, int* err, int* abort) {
    unsigned long long t0 = 0;
    for (unsigned tries = 1;; tries++) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((tries & 31) != 0) continue;
        if (*(volatile int*)abort) return false;
        const unsigned long long now = globaltimer();
        if (tries == 32) t0 = now;
        if (now - t0 > WAIT_LIMIT_NS) {
            atomicOr(err, ERR_WAIT_TIMEOUT);
            *(volatile int*)abort = 1;
            return false;
        }
    }
}

// The same at the end of a pass, whatever the abort word says.
__device__ __forceinline__ void drain(uint64_t* bar, uint32_t parity, int* err, int* abort) {
    const unsigned long long t0 = globaltimer();
    while (!mbar_try_wait(bar, parity))
        if (globaltimer() - t0 > WAIT_LIMIT_NS) {
            atomicOr(err, ERR_WAIT_TIMEOUT);
            *(volatile int*)abort = 1;
            return;
        }
}

// The loading warp: items in order, their tiles into the ring. A stage is full
// when its boxes have landed, zeroed where they must be, and every lane has
// arrived (32 lanes, and lane 0 once more: with the bytes it expects, or for
// them).
template <typename C>
struct Loader {
    const Frame& f;
    const AttnArgs& a;
    int lane;
    int items = 0, issued = 0;
    int patch = -1;  // the stage that waits for its zeros
    uint32_t patch_bits[2] = {0, 0};
    uint32_t landed_parity = 0;  // one bit a stage

    __device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
        fill();  // a warp that has to wait first hands over what it holds
        return __all_sync(0xffffffffu, wait_one(bar, parity, a.status, &f.bar->abort));
    }
    // The pending stage's zeros, once its box has landed: also in a CTA that gives
    // up, or the box could write to shared memory that is another CTA's by then.
    __device__ __forceinline__ void fill() {
        if (patch < 0) return;
        Bars* bar = f.bar;
        const uint32_t parity = landed_parity >> patch & 1;
        if (!wait_one(&bar->landed[patch], parity, a.status, &bar->abort))
            drain(&bar->landed[patch], parity, a.status, &bar->abort);
        landed_parity ^= 1u << patch;
        uint8_t* s = f.ring + patch * 2 * SMALL;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        // 16 lanes a row (both tiles), two rows at a time
        uint8_t* to = s + (lane >> 3 & 1) * SMALL + (lane >> 4) * 128 + (lane & 7) * 16;
        const uint32_t there0 = patch_bits[0] >> (lane >> 4), there1 = patch_bits[1] >> (lane >> 4);
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (!((i < 16 ? there0 : there1) >> (2 * i & 31) & 1)) *reinterpret_cast<uint4*>(to + i * 256) = zero;
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar->full[patch]);
        mbar_arrive(&bar->full[patch]);
        patch = -1;
    }
    // Room for the next item (and what a kernel keeps beside it).
    __device__ __forceinline__ bool slot() { return wait(&f.bar->item_empty[items & 1], ((items >> 1) & 1) ^ 1); }
    // The next item for everyone, and its 128-row tiles (columns `col`) once
    // the one before has no use for the old ones.
    __device__ __forceinline__ bool item(const Item& it, const CUtensorMap* b0, const CUtensorMap* b1) {
        Bars* bar = f.bar;
        const int s = items & 1;
        if (!slot()) return false;
        if (lane == 0) f.slots->item[s] = it;
        mbar_arrive(&bar->item_full[s]);
        if (it.n >= 0) {
            if (!wait(&bar->big_empty, (items & 1) ^ 1)) return false;
            if (lane == 0) {
                mbar_arrive_expect_tx(&bar->big_full, C::BIGS * BIG);
                const int row = it.start + it.row0;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    tma_load_2d(f.big + i * SMALL, b0, &bar->big_full, it.head * 64, row + i * STEP);
                    if (C::BIGS > 1) tma_load_2d(f.big + BIG + i * SMALL, b1, &bar->big_full, it.head * 64, row + i * STEP);
                }
            }
        }
        items++;
        return true;
    }
    __device__ __forceinline__ bool room() { return wait(&f.bar->empty[issued % STAGES], ((issued / STAGES) & 1) ^ 1); }
    // Rows `row` of both arrays (column `col`) into the next stage.
    __device__ __forceinline__ void tile(const CUtensorMap* m0, const CUtensorMap* m1, int col, int row,
                                         const uint32_t (&bits)[2]) {
        Bars* bar = f.bar;
        const int s = issued % STAGES;
        const bool whole = (bits[0] & bits[1]) == ~0u;
        if (lane == 0) {
            uint64_t* b = whole ? &bar->full[s] : &bar->landed[s];
            mbar_arrive_expect_tx(b, 2 * SMALL);
            tma_load_2d(f.ring + 2 * s * SMALL, m0, b, col, row);
            tma_load_2d(f.ring + (2 * s + 1) * SMALL, m1, b, col, row);
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
    // Every box has landed before shared memory goes away. `big`: of this many
    // items the 128-row tiles were asked for.
    __device__ __forceinline__ void finish(int big) {
        fill();
        int* abort = &f.bar->abort;
        for (int j = max(0, issued - STAGES); j < issued; j++)
            drain(&f.bar->full[j % STAGES], (j / STAGES) & 1, a.status, abort);
        if (big > 0) drain(&f.bar->big_full, (big - 1) & 1, a.status, abort);
    }
};

}  // namespace
}  // namespace laya
