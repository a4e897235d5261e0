// The loading warp of the tcgen05 attention operator (csrc/attention_op_loader.cuh)
// on the CPU: 32 threads for its lanes, counted barriers for the mbarriers, and a
// copy engine that lands boxes when it is told to. What is checked is what the
// warp promises: no copy is under way once finish() has returned, not even in a
// CTA that gives up, and a stage is handed over with its box landed and the rows
// of absent tokens zero.
#include <algorithm>
#include <atomic>
#include <barrier>
#include <chrono>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <deque>
#include <map>
#include <mutex>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
using std::max;

// ---- stand-ins for common.cuh
struct alignas(16) uint4 {
    uint32_t x, y, z, w;
};
static uint4 make_uint4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return {a, b, c, d}; }
struct CUtensorMap {};

constexpr unsigned long long WAIT_LIMIT_NS = 20000000000ull;
constexpr int ERR_WAIT_TIMEOUT = 1;

static std::mutex mu;
struct Mbar {
    int count, left;
    long tx;
    uint32_t phase;
};
static std::map<uint64_t*, Mbar> bars;
static void settle(Mbar& b) {
    if (b.left == 0 && b.tx == 0) {
        b.left = b.count;
        b.phase ^= 1;
    }
}
static void mbar_init(uint64_t* p, int count) { bars[p] = Mbar{count, count, 0, 0}; }
static void mbar_arrive(uint64_t* p) {
    std::lock_guard<std::mutex> l(mu);
    Mbar& b = bars.at(p);
    b.left--;
    settle(b);
}
static void mbar_arrive_expect_tx(uint64_t* p, uint32_t bytes) {
    std::lock_guard<std::mutex> l(mu);
    Mbar& b = bars.at(p);
    b.tx += bytes;
    b.left--;
    settle(b);
}
static bool mbar_test_wait(uint64_t* p, uint32_t parity) {
    std::lock_guard<std::mutex> l(mu);
    return bars.at(p).phase != parity;
}
static bool mbar_try_wait(uint64_t* p, uint32_t parity) {
    if (mbar_test_wait(p, parity)) return true;
    std::this_thread::sleep_for(std::chrono::microseconds(200));
    return false;
}
static unsigned long long globaltimer() {
    return std::chrono::duration_cast<std::chrono::nanoseconds>(std::chrono::steady_clock::now().time_since_epoch()).count();
}
static void atomicOr(int* p, int v) { __atomic_fetch_or(p, v, __ATOMIC_SEQ_CST); }
static void fence_proxy_async() {}

static std::barrier<> warp(32);
static std::atomic<int> votes{0};
static void __syncwarp() { warp.arrive_and_wait(); }
static bool __all_sync(uint32_t, bool ok) {
    if (!ok) votes.fetch_add(1);
    warp.arrive_and_wait();
    const bool r = votes.load() == 0;
    warp.arrive_and_wait();
    votes.store(0);
    warp.arrive_and_wait();
    return r;
}

struct Copy {
    void* to;
    uint64_t* bar;
    uint32_t bytes;
};
static std::deque<Copy> under_way;  // guarded by mu
static void tma_load_2d(void* to, const CUtensorMap*, uint64_t* bar, int, int) {
    std::lock_guard<std::mutex> l(mu);
    under_way.push_back({to, bar, 64 * 64 * 2});
}
static bool land_one() {
    std::lock_guard<std::mutex> l(mu);
    if (under_way.empty()) return false;
    const Copy c = under_way.front();
    under_way.pop_front();
    memset(c.to, 0x5a, c.bytes);
    Mbar& b = bars.at(c.bar);
    b.tx -= c.bytes;
    settle(b);
    return true;
}
static size_t flying() {
    std::lock_guard<std::mutex> l(mu);
    return under_way.size();
}

namespace laya {
struct AttnArgs {
    int* status;
};
}  // namespace laya

#include "attention_op_loader.cuh"

using namespace laya;
using Shape2 = Shape<2, 0>;

static int failures = 0;
#define CHECK(x)                                            \
    do {                                                    \
        if (!(x)) {                                         \
            printf("line %d: %s\n", __LINE__, #x);          \
            failures++;                                     \
        }                                                   \
    } while (0)

struct Cta {
    alignas(1024) uint8_t big[2 * BIG];
    alignas(1024) uint8_t ring[STAGES * 2 * SMALL];
    Bars bar;
    Slots slots;
    int status = 0;
    AttnArgs a{&status};
    Frame f{};
    Cta() {
        memset(big, 0, sizeof big);
        memset(ring, 0x11, sizeof ring);
        bars.clear();
        under_way.clear();
        for (int s = 0; s < STAGES; s++) {
            mbar_init(&bar.full[s], 33);
            mbar_init(&bar.empty[s], 1);
            mbar_init(&bar.landed[s], 1);
        }
        mbar_init(&bar.big_full, 1);
        mbar_init(&bar.big_empty, 1);
        for (int s = 0; s < 2; s++) {
            mbar_init(&bar.item_full[s], 32);
            mbar_init(&bar.item_empty[s], 1);
        }
        bar.abort = 0;
        f.big = big;
        f.ring = ring;
        f.bar = &bar;
        f.slots = &slots;
    }
};

template <typename F>
static void run_warp(F lane_code) {
    std::vector<std::thread> lanes;
    for (int l = 0; l < 32; l++) lanes.emplace_back([&, l] { lane_code(l); });
    for (auto& t : lanes) t.join();
}

// A CTA that gives up with copies under way, which land late: `partial` has a bit
// for each tile with absent rows.
static void gives_up(int tiles, unsigned partial) {
    Cta c;
    std::atomic<bool> left{false};
    std::atomic<int> remaining{-1};
    std::thread engine([&] {
        while (!c.bar.abort) std::this_thread::yield();
        // the loader has long come to its end by now if nothing holds it
        for (int i = 0; i < 60 && !left; i++) std::this_thread::sleep_for(std::chrono::milliseconds(1));
        while (land_one()) std::this_thread::sleep_for(std::chrono::milliseconds(2));
    });
    run_warp([&](int lane) {
        Loader<Shape2> ld{c.f, c.a, lane};
        const CUtensorMap m;
        ld.item(Item{0, 500, 0, 0, 0, tiles}, &m, &m);
        for (int j = 0; j < tiles; j++) {
            const uint32_t bits[2] = {partial >> j & 1 ? 0x0000ffffu : ~0u, ~0u};
            if (j == std::min(1, tiles - 1)) {  // another role of the CTA gives up
                __syncwarp();
                if (lane == 0) *(volatile int*)&c.bar.abort = 1;
                __syncwarp();
            }
            ld.tile(&m, &m, 0, 64 * j, bits);
        }
        ld.room();  // nobody makes any, if the ring is full
        ld.finish(ld.items);
        __syncwarp();
        if (lane == 0) {
            remaining = (int)flying();
            left = true;
        }
    });
    engine.join();
    printf("gives up, %d tiles, partial %x: %d copies under way when it left\n", tiles, partial, (int)remaining);
    CHECK(remaining == 0);
}

// An ordinary item: every stage that is handed over is complete.
static void ordinary(int tiles, unsigned partial) {
    Cta c;
    std::atomic<bool> stop{false};
    std::thread engine([&] {
        while (!stop) {
            std::this_thread::sleep_for(std::chrono::microseconds(300));
            land_one();
        }
    });
    std::thread consumer([&] {
        for (int j = 0; j < tiles; j++) {
            const int s = j % STAGES;
            while (!mbar_try_wait(&c.bar.full[s], (j / STAGES) & 1)) {
            }
            bool good = true;
            for (int t = 0; t < 2; t++)
                for (int r = 0; r < STEP; r++) {
                    const bool there = !(partial >> j & 1) || (r < 16 || r >= 32);
                    for (int b = 0; b < 128; b++)
                        good &= c.ring[(2 * s + t) * SMALL + r * 128 + b] == (there ? 0x5a : 0);
                }
            CHECK(good);
            memset(c.ring + 2 * s * SMALL, 0x11, 2 * SMALL);
            mbar_arrive(&c.bar.empty[s]);
        }
    });
    run_warp([&](int lane) {
        Loader<Shape2> ld{c.f, c.a, lane};
        const CUtensorMap m;
        ld.item(Item{0, 500, 0, 0, 0, tiles}, &m, &m);
        for (int j = 0; j < tiles; j++) {
            const uint32_t bits[2] = {partial >> j & 1 ? 0x0000ffffu : ~0u, ~0u};
            if (!ld.room()) break;
            ld.tile(&m, &m, 0, 64 * j, bits);
        }
        ld.finish(ld.items);
    });
    consumer.join();
    stop = true;
    engine.join();
    CHECK(flying() == 0 && c.status == 0);
}

int main() {
    for (unsigned partial = 0; partial < 8; partial++) {
        gives_up(3, partial);
        ordinary(7, partial * 0x15);
    }
    gives_up(1, 1);
    gives_up(2, 2);
    return failures ? 1 : 0;
}
