// operators.cuh -- the training-step operators' kernels (declarations) and
// what they share. Entry points and argument checks: operators.cu.
#pragma once
#include "../../include/laya_gpu.h"
#include "common.cuh"

namespace laya {

// The kernels that use no tensor memory are launched by launch_k and start with
// this: they are set up while the kernel before them ends. The next kernel is let
// in only when that one is complete: one that allocates tensor memory before it
// waits would otherwise keep it from a kernel two places back that has yet to.
__device__ __forceinline__ void griddep_begin() {
    griddep_wait();
    griddep_launch();
}

// ------------------------------------------------------------------ offset tables
// The largest s of [0, n) with key(s) <= x, by the whole warp: 32 probes a
// round, so 1,024 entries take two dependent loads (a bisection takes ten).
// -1 if key(0) > x. On a table that is not sorted the result is some index of
// [-1, n), which the callers check.
template <typename Key>
__device__ __forceinline__ int warp_search(int n, int lane, Key key, long long x) {
    int lo = 0;
    bool first = true;
    while (n > 1 || first) {
        const int step = (n + 31) / 32;
        const int i = lane * step;
        const bool le = i < n && key(lo + i) <= x;
        const int c = __popc(__ballot_sync(0xffffffffu, le));
        if (c == 0) return first ? -1 : lo;
        lo += (c - 1) * step;
        n = min(step, n - (c - 1) * step);
        first = false;
    }
    return lo;
}

// Sequence s of an offset table: a run of [0, rows) no longer than max_len.
__device__ __forceinline__ bool run_ok(int start, int end, long long rows, long long max_len) {
    return start >= 0 && end >= start && end <= rows && (long long)end - start <= max_len;
}

// A block of attention work: one tile of `tile_rows` rows of one sequence.
struct SeqTile {
    int start, len, row0;  // the sequence's first row and length, the tile's first row within it
};

// Block x of a grid of seq_tiles() blocks -> its tile; false if it has none.
// Sequence s owns the blocks from start(s) / tile_rows + s up to the next
// sequence's: at least ceil(len / tile_rows) of them, whatever the lengths,
// so the grid needs no table of its own. Every warp finds its tile alone.
__device__ __forceinline__ bool find_tile(const int* __restrict__ cu, int n_seqs, int n_tokens, int max_len,
                                          int tile_rows, long long x, int lane, SeqTile* t) {
    const int s = warp_search(
        n_seqs, lane, [&](int i) { return (long long)(max(cu[i], 0) / tile_rows) + i; }, x);
    if (s < 0) return false;
    const int start = cu[s], end = cu[s + 1];
    if (!run_ok(start, end, n_tokens, max_len)) return false;  // recorded by check_table
    const long long tile = x - ((long long)(start / tile_rows) + s);
    t->start = start;
    t->len = end - start;
    if (tile < 0 || tile * tile_rows >= t->len) return false;
    t->row0 = (int)tile * tile_rows;
    return true;
}

inline long long seq_tiles(long long n_tokens, long long n_seqs, int tile_rows) {
    return n_tokens / tile_rows + n_seqs;
}

// Entry x of the table: the threads of a launch check all of them together.
__device__ __forceinline__ void check_table(const int* __restrict__ cu, int n_seqs, int n_tokens, int max_len,
                                            long long x, int* status) {
    if (x < n_seqs && !run_ok(cu[x], cu[x + 1], n_tokens, max_len)) atomicOr(status, ERR_BAD_INDEX);
}

// ------------------------------------------------------------------ element types
template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// ------------------------------------------------------------------ launchers
// rope.cu. vec: rows and chunks are 16-byte aligned (the host's check).
cudaError_t launch_rope(const laya_rope_plan& plan, const void* x, long long x_stride, void* y, long long y_stride,
                        int n_tokens, int heads, const int* cu, int n_seqs, const int* positions, bool inverse,
                        int dtype, bool vec, int* status, cudaStream_t stream);

// policy.cu
struct PolicyIO {
    const void *logits, *ref;
    const int* actions;
    const float *adv, *old_logp, *grad;
    float *loss, *logp, *kl, *entropy;
    void* dlogits;
};
cudaError_t launch_policy(const laya_policy& p, const PolicyIO& io, cudaStream_t stream);

// attention_op.cu
struct AttnRows {
    void* p;
    long long ld;  // elements from row to row
};
struct AttnIO {
    AttnRows q, k, v, out, dout, dq, dk, dv;
    float* lse;    // [n_heads][n_tokens]
    float* delta;  // [n_heads][n_tokens], of the backward pass's workspace
    float* delta_short;  // the same for short sequences: delta, or an array of its own
    unsigned long long* tickets;  // two counters, of the workspace
};
cudaError_t launch_attention_fwd(const laya_attention& a, const AttnIO& io, cudaStream_t stream);
cudaError_t launch_attention_bwd(const laya_attention& a, const AttnIO& io, cudaStream_t stream);

}  // namespace laya
