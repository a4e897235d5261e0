// attention_op.cuh -- what the attention operator's kernels share.
// attention_op.cu: 64 x 64 tiles on mma.sync; attention_op_tc.cu: tcgen05;
// attention_op_delta.cu: the backward pass's row sums.
#pragma once
#include "operators.cuh"

namespace laya {

constexpr float LOG2E = 1.4426950408889634f;

struct AttnArgs {
    const int* cu;
    const uint8_t* mask;
    int* status;
    int n_seqs, n_tokens, max_len;
    int group;  // query heads per key head
    int window;
    float scale;
    AttnIO io;
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
}

// c (16 x 8) += a (16 x 16) . b (16 x 8)
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16 (or 4) bytes from global to shared memory, zeros where !ok
__device__ __forceinline__ void copy16(void* s, const void* g, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(s)), "l"(g), "r"(ok ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy4(void* s, const void* g, bool ok) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(s)), "l"(g), "r"(ok ? 4 : 0)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Is token `i` of the sequence (any integer) there?
__device__ __forceinline__ bool present(const AttnArgs& a, const SeqTile& t, int i) {
    return i >= 0 && i < t.len && (!a.mask || a.mask[t.start + i] != 0);
}

// Tiles [t0, t1) of `tile` rows of the sequence that rows row0 .. row0 + rows
// - 1 see (the window is symmetric: keys of queries or queries of keys).
__device__ __forceinline__ void visible_tiles(const AttnArgs& a, const SeqTile& t, int rows, int tile, int* t0,
                                              int* t1) {
    int lo = 0, hi = t.len;
    if (a.window >= 0) {
        lo = max(0, t.row0 - a.window);
        hi = (int)min((long long)t.len, (long long)t.row0 + rows + a.window);
    }
    *t0 = lo / tile;
    *t1 = (hi + tile - 1) / tile;
}

// Does some pair of rows row0 .. + rows - 1 and col0 .. + cols - 1 lie outside the window?
__device__ __forceinline__ bool edge(int window, int row0, int rows, int col0, int cols) {
    return window >= 0 && (row0 + rows - 1 - col0 > window || col0 + cols - 1 - row0 > window);
}

// Rows whose delta is the sum of P dP whatever else the call holds: those of
// sequences of SHORT tokens at most, those of windows of NARROW at most, and those
// that see FEW keys at most (attention_op_delta.cu).
constexpr int SHORT = 32, NARROW = 4, FEW = 5;
static_assert(FEW <= NARROW + 1, "at the ends of a sequence a wider window has more keys");
inline bool narrow(int window) { return window >= 0 && window <= NARROW; }

// The keys of a sequence that its row i may see: lo .. hi.
__device__ __forceinline__ void span(const AttnArgs& a, const SeqTile& t, int i, int* lo, int* hi) {
    *lo = 0;
    *hi = t.len - 1;
    if (a.window >= 0) {
        *lo = max(*lo, i - a.window);
        *hi = (int)min((long long)*hi, (long long)i + a.window);
    }
}

// Eight elements of a row of a head.
template <typename T>
__device__ __forceinline__ uint4 piece(const AttnRows& r, long long row, int head, int c) {
    return *reinterpret_cast<const uint4*>(static_cast<const T*>(r.p) + row * r.ld + head * 64 + c);
}
template <typename T>
__device__ __forceinline__ float dot8(const uint4& x, const uint4& y) {
    const T* p = reinterpret_cast<const T*>(&x);
    const T* q = reinterpret_cast<const T*>(&y);
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) sum = fmaf(to_float(p[e]), to_float(q[e]), sum);
    return sum;
}

// attention_op_delta.cu: delta of every present token and head (of short sequences in
// io.delta_short), and the two counters set to 0.
cudaError_t launch_attention_delta(bool bf16, int n_heads, const AttnArgs& a, cudaStream_t stream);

// attention_op_tc.cu
cudaError_t launch_attention_fwd_tc(bool bf16, int n_heads, const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_attention_bwd_tc(bool bf16, int n_heads, int n_kv_heads, const AttnArgs& a, cudaStream_t stream);

}  // namespace laya
