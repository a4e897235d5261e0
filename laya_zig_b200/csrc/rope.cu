// rope.cu -- rotary positions over strided rows, and their transpose.
//
// Pair i of a head at position p turns by p * f_i radians. The angle is kept
// in turns, as a 64-bit fraction: the plan holds f_i / (2 pi) modulo 1 in
// units of 2^-64, so p * turn[i] modulo 2^64 is the exact fractional turn of
// that frequency for every 32-bit position, and its top 32 bits, as a signed
// number, are what sincospi gets. A product in f32 would be off by p * f_i *
// 2^-24 radians, 2e-3 at position 32,768; this is off by 2^-25 turns.
//
// Reads and writes each element once and computes one sine and cosine per
// (token, pair), which all heads of the token share: a warp owns a token,
// its lanes take a pair each for the table (in shared memory) and then 16
// bytes each of the row. Bound by memory: 64 sequences of 175-180 tokens, 24
// heads of 64, bf16 (70 MB) 14.9 us, 4.7 TB/s; 32,768 tokens with 32 of 64
// elements rotated, f16 (201 MB) 33.7 us, 6.0 TB/s; the former in f32 (139 MB) 23.2
// us, 6.0 TB/s, in place 15.1 us, with a position a row 14.0; rows that are not 16-byte
// aligned, an element at a time, 41 us; one sequence of 64 tokens
// 2.5 us. The first pieces are loaded before the search of the position and
// the table, which leave the memory idle at a call's beginning and end; set up
// while the kernel before ends, calls in a row take 14.8 instead of 16.4 us and 34.9
// instead of 37.4.
#include <cmath>

#include "operators.cuh"

namespace laya {
namespace {

constexpr int WARPS = 4;
constexpr int PAIRS = LAYA_ROPE_MAX_HEAD_DIM / 2;
constexpr int BATCH = 4;  // pieces a lane has in flight

template <typename T>
struct Chunk {
    static constexpr int N = 16 / sizeof(T);
    T e[N];
};

template <typename T>
__device__ __forceinline__ Chunk<T> load_chunk(const T* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    return *reinterpret_cast<const Chunk<T>*>(&u);
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const Chunk<T>& c) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&c);
}

// HALF: pairs (i, i + rot/2), else (2i, 2i + 1). VEC: 16-byte pieces, which
// need rot/2 (HALF) or rot (interleaved) and head_dim to be whole chunks.
template <typename T, bool HALF, bool VEC>
__global__ void __launch_bounds__(WARPS * 32) rope_kernel(const __grid_constant__ laya_rope_plan plan,
                                                          const T* x, long long x_stride, T* y,
                                                          long long y_stride, int n_tokens, int heads,
                                                          const int* __restrict__ cu, int n_seqs,
                                                          const int* __restrict__ positions, float sign,
                                                          int* status) {
    __shared__ float2 table[WARPS][PAIRS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * WARPS + warp;
    griddep_begin();
    if (cu) {  // every thread of the grid checks table entries
        for (long long s = (long long)blockIdx.x * blockDim.x + threadIdx.x; s < n_seqs;
             s += (long long)gridDim.x * blockDim.x)
            if (!run_ok(cu[s], cu[s + 1], n_tokens, n_tokens)) atomicOr(status, ERR_BAD_INDEX);
    }
    if (t >= n_tokens) return;
    const T* xr = x + t * x_stride;
    T* yr = y + t * y_stride;
    const bool copy = x != y;  // elements that no pair holds
    // The row in pieces: 16 bytes, or two of the pair's halves. The first
    // batch is on its way before the token's position is known.
    constexpr int N = Chunk<T>::N;
    const int rot_items = HALF ? (int)plan.rot_dim / (2 * N) : (int)plan.rot_dim / N;
    const int items = rot_items + (copy ? (int)(plan.head_dim - plan.rot_dim) / N : 0);
    int h = VEC ? lane / items : 0, it = VEC ? lane % items : 0;
    const int dh = VEC ? 32 / items : 0, di = VEC ? 32 % items : 0;
    Chunk<T> a[BATCH], b[BATCH];
    int at[BATCH], piece[BATCH];
    auto load_batch = [&]() {
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            at[u] = -1;
            piece[u] = it;
            if (h < heads) {
                at[u] = h * (int)plan.head_dim +
                        (it >= rot_items ? (int)plan.rot_dim + (it - rot_items) * N : it * N);
                a[u] = load_chunk(xr + at[u]);
                if (HALF && it < rot_items) b[u] = load_chunk(xr + at[u] + plan.rot_dim / 2);
            }
            h += dh;
            it += di;
            if (it >= items) {
                it -= items;
                h++;
            }
        }
    };
    if constexpr (VEC) load_batch();
    int pos;
    if (positions) {
        pos = positions[t];
    } else {
        const int s = warp_search(n_seqs, lane, [&](int i) { return (long long)cu[i]; }, t);
        if (s < 0) return;
        const int start = cu[s], end = cu[s + 1];
        if (!run_ok(start, end, n_tokens, n_tokens) || t < start || t >= end) return;
        pos = t - start;
    }
    const int half = plan.rot_dim / 2, hd = plan.head_dim, rot = plan.rot_dim;
    for (int i = lane; i < half; i += 32) {
        const uint64_t turns = (uint64_t)(int64_t)pos * plan.turn[i];
        const float f = (float)(int32_t)(uint32_t)(turns >> 32) * 0x1p-31f;  // half turns, [-1, 1]
        float s, c;
        sincospif(f, &s, &c);
        table[warp][i] = make_float2(c * plan.magnitude, s * plan.magnitude * sign);
    }
    __syncwarp();
    const float2* tab = table[warp];
    if constexpr (VEC) {
        while (true) {
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                if (at[u] < 0) continue;
                const int i = piece[u];
                if (i >= rot_items) {
                    store_chunk(yr + at[u], a[u]);
                } else if (HALF) {
#pragma unroll
                    for (int j = 0; j < N; j++) {
                        const float2 cs = tab[i * N + j];
                        const float p = to_float(a[u].e[j]), q = to_float(b[u].e[j]);
                        a[u].e[j] = from_float<T>(p * cs.x - q * cs.y);
                        b[u].e[j] = from_float<T>(p * cs.y + q * cs.x);
                    }
                    store_chunk(yr + at[u], a[u]);
                    store_chunk(yr + at[u] + half, b[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < N; j += 2) {
                        const float2 cs = tab[(i * N + j) / 2];
                        const float p = to_float(a[u].e[j]), q = to_float(a[u].e[j + 1]);
                        a[u].e[j] = from_float<T>(p * cs.x - q * cs.y);
                        a[u].e[j + 1] = from_float<T>(p * cs.y + q * cs.x);
                    }
                    store_chunk(yr + at[u], a[u]);
                }
            }
            if (h >= heads) break;
            load_batch();
        }
    } else {
        const int rest = copy ? hd - rot : 0;
        const int items = half + rest;
        const int total = items * heads;
        for (int w = lane; w < total; w += 32) {
            const int h = w / items, i = w - h * items;
            const long long at = (long long)h * hd;
            if (i >= half) {
                yr[at + rot + i - half] = xr[at + rot + i - half];
            } else {
                const long long o0 = at + (HALF ? i : 2 * i), o1 = HALF ? o0 + half : o0 + 1;
                const float2 cs = tab[i];
                const float u = to_float(xr[o0]), v = to_float(xr[o1]);
                yr[o0] = from_float<T>(u * cs.x - v * cs.y);
                yr[o1] = from_float<T>(u * cs.y + v * cs.x);
            }
        }
    }
}

template <typename T>
cudaError_t launch_t(const laya_rope_plan& plan, const void* x, long long x_stride, void* y, long long y_stride,
                     int n_tokens, int heads, const int* cu, int n_seqs, const int* positions, float sign, bool vec,
                     int* status, cudaStream_t stream) {
    const bool half = plan.layout == LAYA_ROPE_HALF;
    const int n = Chunk<T>::N;
    vec = vec && plan.head_dim % n == 0 && plan.rot_dim % (half ? 2 * n : n) == 0;
    const unsigned grid = ((unsigned)n_tokens + WARPS - 1) / WARPS;
    auto k = half ? (vec ? rope_kernel<T, true, true> : rope_kernel<T, true, false>)
                  : (vec ? rope_kernel<T, false, true> : rope_kernel<T, false, false>);
    return launch_k(k, dim3(grid), dim3(WARPS * 32), 0, stream, plan, static_cast<const T*>(x), x_stride,
                    static_cast<T*>(y), y_stride, n_tokens, heads, cu, n_seqs, positions, sign, status);
}

}  // namespace

cudaError_t launch_rope(const laya_rope_plan& plan, const void* x, long long x_stride, void* y, long long y_stride,
                        int n_tokens, int heads, const int* cu, int n_seqs, const int* positions, bool inverse,
                        int dtype, bool vec, int* status, cudaStream_t stream) {
    const float sign = inverse ? -1.f : 1.f;
    if (dtype == LAYA_DT_F32)
        return launch_t<float>(plan, x, x_stride, y, y_stride, n_tokens, heads, cu, n_seqs, positions, sign, vec,
                               status, stream);
    if (dtype == LAYA_DT_F16)
        return launch_t<__half>(plan, x, x_stride, y, y_stride, n_tokens, heads, cu, n_seqs, positions, sign, vec,
                                status, stream);
    return launch_t<__nv_bfloat16>(plan, x, x_stride, y, y_stride, n_tokens, heads, cu, n_seqs, positions, sign, vec,
                                   status, stream);
}

}  // namespace laya
