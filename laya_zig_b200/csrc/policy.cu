// policy.cu -- the clipped policy loss over each decision's options, with its
// gradient, in one pass over the logits.
//
// Per decision, z = logits / t: lse = log sum e^z, lp_j = z_j - lse, p_j =
// e^lp_j; H = -sum p_j lp_j; d_j = lp_j - log ref_j and
//   KL(p||ref) = sum p_j d_j = sum (p_j d_j - p_j + ref_j),
// whose terms p (d + e^-d - 1) are never negative and vanish quadratically in
// d: a rounding error in either lse cancels to first order, so a policy that
// has hardly moved still gets its KL to f32 accuracy. The gradient with
// respect to z is
//   g (delta_ja - p_j) + kl_coef p_j (d_j - KL) + entropy_coef p_j (lp_j + H),
// g = -r A while the unclipped term is the smaller one, else 0.
//
// A decision's options are read once and stay in registers (a group of G
// lanes, V options each, G * V >= max_options); sums are warp shuffles in a
// fixed order. Above 1,024 options a block takes a decision and reads it
// three times. The bytes are 3 per option and element byte; what bounds the
// small ones is the launch.
#include "operators.cuh"

namespace laya {
namespace {

constexpr int THREADS = 256;

struct Scalars {
    const int* cu;
    const uint32_t* qtypes;
    int n, G;
    int max_k;
    float inv_t[3];
    float lo, hi, kl_coef, ent_coef;
    int* status;
};

template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What one thread needs of its decision besides the options.
struct Decision {
    int start, k, action;
    float adv, old_logp, grad, inv_t;
    bool ok;
};

__device__ __forceinline__ Decision load_decision(const Scalars& s, const PolicyIO& io, int i) {
    Decision d;
    const int start = s.cu[i], end = s.cu[i + 1];
    d.start = start;
    d.k = end - start;
    d.action = io.actions[i];
    const uint32_t q = s.qtypes ? s.qtypes[i] : 0u;
    d.adv = io.adv[i];
    d.old_logp = io.old_logp[i];
    d.grad = io.grad ? io.grad[i] : 1.f;
    const bool run = run_ok(start, end, s.G, s.max_k);
    d.ok = run && q <= 2u && (d.k == 0 || (d.action >= 0 && d.action < d.k));
    d.inv_t = s.inv_t[q <= 2u ? q : 0u];
    if (!run) d.k = 0;  // nothing of it can be addressed
    return d;
}

struct Result {
    float loss, logp, kl, ent;
    float g;  // d loss / d logp through the clipped ratio
};

__device__ __forceinline__ Result finish(const Scalars& s, const Decision& d, float logp, float kl, float ent) {
    Result r;
    r.logp = logp;
    r.kl = kl;
    r.ent = ent;
    const float ratio = expf(logp - d.old_logp);
    const float free_ = ratio * d.adv;
    const float held = fminf(fmaxf(ratio, s.lo), s.hi) * d.adv;
    const bool active = !(free_ > held);  // NaN stays NaN
    r.loss = -(active ? free_ : held) + s.kl_coef * kl - s.ent_coef * ent;
    r.g = active ? -free_ : 0.f;
    return r;
}

__device__ __forceinline__ void store_scalars(const PolicyIO& io, int i, const Result& r) {
    if (io.loss) io.loss[i] = r.loss;
    if (io.logp) io.logp[i] = r.logp;
    if (io.kl) io.kl[i] = r.kl;
    if (io.entropy) io.entropy[i] = r.ent;
}

// One option's share of the KL, from its log probabilities.
__device__ __forceinline__ float kl_term(float lp, float p, float lr) {
    const float d = lp - lr;
    // p (d + e^-d - 1); away from 0 the plain difference of probabilities
    return p > 0.f ? p * d + (fabsf(d) < 0.5f ? p * expm1f(-d) : expf(lr) - p) : expf(lr);
}

template <typename T, int G, int V>
__global__ void __launch_bounds__(THREADS) policy_kernel(Scalars s, PolicyIO io) {
    const int group = threadIdx.x / G, l = threadIdx.x % G;
    const long long at = (long long)blockIdx.x * (THREADS / G) + group;
    const bool live = at < s.n;
    const int i = live ? (int)at : s.n - 1;  // whole warps take part in the shuffles
    Decision d = load_decision(s, io, i);
    if (live && !d.ok && l == 0) atomicOr(s.status, ERR_BAD_INDEX);
    const T* x = static_cast<const T*>(io.logits) + d.start;
    const T* xr = static_cast<const T*>(io.ref) + d.start;
    const int k = d.k;
    float z[V], zr[V];
    float m = -INFINITY, mr = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int j = l + v * G;
        z[v] = j < k ? to_float(x[j]) * d.inv_t : -INFINITY;
        zr[v] = io.ref && j < k ? to_float(xr[j]) * d.inv_t : -INFINITY;
    }
#pragma unroll
    for (int v = 0; v < V; v++) {
        m = fmaxf(m, z[v]);
        mr = fmaxf(mr, zr[v]);
    }
    m = group_max<G>(m);
    mr = group_max<G>(mr);
    const float mz = m == -INFINITY ? 0.f : m, mrz = mr == -INFINITY ? 0.f : mr;
    float sum = 0.f, sumr = 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
        sum += expf(z[v] - mz);
        sumr += expf(zr[v] - mrz);
    }
    sum = group_sum<G>(sum);
    sumr = group_sum<G>(sumr);
    const bool some = d.ok && !(sum == 0.f);  // an option that is not ruled out
    const float lse = mz + logf(sum), lser = mrz + logf(sumr);
    float ent = 0.f, kl = 0.f, lpa = 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
        const int j = l + v * G;
        z[v] -= lse;  // log p
        const float p = expf(z[v]);
        if (p > 0.f) ent -= p * z[v];
        if (j == d.action) lpa = z[v];
        if (io.ref && j < k) {
            zr[v] -= lser;
            kl += kl_term(z[v], p, zr[v]);
        }
    }
    ent = group_sum<G>(ent);
    kl = group_sum<G>(kl);
    lpa = group_sum<G>(lpa);  // one lane holds it
    Result r = some ? finish(s, d, lpa, kl, ent) : Result{};
    if (!live) return;
    if (l == 0) store_scalars(io, i, r);
    if (io.dlogits) {
        T* dx = static_cast<T*>(io.dlogits) + d.start;
        const float w = d.grad * d.inv_t;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const int j = l + v * G;
            if (j >= k) continue;
            float g = 0.f;
            if (some && !(z[v] == -INFINITY)) {  // not ruled out
                const float lp = z[v], p = expf(lp);
                g = r.g * ((j == d.action ? 1.f : 0.f) - p);
                if (!(p == 0.f)) {
                    if (io.ref) g += s.kl_coef * p * (lp - zr[v] - r.kl);
                    g += s.ent_coef * p * (lp + r.ent);
                }
                g *= w;
            }
            dx[j] = from_float<T>(g);
        }
    }
}

__device__ __forceinline__ float block_reduce(float v, bool is_max, float* buf) {
    v = is_max ? warp_max(v) : warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = buf[0];
    for (int w = 1; w < THREADS / 32; w++) r = is_max ? fmaxf(r, buf[w]) : r + buf[w];
    return r;
}

// A decision of any number of options: a block reads it three times.
template <typename T>
__global__ void __launch_bounds__(THREADS) policy_wide_kernel(Scalars s, PolicyIO io) {
    __shared__ float buf[THREADS / 32];
    for (long long at = blockIdx.x; at < s.n; at += gridDim.x) {
        const int i = (int)at;
        Decision d = load_decision(s, io, i);
        if (!d.ok && threadIdx.x == 0) atomicOr(s.status, ERR_BAD_INDEX);
        const T* x = static_cast<const T*>(io.logits) + d.start;
        const T* xr = static_cast<const T*>(io.ref) + d.start;
        const int k = d.k;
        float m = -INFINITY, mr = -INFINITY;
        for (int j = threadIdx.x; j < k; j += THREADS) {
            m = fmaxf(m, to_float(x[j]) * d.inv_t);
            if (io.ref) mr = fmaxf(mr, to_float(xr[j]) * d.inv_t);
        }
        m = block_reduce(m, true, buf);
        mr = block_reduce(mr, true, buf);
        const float mz = m == -INFINITY ? 0.f : m, mrz = mr == -INFINITY ? 0.f : mr;
        float sum = 0.f, sumr = 0.f;
        for (int j = threadIdx.x; j < k; j += THREADS) {
            sum += expf(to_float(x[j]) * d.inv_t - mz);
            if (io.ref) sumr += expf(to_float(xr[j]) * d.inv_t - mrz);
        }
        sum = block_reduce(sum, false, buf);
        sumr = block_reduce(sumr, false, buf);
        const bool some = d.ok && !(sum == 0.f);
        const float lse = mz + logf(sum), lser = mrz + logf(sumr);
        float ent = 0.f, kl = 0.f, lpa = 0.f;
        for (int j = threadIdx.x; j < k; j += THREADS) {
            const float lp = to_float(x[j]) * d.inv_t - lse, p = expf(lp);
            if (p > 0.f) ent -= p * lp;
            if (j == d.action) lpa = lp;
            if (io.ref) kl += kl_term(lp, p, to_float(xr[j]) * d.inv_t - lser);
        }
        ent = block_reduce(ent, false, buf);
        kl = block_reduce(kl, false, buf);
        lpa = block_reduce(lpa, false, buf);
        const Result r = some ? finish(s, d, lpa, kl, ent) : Result{};
        if (threadIdx.x == 0) store_scalars(io, i, r);
        if (io.dlogits) {
            T* dx = static_cast<T*>(io.dlogits) + d.start;
            const float w = d.grad * d.inv_t;
            for (int j = threadIdx.x; j < k; j += THREADS) {
                float g = 0.f;
                const float lp = to_float(x[j]) * d.inv_t - lse;
                if (some && !(lp == -INFINITY)) {
                    const float p = expf(lp);
                    g = r.g * ((j == d.action ? 1.f : 0.f) - p);
                    if (!(p == 0.f)) {
                        if (io.ref) g += s.kl_coef * p * (lp - (to_float(xr[j]) * d.inv_t - lser) - r.kl);
                        g += s.ent_coef * p * (lp + r.ent);
                    }
                    g *= w;
                }
                dx[j] = from_float<T>(g);
            }
        }
    }
}

template <typename T, int G, int V>
cudaError_t launch_g(const Scalars& s, const PolicyIO& io, cudaStream_t stream) {
    constexpr int per = THREADS / G;
    policy_kernel<T, G, V><<<(unsigned)(((long long)s.n + per - 1) / per), THREADS, 0, stream>>>(s, io);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const Scalars& s, const PolicyIO& io, cudaStream_t stream) {
    if (s.max_k <= 16) return launch_g<T, 8, 2>(s, io, stream);
    if (s.max_k <= 128) return launch_g<T, 32, 4>(s, io, stream);
    if (s.max_k <= 1024) return launch_g<T, 32, 32>(s, io, stream);
    policy_wide_kernel<T><<<(unsigned)(s.n < 148 * 8 ? s.n : 148 * 8), THREADS, 0, stream>>>(s, io);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_policy(const laya_policy& p, const PolicyIO& io, cudaStream_t stream) {
    Scalars s;
    s.cu = p.cu_options;
    s.qtypes = p.qtypes;
    s.n = (int)p.n_decisions;
    s.G = (int)p.n_options;
    s.max_k = (int)p.max_options;
    for (int i = 0; i < 3; i++) s.inv_t[i] = 1.f / fmaxf(1e-3f, p.temperature[i]);
    s.lo = 1.f - p.clip_low;
    s.hi = 1.f + p.clip_high;
    s.kl_coef = p.kl_coef;
    s.ent_coef = p.entropy_coef;
    s.status = p.status;
    if (p.elem_dtype == LAYA_DT_F32) return launch_t<float>(s, io, stream);
    if (p.elem_dtype == LAYA_DT_F16) return launch_t<__half>(s, io, stream);
    return launch_t<__nv_bfloat16>(s, io, stream);
}

}  // namespace laya
