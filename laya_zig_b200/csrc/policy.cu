// policy.cu -- the clipped policy loss over each decision's options, with its
// gradient, in one pass over the logits.
//
// Per decision, z = (logits - their maximum) / t: the difference first, so that a
// number added to all of a decision's logits costs no digits. lse = log sum e^z,
// lp_j = z_j - lse, p_j = e^lp_j; H = -sum p_j lp_j; d_j = lp_j - log ref_j and
//   KL(p||ref) = sum p_j d_j = sum (p_j d_j - p_j + ref_j),
// whose terms p (d + e^-d - 1) are never negative and vanish quadratically in
// d: a rounding error in either lse cancels to first order, so a policy that
// has hardly moved still gets its KL to f32 accuracy. The gradient with
// respect to z is
//   g (delta_ja - p_j) + kl_coef p_j (d_j - KL) + entropy_coef p_j (lp_j + H),
// g = -r A while the unclipped term is the smaller one, else 0.
//
// A decision's options are read once and stay in registers (a group of G
// threads, V options each, G * V >= max_options); sums are shuffles, over a
// block joined in shared memory, in a fixed order. Above 1,024 options a block
// takes a decision and reads it four times (maximum, sum, statistics, gradient),
// after the first time from cache.
//
// The bytes are logits, reference and gradient once each. On the device, f32
// with a reference: 64 decisions of 4 options 2.0 us, a launch; 65,536 of 4 to
// 16 (10.5 MB) 8.4 us, 1.3 TB/s (6.0 from L2); bf16, 16,384 of 1 to 1,024 (51 MB) 50
// us, 1.0 TB/s (42 from L2), bound by instructions (649 a warp, 3.1 of 4 a cycle issued): about half for
// the decision's scalars and three reductions over a block, however few its options,
// and some 70 for each of the four that a thread has on average.
#include "operators.cuh"

namespace laya {
namespace {

constexpr int THREADS = 128;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Scalars {
    const int* cu;
    const uint32_t* qtypes;
    int n, G;
    int max_k;
    float scale[3];   // log2(e) / temperature: differences of logits -> z in units of log 2
    float inv_t[3];
    float lo, hi, kl_coef, ent_coef;
    int* status;
};

// Sums or maxima of two values over the G threads of a decision, in a fixed
// order: part of a warp, a warp, or the whole block.
template <int G, bool MAX>
__device__ __forceinline__ void group_reduce(float& a, float& b, float2* buf) {
    auto join = [](float u, float v) { return MAX ? fmaxf(u, v) : u + v; };
#pragma unroll
    for (int o = (G < 32 ? G : 32) / 2; o > 0; o >>= 1) {
        const float u = __shfl_xor_sync(0xffffffffu, a, o), v = __shfl_xor_sync(0xffffffffu, b, o);
        a = join(a, u);
        b = join(b, v);
    }
    if (G > 32) {
        if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = make_float2(a, b);
        __syncthreads();
        a = buf[0].x;
        b = buf[0].y;
#pragma unroll
        for (int w = 1; w < G / 32; w++) {
            a = join(a, buf[w].x);
            b = join(b, buf[w].y);
        }
    }
}

// What one thread needs of its decision besides the options.
struct Decision {
    int start, k, action;
    float adv, old_logp, grad, inv_t, scale;
    float taken;  // the action's logit
    bool ok;
};

template <typename T>
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
    d.inv_t = q == 1u ? s.inv_t[1] : q == 2u ? s.inv_t[2] : s.inv_t[0];
    d.scale = q == 1u ? s.scale[1] : q == 2u ? s.scale[2] : s.scale[0];
    if (!run) d.k = 0;  // nothing of it can be addressed
    d.taken = d.ok && d.k > 0 ? to_float(static_cast<const T*>(io.logits)[start + d.action]) : -INFINITY;
    return d;
}

// log2 on the SFU: absolute error about 2^-22
__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What is made of the sum of e^z over the options that were not taken.
struct Sum {
    float taken;   // z of the option that was taken
    float others;  // 1 - p of it
    float lse;     // log2
    bool some;     // an option is not ruled out
};
// In a decision that is nearly certain the others are all that log p is made of:
// lg2.approx of 1 + rest would be off by 2^-22, not by that much of log p. With q = 1 -
// p <= 1/9, -log(1 - q) = q + q^2 / 2 + ... up to q^7 / 7; the next term is below 2^-25
// of the sum.
__device__ __forceinline__ Sum make_sum(const Decision& d, float mz, float rest) {
    Sum s;
    s.taken = (d.taken - mz) * d.scale;
    const float total = ex2_approx(s.taken) + rest;
    const float q = __fdividef(rest, total);
    s.some = d.ok && !(total == 0.f);
    s.others = q;
    float y = fmaf(q, LOG2E / 7.f, LOG2E / 6.f);
    y = fmaf(q, y, LOG2E / 5.f);
    y = fmaf(q, y, LOG2E / 4.f);
    y = fmaf(q, y, LOG2E / 3.f);
    y = fmaf(q, y, LOG2E / 2.f);
    y = fmaf(q, y, LOG2E);
    s.lse = s.taken == 0.f && rest < 0.125f ? q * y : lg2_approx(total);
    return s;
}

struct Result {
    float loss, logp, kl, ent;
    float g;  // d loss / d logp through the clipped ratio
};

// kl_coef times x, and 0 where the divergence is only reported: it may be infinite
// (a reference that rules out what the policy does not).
__device__ __forceinline__ float kl_times(const Scalars& s, float x) { return s.kl_coef == 0.f ? 0.f : s.kl_coef * x; }

__device__ __forceinline__ Result finish(const Scalars& s, const Decision& d, float logp, float kl, float ent) {
    Result r;
    r.logp = logp;
    r.kl = kl;
    r.ent = ent;
    const float ratio = ex2_approx((logp - d.old_logp) * LOG2E);
    const float free_ = ratio * d.adv;
    const float held = fminf(fmaxf(ratio, s.lo), s.hi) * d.adv;
    const bool active = !(free_ > held);  // NaN stays NaN
    r.loss = -(active ? free_ : held) + kl_times(s, kl) - s.ent_coef * ent;
    r.g = active ? -free_ : 0.f;
    return r;
}

__device__ __forceinline__ void store_scalars(const PolicyIO& io, int i, const Result& r) {
    if (io.loss) io.loss[i] = r.loss;
    if (io.logp) io.logp[i] = r.logp;
    if (io.kl) io.kl[i] = r.kl;
    if (io.entropy) io.entropy[i] = r.ent;
}

// One option's share of the KL in units of log 2, from its log2
// probabilities: p d - p + ref. For |d| < 1/4 that is p times the series of
// d + e^-d - 1 = d^2 (1/2 - d/6 + d^2/24 - ...), six terms of it (the next is
// below 2^-23 of the sum); from there on the plain differences, off by 2^-22 of p
// and ref each: 2^-16 of the term at 1/4, 2^-20 from 1 on. In units of log 2: a = log
// 2 times d.
__device__ __forceinline__ float kl_term(float d, float p, float lr) {
    constexpr float L = LN2;
    float g = fmaf(d, -L * L * L * L * L * L / 5040.f, L * L * L * L * L / 720.f);
    g = fmaf(d, g, -L * L * L * L / 120.f);
    g = fmaf(d, g, L * L * L / 24.f);
    g = fmaf(d, g, -L * L / 6.f);
    g = fmaf(d, g, L / 2.f);
    const float near = p * d * (d * g);
    const float far = fmaf(p, d, (ex2_approx(lr) - p) * (1.f / L));
    return !(p == 0.f) && fabsf(d) < 0.25f / L ? near : p == 0.f ? ex2_approx(lr) * (1.f / L) : far;
}

// dloss/dz of one option, times the weights: p (c0 + c1 d + c2 lp); of the option
// that was taken p (c + c1 d + c2 lp) plus own, which is g (1 - p) from the other
// options' sum: 1 - p as a difference would leave a certain decision's gradients no
// digits.
struct Slope {
    float own, c, c0, c1, c2;
};
__device__ __forceinline__ Slope slope(const Scalars& s, const Decision& d, const Result& r, float others) {
    const float w = d.grad * d.inv_t;
    Slope c;
    c.own = r.g * w * others;
    c.c = w * (s.ent_coef * r.ent - kl_times(s, r.kl));
    c.c0 = c.c - w * r.g;
    c.c1 = w * s.kl_coef * LN2;
    c.c2 = w * s.ent_coef * LN2;
    return c;
}

// REF: there are reference logits.
template <typename T, int G, int V, bool REF>
__global__ void __launch_bounds__(THREADS) policy_kernel(Scalars s, PolicyIO io) {
    static_assert(G <= 32 || G == THREADS, "a decision is part of a warp, a warp or a block");
    __shared__ float2 buf[3][THREADS / 32];  // one row for each block-wide reduction
    const int group = threadIdx.x / G, l = threadIdx.x % G;
    const long long at = (long long)blockIdx.x * (THREADS / G) + group;
    const bool live = at < s.n;
    const int i = live ? (int)at : s.n - 1;  // whole warps take part in the shuffles
    griddep_begin();
    Decision d = load_decision<T>(s, io, i);
    if (live && !d.ok && l == 0) atomicOr(s.status, ERR_BAD_INDEX);
    const T* x = static_cast<const T*>(io.logits) + d.start;
    const T* xr = REF ? static_cast<const T*>(io.ref) + d.start : x;
    const int k = d.k, mine = d.action - l;  // v * G if option v of this thread was taken
    // thread l holds options l, l + G, ..; all loads are under way before the
    // first is used
    float z[V], zr[V], p[V];
    {
        T raw[V], rawr[V];
#pragma unroll
        for (int v = 0; v < V; v++)
            if (l + v * G < k) raw[v] = x[l + v * G];
        if (REF) {
#pragma unroll
            for (int v = 0; v < V; v++)
                if (l + v * G < k) rawr[v] = xr[l + v * G];
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
            z[v] = l + v * G < k ? to_float(raw[v]) : -INFINITY;
            zr[v] = REF && l + v * G < k ? to_float(rawr[v]) : -INFINITY;
        }
    }
    float m = -INFINITY, mr = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; v++) {
        m = fmaxf(m, z[v]);
        mr = fmaxf(mr, zr[v]);
    }
    group_reduce<G, true>(m, mr, buf[0]);
    const float mz = m == -INFINITY ? 0.f : m, mrz = mr == -INFINITY ? 0.f : mr;
    float sum = 0.f, sumr = 0.f;
    // ex2.approx here and below: 2^-22 relative, of exponents whose own
    // rounding is small for every term that carries weight in a sum
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (v * G >= k) break;  // of the whole group
        z[v] = (z[v] - mz) * d.scale;
        if (v * G != mine) sum += ex2_approx(z[v]);
        if (REF) {
            zr[v] = (zr[v] - mrz) * d.scale;
            sumr += ex2_approx(zr[v]);
        }
    }
    group_reduce<G, false>(sum, sumr, buf[1]);
    const Sum t = make_sum(d, mz, sum);
    const float lse = t.lse, lser = lg2_approx(sumr);
    float ent = 0.f, kl = 0.f;
#pragma unroll
    for (int v = 0; v < V; v++) {
        if (v * G >= k) break;
        z[v] -= lse;  // log2 p
        p[v] = ex2_approx(z[v]);
        if (!(p[v] == 0.f)) ent = fmaf(-p[v], z[v], ent);
        if (REF && l + v * G < k) {
            zr[v] -= lser;
            const float dv = z[v] - zr[v];
            kl += kl_term(dv, p[v], zr[v]);
            zr[v] = dv;
        }
    }
    group_reduce<G, false>(ent, kl, buf[2]);
    Result r = t.some ? finish(s, d, (t.taken - lse) * LN2, kl * LN2, ent * LN2) : Result{};
    if (!live) return;
    if (l == 0) store_scalars(io, i, r);
    if (io.dlogits) {
        T* dx = static_cast<T*>(io.dlogits) + d.start;
        const Slope c = slope(s, d, r, t.others);
#pragma unroll
        for (int v = 0; v < V; v++) {
            if (v * G >= k) break;
            const int j = l + v * G;
            float g = fmaf(c.c2, z[v], v * G == mine ? c.c : c.c0);
            if (REF && s.kl_coef != 0.f) g = fmaf(c.c1, zr[v], g);
            g = p[v] == 0.f ? 0.f : p[v] * g;  // an option that is ruled out has log p = -inf
            if (v * G == mine) g += c.own;
            if (j < k) dx[j] = from_float<T>(t.some ? g : 0.f);
        }
    }
}

// A decision of any number of options: a block reads it four times.
template <typename T>
__global__ void __launch_bounds__(THREADS) policy_wide_kernel(Scalars s, PolicyIO io) {
    __shared__ float2 buf[3][THREADS / 32];
    griddep_begin();
    for (long long at = blockIdx.x; at < s.n; at += gridDim.x) {
        const int i = (int)at;
        Decision d = load_decision<T>(s, io, i);
        if (!d.ok && threadIdx.x == 0) atomicOr(s.status, ERR_BAD_INDEX);
        const T* x = static_cast<const T*>(io.logits) + d.start;
        const T* xr = static_cast<const T*>(io.ref) + d.start;
        const int k = d.k;
        float m = -INFINITY, mr = -INFINITY;
        for (int j = threadIdx.x; j < k; j += THREADS) {
            m = fmaxf(m, to_float(x[j]));
            if (io.ref) mr = fmaxf(mr, to_float(xr[j]));
        }
        group_reduce<THREADS, true>(m, mr, buf[0]);
        const float mz = m == -INFINITY ? 0.f : m, mrz = mr == -INFINITY ? 0.f : mr;
        float sum = 0.f, sumr = 0.f;
        for (int j = threadIdx.x; j < k; j += THREADS) {
            if (j != d.action) sum += ex2_approx((to_float(x[j]) - mz) * d.scale);
            if (io.ref) sumr += ex2_approx((to_float(xr[j]) - mrz) * d.scale);
        }
        group_reduce<THREADS, false>(sum, sumr, buf[1]);
        const Sum t = make_sum(d, mz, sum);
        const float lse = t.lse, lser = lg2_approx(sumr);
        float ent = 0.f, kl = 0.f;
        for (int j = threadIdx.x; j < k; j += THREADS) {
            const float lp = (to_float(x[j]) - mz) * d.scale - lse, p = ex2_approx(lp);
            if (!(p == 0.f)) ent = fmaf(-p, lp, ent);
            if (io.ref) {
                const float lr = (to_float(xr[j]) - mrz) * d.scale - lser;
                kl += kl_term(lp - lr, p, lr);
            }
        }
        group_reduce<THREADS, false>(ent, kl, buf[2]);
        const Result r = t.some ? finish(s, d, (t.taken - lse) * LN2, kl * LN2, ent * LN2) : Result{};
        __syncthreads();  // buf is free for the next decision
        if (threadIdx.x == 0) store_scalars(io, i, r);
        if (io.dlogits) {
            T* dx = static_cast<T*>(io.dlogits) + d.start;
            const Slope c = slope(s, d, r, t.others);
            for (int j = threadIdx.x; j < k; j += THREADS) {
                const float lp = (to_float(x[j]) - mz) * d.scale - lse, p = ex2_approx(lp);
                float g = fmaf(c.c2, lp, j == d.action ? c.c : c.c0);
                if (io.ref && s.kl_coef != 0.f) g = fmaf(c.c1, lp - ((to_float(xr[j]) - mrz) * d.scale - lser), g);
                g = p == 0.f ? 0.f : p * g;
                if (j == d.action) g += c.own;
                dx[j] = from_float<T>(t.some ? g : 0.f);
            }
        }
    }
}

template <typename T, int G, int V>
cudaError_t launch_g(const Scalars& s, const PolicyIO& io, cudaStream_t stream) {
    constexpr int per = THREADS / G;
    const unsigned grid = (unsigned)(((long long)s.n + per - 1) / per);
    return launch_k(io.ref ? policy_kernel<T, G, V, true> : policy_kernel<T, G, V, false>, dim3(grid), dim3(THREADS), 0,
                    stream, s, io);
}

template <typename T>
cudaError_t launch_t(const Scalars& s, const PolicyIO& io, cudaStream_t stream) {
    // The fewest threads to a decision that hold its options in registers:
    // what a group does once (its scalars, three reductions) is half the work.
    // 4 M options (f32) in decisions of up to 16 / 64 / 256: 17 / 14 / 13 us;
    // with the next larger group 26 / 19 / 19 us. (Up to 1,024, groups of 32
    // and 64 threads with more options each were no faster than the block.)
    if (s.max_k <= 16) return launch_g<T, 4, 4>(s, io, stream);
    if (s.max_k <= 32) return launch_g<T, 8, 4>(s, io, stream);
    if (s.max_k <= 64) return launch_g<T, 8, 8>(s, io, stream);
    if (s.max_k <= 128) return launch_g<T, 16, 8>(s, io, stream);
    if (s.max_k <= 256) return launch_g<T, 32, 8>(s, io, stream);
    if (s.max_k <= 512) return launch_g<T, 32, 16>(s, io, stream);
    if (s.max_k <= 1024) return launch_g<T, THREADS, 8>(s, io, stream);
    return launch_k(policy_wide_kernel<T>, dim3((unsigned)(s.n < 148 * 8 ? s.n : 148 * 8)), dim3(THREADS), 0, stream, s, io);
}

}  // namespace

cudaError_t launch_policy(const laya_policy& p, const PolicyIO& io, cudaStream_t stream) {
    Scalars s;
    s.cu = p.cu_options;
    s.qtypes = p.qtypes;
    s.n = (int)p.n_decisions;
    s.G = (int)p.n_options;
    s.max_k = (int)(p.max_options < p.n_options ? p.max_options : p.n_options);
    for (int i = 0; i < 3; i++) {
        s.inv_t[i] = 1.f / fmaxf(1e-3f, p.temperature[i]);
        s.scale[i] = (float)(1.4426950408889634 / fmaxf(1e-3f, p.temperature[i]));
    }
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
