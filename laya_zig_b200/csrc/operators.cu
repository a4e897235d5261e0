// operators.cu -- entry points of the training-step operators: argument
// checks, then the launches. Nothing is allocated and nothing waited for, so
// every call but laya_gpu_op_status may be captured.
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "operators.cuh"

using namespace laya;

int laya_ctx_fail(laya_ctx* c, int code, const char* msg);  // laya_gpu.cu

namespace {

int fail(int code, const char* fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return laya_ctx_fail(nullptr, code, buf);
}

int cuda_fail(const char* op, cudaError_t e) {
    cudaGetLastError();  // a launch error is reported once, here
    return fail(LAYA_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
}

constexpr uint32_t MAX_ROWS = 1u << 30;  // row indexes and their sums with a tile stay inside 32 bits

// Is every pointer (nullptr entries skipped) aligned, and memory that a kernel
// on the current device may use? Host memory and another device's are refused
// here instead of faulting there.
struct Ptr {
    const char* name;
    const void* p;
    unsigned align = 4;  // bytes
};
template <int N>
int check_pointers(const char* op, const Ptr (&ptrs)[N]) {
    for (const Ptr& x : ptrs)
        if ((uintptr_t)x.p % x.align)
            return fail(LAYA_ERR_ARG, "%s: %s must be %u-byte aligned", op, x.name, x.align);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver ? LAYA_ERR_NO_DEVICE : LAYA_ERR_CUDA,
                    "%s: %s", op, cudaGetErrorString(e));
    }
    for (const Ptr& x : ptrs) {
        if (!x.p) continue;
        cudaPointerAttributes at;
        e = cudaPointerGetAttributes(&at, x.p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return fail(e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver ? LAYA_ERR_NO_DEVICE
                                                                                   : LAYA_ERR_CUDA,
                        "%s: %s: %s", op, x.name, cudaGetErrorString(e));
        }
        if (at.type == cudaMemoryTypeManaged) continue;
        if (at.type != cudaMemoryTypeDevice)
            return fail(LAYA_ERR_ARG, "%s: %s is not device memory", op, x.name);
        if (at.device != dev)
            return fail(LAYA_ERR_ARG, "%s: %s belongs to device %d, the current device is %d", op, x.name, at.device,
                        dev);
    }
    return LAYA_OK;
}

// A strided array of rows, in bytes.
struct Span {
    const char* name;
    const void* p;
    int64_t ld, width;
    uint64_t rows;
    bool written;
};

// May the two hold a byte in common? Exact for equal strides (columns of one
// packed row array do not overlap); otherwise any common address counts.
bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || !a.rows || !b.rows) return false;
    const uintptr_t pa = (uintptr_t)a.p, pb = (uintptr_t)b.p;
    const uintptr_t ea = pa + (a.rows - 1) * (uint64_t)a.ld + a.width, eb = pb + (b.rows - 1) * (uint64_t)b.ld + b.width;
    if (pa >= eb || pb >= ea) return false;
    if (a.ld != b.ld) return true;
    const uint64_t d = pb >= pa ? (pb - pa) % (uint64_t)a.ld : (a.ld - (pa - pb) % (uint64_t)a.ld) % (uint64_t)a.ld;
    return d < (uint64_t)a.width || d + b.width > (uint64_t)a.ld;
}

// What is written overlaps nothing else.
template <int N>
int check_overlap(const char* op, const Span (&s)[N]) {
    for (int i = 0; i < N; i++)
        for (int j = i + 1; j < N; j++)
            if ((s[i].written || s[j].written) && overlap(s[i], s[j]))
                return fail(LAYA_ERR_ARG, "%s: %s overlaps %s", op, s[i].name, s[j].name);
    return LAYA_OK;
}

int elem_size(int dtype) { return dtype == LAYA_DT_F32 ? 4 : 2; }

int check_attention(const char* op, const laya_attention* a) {
    if (!a) return fail(LAYA_ERR_ARG, "%s: NULL description", op);
    if (a->elem_dtype != LAYA_DT_BF16 && a->elem_dtype != LAYA_DT_F16)
        return fail(LAYA_ERR_DTYPE, "%s: elem_dtype %d (BF16 or F16)", op, a->elem_dtype);
    if (a->n_tokens > MAX_ROWS || a->n_seqs > MAX_ROWS)
        return fail(LAYA_ERR_ARG, "%s: %u tokens, %u sequences (2^30 at most)", op, a->n_tokens, a->n_seqs);
    if (!a->n_heads || !a->n_kv_heads || a->n_heads % a->n_kv_heads || a->n_heads > 65535)
        return fail(LAYA_ERR_ARG, "%s: %u heads over %u key heads", op, a->n_heads, a->n_kv_heads);
    if ((uint64_t)a->n_tokens * a->n_heads > 0xffff0000u)
        return fail(LAYA_ERR_ARG, "%s: %u tokens of %u heads (2^32 in all)", op, a->n_tokens, a->n_heads);
    if (!(a->scale > 0.f) || !std::isfinite(2.f * a->scale))  // it is multiplied by log2 e
        return fail(LAYA_ERR_ARG, "%s: scale must be positive and finite", op);
    if (a->n_tokens && a->n_seqs && (!a->cu_seqlens || !a->status))
        return fail(LAYA_ERR_ARG, "%s: NULL cu_seqlens or status", op);
    return LAYA_OK;
}

// Two counters, then delta twice: of all rows, and of those of short sequences.
constexpr uint64_t WORKSPACE_HEAD = 16;
uint64_t workspace_bytes_of(const laya_attention* a) {
    return WORKSPACE_HEAD + 2 * (uint64_t)a->n_heads * a->n_tokens * sizeof(float);
}

struct Rows {
    const char* name;
    const void* p;
    int64_t ld;
    uint32_t heads;
    bool written;
};

int check_rows(const char* op, const Rows& r) {
    if (!r.p) return fail(LAYA_ERR_ARG, "%s: %s is NULL", op, r.name);
    if ((uintptr_t)r.p & 15) return fail(LAYA_ERR_ARG, "%s: %s must be 16-byte aligned", op, r.name);
    if (r.ld < (int64_t)r.heads * LAYA_HEAD_DIM || r.ld % 8 || r.ld > (int64_t)1 << 31)
        return fail(LAYA_ERR_ARG, "%s: %s stride %lld (a multiple of 8, at least %u heads x %d)", op, r.name,
                    (long long)r.ld, r.heads, LAYA_HEAD_DIM);
    return LAYA_OK;
}

Span span(const Rows& r, uint64_t rows) {
    return Span{r.name, r.p, r.ld * 2, (int64_t)r.heads * LAYA_HEAD_DIM * 2, rows, r.written};
}

}  // namespace

extern "C" {

int laya_gpu_op_status(int32_t* status, void* stream) {
    if (!status) return fail(LAYA_ERR_ARG, "op_status: status is NULL");
    const Ptr ptrs[] = {{"status", status}};
    if (int rc = check_pointers("op_status", ptrs)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int32_t v = 0;
    cudaError_t e = cudaMemcpyAsync(&v, status, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(status, 0, 4, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return cuda_fail("op_status", e);
    if (v & ERR_WAIT_TIMEOUT) return fail(LAYA_ERR_TIMEOUT, "operator: a device-side wait ran out");
    if (v) return fail(LAYA_ERR_ARG, "operator: an offset table or an index failed a kernel's check");
    return LAYA_OK;
}

int laya_gpu_rope_plan(uint32_t head_dim, uint32_t rot_dim, double theta, int layout, double factor,
                       uint32_t original_len, double beta_fast, double beta_slow, float magnitude,
                       laya_rope_plan* plan) {
    if (!plan) return fail(LAYA_ERR_ARG, "rope_plan: plan is NULL");
    if (!head_dim || head_dim % 2 || head_dim > LAYA_ROPE_MAX_HEAD_DIM || !rot_dim || rot_dim % 2 ||
        rot_dim > head_dim)
        return fail(LAYA_ERR_ARG, "rope_plan: rot_dim %u of head_dim %u (even, at most %d)", rot_dim, head_dim,
                    LAYA_ROPE_MAX_HEAD_DIM);
    if (layout != LAYA_ROPE_HALF && layout != LAYA_ROPE_INTERLEAVED)
        return fail(LAYA_ERR_ARG, "rope_plan: layout %d", layout);
    if (!(theta > 1.0) || !std::isfinite(theta) || !(factor >= 1.0) || !std::isfinite(factor) ||
        !std::isfinite(magnitude))
        return fail(LAYA_ERR_ARG, "rope_plan: theta > 1, factor >= 1, all finite");
    if (original_len && (!(beta_slow >= 0.0) || !(beta_fast > beta_slow) || !std::isfinite(beta_fast)))
        return fail(LAYA_ERR_ARG, "rope_plan: beta_fast > beta_slow >= 0");
    *plan = laya_rope_plan{};
    plan->head_dim = head_dim;
    plan->rot_dim = rot_dim;
    plan->layout = layout;
    plan->magnitude = magnitude;
    const long double two_pi = 6.283185307179586476925286766559L;
    for (uint32_t i = 0; i < rot_dim / 2; i++) {
        long double f = powl((long double)theta, -2.0L * i / rot_dim);
        if (original_len) {
            const long double turns = original_len * f / two_pi;
            long double g = (turns - (long double)beta_slow) / ((long double)beta_fast - (long double)beta_slow);
            g = g < 0.0L ? 0.0L : g > 1.0L ? 1.0L : g;
            f *= g + (1.0L - g) / (long double)factor;
        } else {
            f /= (long double)factor;
        }
        // f <= 1 radian: under a sixth of a turn
        plan->turn[i] = (uint64_t)(f / two_pi * 18446744073709551616.0L + 0.5L);
    }
    return LAYA_OK;
}

int laya_gpu_rope(const laya_rope_plan* plan, const void* x, int64_t x_stride, void* y, int64_t y_stride,
                  uint32_t n_tokens, uint32_t heads, const int32_t* cu_seqlens, uint32_t n_seqs,
                  const int32_t* positions, int inverse, int elem_dtype, int32_t* status, void* stream) {
    if (!plan || !plan->rot_dim || plan->rot_dim > plan->head_dim || plan->head_dim > LAYA_ROPE_MAX_HEAD_DIM ||
        (plan->rot_dim | plan->head_dim) % 2 ||
        (plan->layout != LAYA_ROPE_HALF && plan->layout != LAYA_ROPE_INTERLEAVED))
        return fail(LAYA_ERR_ARG, "rope: the plan was not made by laya_gpu_rope_plan");
    if (elem_dtype != LAYA_DT_F32 && elem_dtype != LAYA_DT_BF16 && elem_dtype != LAYA_DT_F16)
        return fail(LAYA_ERR_DTYPE, "rope: elem_dtype %d", elem_dtype);
    if (n_tokens > MAX_ROWS || n_seqs > MAX_ROWS)
        return fail(LAYA_ERR_ARG, "rope: %u tokens, %u sequences (2^30 at most)", n_tokens, n_seqs);
    if (!positions == !cu_seqlens && n_tokens)
        return fail(LAYA_ERR_ARG, "rope: one of cu_seqlens and positions, not both");
    if (n_tokens == 0 || heads == 0 || (!positions && n_seqs == 0)) return LAYA_OK;
    if (!x || !y || !status) return fail(LAYA_ERR_ARG, "rope: NULL x, y or status");
    const int e = elem_size(elem_dtype);
    const int64_t width = (int64_t)heads * plan->head_dim;
    if (width > (int64_t)1 << 30) return fail(LAYA_ERR_ARG, "rope: %u heads of %u", heads, plan->head_dim);
    if (x_stride < width || y_stride < width || x_stride > (int64_t)1 << 31 || y_stride > (int64_t)1 << 31)
        return fail(LAYA_ERR_ARG, "rope: a stride is less than %u heads x %u", heads, plan->head_dim);
    if (x != y || x_stride != y_stride) {
        const Span s[] = {{"x", x, x_stride * e, width * e, n_tokens, false},
                          {"y", y, y_stride * e, width * e, n_tokens, true}};
        if (int rc = check_overlap("rope", s)) return rc;
    }
    const Ptr ptrs[] = {{"x", x, (unsigned)e}, {"y", y, (unsigned)e}, {"cu_seqlens", cu_seqlens}, {"positions", positions}, {"status", status}};
    if (int rc = check_pointers("rope", ptrs)) return rc;
    const bool vec = !(((uintptr_t)x | (uintptr_t)y | (uint64_t)(x_stride * e) | (uint64_t)(y_stride * e)) & 15);
    const cudaError_t err = launch_rope(*plan, x, x_stride, y, y_stride, (int)n_tokens, (int)heads, cu_seqlens,
                                        (int)n_seqs, positions, inverse != 0, elem_dtype, vec, status,
                                        static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? LAYA_OK : cuda_fail("rope", err);
}

int laya_gpu_attention(const laya_attention* a, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                       const void* v, int64_t v_stride, void* out, int64_t out_stride, float* lse, void* stream) {
    const char* op = "attention";
    if (int rc = check_attention(op, a)) return rc;
    if (a->n_tokens == 0 || a->n_seqs == 0) return LAYA_OK;
    const uint32_t hq = a->n_heads, hk = a->n_kv_heads;
    const Rows r[] = {{"q", q, q_stride, hq, false},
                      {"k", k, k_stride, hk, false},
                      {"v", v, v_stride, hk, false},
                      {"out", out, out_stride, hq, true}};
    for (const Rows& x : r)
        if (int rc = check_rows(op, x)) return rc;
    const uint64_t T = a->n_tokens;
    const Span s[] = {span(r[0], T), span(r[1], T), span(r[2], T), span(r[3], T),
                      {"lse", lse, (int64_t)T * 4, (int64_t)T * 4, hq, true}};
    if (int rc = check_overlap(op, s)) return rc;
    const Ptr ptrs[] = {{"q", q}, {"k", k}, {"v", v}, {"out", out}, {"lse", lse}, {"cu_seqlens", a->cu_seqlens},
                        {"token_mask", a->token_mask, 1}, {"status", a->status}};
    if (int rc = check_pointers(op, ptrs)) return rc;
    AttnIO io{};
    io.q = {const_cast<void*>(q), q_stride};
    io.k = {const_cast<void*>(k), k_stride};
    io.v = {const_cast<void*>(v), v_stride};
    io.out = {out, out_stride};
    io.lse = lse;
    const cudaError_t e = launch_attention_fwd(*a, io, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LAYA_OK : cuda_fail(op, e);
}

uint64_t laya_gpu_attention_backward_workspace(const laya_attention* a) {
    if (check_attention("attention_backward_workspace", a)) return 0;
    return a->n_tokens ? workspace_bytes_of(a) : 0;
}

int laya_gpu_attention_backward(const laya_attention* a, const void* q, int64_t q_stride, const void* k,
                                int64_t k_stride, const void* v, int64_t v_stride, const void* out,
                                int64_t out_stride, const float* lse, const void* dout, int64_t dout_stride, void* dq,
                                int64_t dq_stride, void* dk, int64_t dk_stride, void* dv, int64_t dv_stride,
                                void* workspace, uint64_t workspace_bytes, void* stream) {
    const char* op = "attention_backward";
    if (int rc = check_attention(op, a)) return rc;
    if (a->n_tokens == 0 || a->n_seqs == 0) return LAYA_OK;
    const uint32_t hq = a->n_heads, hk = a->n_kv_heads;
    const Rows r[] = {{"q", q, q_stride, hq, false},       {"k", k, k_stride, hk, false},
                      {"v", v, v_stride, hk, false},       {"out", out, out_stride, hq, false},
                      {"dout", dout, dout_stride, hq, false}, {"dq", dq, dq_stride, hq, true},
                      {"dk", dk, dk_stride, hk, true},     {"dv", dv, dv_stride, hk, true}};
    for (const Rows& x : r)
        if (int rc = check_rows(op, x)) return rc;
    if (!lse) return fail(LAYA_ERR_ARG, "%s: lse is NULL", op);
    const uint64_t need = workspace_bytes_of(a);
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need)
        return fail(LAYA_ERR_ARG, "%s: the workspace needs %llu bytes, 16-byte aligned", op,
                    (unsigned long long)need);
    const uint64_t T = a->n_tokens;
    const Span s[] = {span(r[0], T), span(r[1], T), span(r[2], T), span(r[3], T), span(r[4], T), span(r[5], T),
                      span(r[6], T), span(r[7], T),
                      {"lse", lse, (int64_t)T * 4, (int64_t)T * 4, hq, false},
                      {"workspace", workspace, (int64_t)need, (int64_t)need, 1, true}};
    if (int rc = check_overlap(op, s)) return rc;
    const Ptr ptrs[] = {{"q", q}, {"k", k}, {"v", v}, {"out", out}, {"lse", lse}, {"dout", dout}, {"dq", dq},
                        {"dk", dk}, {"dv", dv}, {"workspace", workspace}, {"cu_seqlens", a->cu_seqlens},
                        {"token_mask", a->token_mask, 1}, {"status", a->status}};
    if (int rc = check_pointers(op, ptrs)) return rc;
    AttnIO io{};
    io.q = {const_cast<void*>(q), q_stride};
    io.k = {const_cast<void*>(k), k_stride};
    io.v = {const_cast<void*>(v), v_stride};
    io.out = {const_cast<void*>(out), out_stride};
    io.dout = {const_cast<void*>(dout), dout_stride};
    io.dq = {dq, dq_stride};
    io.dk = {dk, dk_stride};
    io.dv = {dv, dv_stride};
    io.lse = const_cast<float*>(lse);
    io.tickets = static_cast<unsigned long long*>(workspace);
    io.delta = static_cast<float*>(workspace) + WORKSPACE_HEAD / sizeof(float);
    io.delta_short = io.delta + (uint64_t)hq * T;
    const cudaError_t e = launch_attention_bwd(*a, io, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? LAYA_OK : cuda_fail(op, e);
}

int laya_gpu_policy_loss(const laya_policy* p, const void* logits, const void* ref_logits, const int32_t* actions,
                         const float* advantages, const float* old_logp, const float* grad, float* loss, float* logp,
                         float* kl, float* entropy, void* dlogits, void* stream) {
    const char* op = "policy_loss";
    if (!p) return fail(LAYA_ERR_ARG, "%s: NULL description", op);
    if (p->elem_dtype != LAYA_DT_F32 && p->elem_dtype != LAYA_DT_BF16 && p->elem_dtype != LAYA_DT_F16)
        return fail(LAYA_ERR_DTYPE, "%s: elem_dtype %d", op, p->elem_dtype);
    if (p->n_decisions > MAX_ROWS || p->n_options > MAX_ROWS)
        return fail(LAYA_ERR_ARG, "%s: %u decisions, %u options (2^30 at most)", op, p->n_decisions, p->n_options);
    for (float t : p->temperature)
        if (!std::isfinite(t)) return fail(LAYA_ERR_ARG, "%s: temperature must be finite", op);
    if (!(p->clip_low >= 0.f && p->clip_low <= 1.f) || !(p->clip_high >= 0.f) || !std::isfinite(p->clip_high))
        return fail(LAYA_ERR_ARG, "%s: 0 <= clip_low <= 1, clip_high >= 0", op);
    if (!std::isfinite(p->kl_coef) || !std::isfinite(p->entropy_coef))
        return fail(LAYA_ERR_ARG, "%s: a coefficient is not finite", op);
    if (p->n_decisions == 0) return LAYA_OK;
    if (!p->cu_options || !p->status || !actions || !advantages || !old_logp || (p->n_options && !logits))
        return fail(LAYA_ERR_ARG, "%s: NULL input or status", op);
    const int e = elem_size(p->elem_dtype);
    const int64_t G = (int64_t)p->n_options * e, n = (int64_t)p->n_decisions * 4;
    const Span s[] = {{"logits", logits, G, G, G != 0, false}, {"ref_logits", ref_logits, G, G, G != 0, false},
                      {"actions", actions, n, n, 1, false},    {"advantages", advantages, n, n, 1, false},
                      {"old_logp", old_logp, n, n, 1, false},  {"grad", grad, n, n, 1, false},
                      {"loss", loss, n, n, 1, true},           {"logp", logp, n, n, 1, true},
                      {"kl", kl, n, n, 1, true},               {"entropy", entropy, n, n, 1, true},
                      {"dlogits", dlogits, G, G, G != 0, true}};
    if (int rc = check_overlap(op, s)) return rc;
    const unsigned el = (unsigned)e;
    const Ptr ptrs[] = {{"logits", logits, el}, {"ref_logits", ref_logits, el}, {"actions", actions},
                        {"advantages", advantages}, {"old_logp", old_logp}, {"grad", grad}, {"loss", loss},
                        {"logp", logp}, {"kl", kl}, {"entropy", entropy}, {"dlogits", dlogits, el},
                        {"cu_options", p->cu_options}, {"qtypes", p->qtypes}, {"status", p->status}};
    if (int rc = check_pointers(op, ptrs)) return rc;
    const PolicyIO io{logits, ref_logits, actions, advantages, old_logp, grad, loss, logp, kl, entropy, dlogits};
    const cudaError_t err = launch_policy(*p, io, static_cast<cudaStream_t>(stream));
    return err == cudaSuccess ? LAYA_OK : cuda_fail(op, err);
}

}  // extern "C"
