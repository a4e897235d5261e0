"""Definitions of the training-step operators in 64 bits (torch, any device)
and the error bounds their kernels are held to, for the operator tests."""
import math

import torch

DT = {"BF16": torch.bfloat16, "F16": torch.float16, "F32": torch.float32}
F32 = 2.0 ** -24  # half a step of f32, relative


def half_step(dtype):
    return torch.finfo(DT[dtype]).eps / 2


def tiny(dtype):
    """Half a step among the subnormals, absolute."""
    return torch.finfo(DT[dtype]).smallest_normal * torch.finfo(DT[dtype]).eps / 2


# ------------------------------------------------------------------ rotary

def rope_frequencies(rot_dim, theta=160000.0, factor=1.0, original_len=0, fast=32.0, slow=1.0):
    out = []
    for i in range(rot_dim // 2):
        f = theta ** (-2.0 * i / rot_dim)
        if original_len:
            g = min(1.0, max(0.0, (original_len * f / (2 * math.pi) - slow) / (fast - slow)))
            f *= g + (1 - g) / factor
        else:
            f /= factor
        out.append(f)
    return out


def rope(x, pos, freqs, layout="half", magnitude=1.0, inverse=False):
    """x [T][heads][head_dim] f64, pos [T]; the rotated heads."""
    r = 2 * len(freqs)
    a = pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64, device=x.device)
    z = torch.polar(torch.full_like(a, float(magnitude)), -a if inverse else a)[:, None, :]
    h = x[..., :r]
    if layout == "half":
        z = torch.complex(h[..., :r // 2].contiguous(), h[..., r // 2:].contiguous()) * z
        h = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(h.reshape(*h.shape[:-1], r // 2, 2).contiguous()) * z
        h = torch.view_as_real(z).reshape(h.shape)
    return torch.cat([h, x[..., r:]], -1)


# ------------------------------------------------------------------ attention

def attention(q, k, v, scale, window, pos, dout=None):
    """One sequence's present tokens: q [n][hq][64], k, v [n][hk][64] f64, pos
    [n] their places. Returns out, lse [n][hq], the gradients of
    sum(out * dout), and elementwise bounds on the kernels' error for 16-bit
    operands with half a step `u` (see attention_bounds)."""
    n, hq, _ = q.shape
    rep = hq // k.shape[1]
    q, k, v = (t.detach().clone().requires_grad_(dout is not None) for t in (q, k, v))
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = scale * torch.einsum("ihd,jhd->hij", q, kk)
    if window >= 0:
        s = s.masked_fill((pos[:, None] - pos[None, :]).abs() > window, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[..., None])
    out = torch.einsum("hij,jhd->ihd", p, vv)
    grads = None
    if dout is not None:
        grads = torch.autograd.grad(out, (q, k, v), dout)
    return out.detach(), lse.detach().t(), grads, p.detach()


def attention_bounds(q, k, v, scale, p, out, lse, u, t0, dout=None, grads=None):
    """Elementwise bounds on |kernel - definition|.

    Scores: 64 exact products summed in f32, so |ds| <= e_s = 80 * 2^-24 *
    scale * sum |q k| (80: the sum's steps, the scale and log2 e). Probability:
    exp of that, ex2.approx (2^-22), the row sum or, in the backward pass, the
    rounding of lse times log2 e: relative e_p = 2 e_s + 2^-20 + 2^-22 |lse|.
    The product operands P and dS are rounded to 16 bits (u relative, t0
    absolute among the subnormals), dS perhaps from the rounded P (so 2 u, and
    t0 times |dP - delta|), results once more. P enters the products
    after exp2 of a difference from the row's maximum or from lse; both are
    <= 1 (or below 2^8 with its own relative rounding), so t0 counts 256
    times at most. ex2.approx.ftz gives 0 below 2^-126: an absolute error of
    2^-126 = `flushed` for a probability, times |dP - delta| for dS."""
    rep = q.shape[1] // k.shape[1]
    kk, vv = k.repeat_interleave(rep, 1).abs(), v.repeat_interleave(rep, 1).abs()
    es = 80 * F32 * scale * torch.einsum("ihd,jhd->hij", q.abs(), kk)
    es = torch.where(p > 0, es, 0.0).amax(-1)  # [h][i]
    L = lse.t()
    ep = 2 * es + 2.0 ** -20 + 2.0 ** -22 * L.abs()
    b = {}
    b["lse"] = (es + 2.0 ** -21 * (1 + L.abs())).t()
    pv = torch.einsum("hij,jhd->ihd", p, vv)
    seen = (p > 0).double()
    b["out"] = (u + 2 * ep.t()[..., None]) * pv + u * out.abs() + 2 * t0 * (
        1 + torch.einsum("hij,jhd->ihd", seen, vv))
    if dout is None:
        return b
    gq, gk, gv = grads
    d_out = dout.abs()
    dp = torch.einsum("ihd,jhd->hij", dout, v.repeat_interleave(rep, 1))
    dp_abs = torch.einsum("ihd,jhd->hij", d_out, vv)
    delta = (dout * out).sum(-1).t()[..., None]
    # delta comes from the out the forward left, itself off by b["out"]
    e_delta = ((d_out * (b["out"] + 70 * F32 * out.abs())).sum(-1)).t()[..., None]
    e_ds = p * (ep[..., None] * (dp - delta).abs() + 70 * F32 * dp_abs + e_delta) + 2 * u * (p * (dp - delta)).abs()
    flushed = 2.0 ** -126
    e_ds = e_ds * (1 + 4 * u) + (t0 + (t0 + flushed) * (dp - delta).abs()) * seen

    def shared(x):  # sum over the heads that share a key head
        return x.reshape(x.shape[0], k.shape[1], rep, 64).sum(2)

    b["dq"] = scale * torch.einsum("hij,jhd->ihd", e_ds, kk) * 1.01 + u * gq.abs() + 2 * t0
    b["dk"] = scale * shared(torch.einsum("hij,ihd->jhd", e_ds, q.abs())) * 1.01 + u * gk.abs() + 2 * t0
    e_p = (u + ep[..., None]) * p + (t0 + flushed) * seen
    b["dv"] = shared(torch.einsum("hij,ihd->jhd", e_p, d_out)) * 1.01 + u * gv.abs() + 2 * t0
    return b


# ------------------------------------------------------------------ policy loss

def policy(z, zr, action, adv, old, t, lo, hi, klc, entc):
    """One decision: logits [K] f64 (requires_grad ok); -inf = ruled out."""
    alive = z > -math.inf
    lp = torch.log_softmax(torch.where(alive, z, -math.inf) / t, 0)
    lp = torch.where(alive, lp, 0.0)
    p = torch.where(alive, torch.exp(lp), 0.0)
    ent = -(p * lp).sum()
    kl = torch.zeros((), dtype=torch.float64)
    if zr is not None:
        lr = torch.where(alive, torch.log_softmax(zr / t, 0), 0.0)
        kl = (p * (lp - lr)).sum()
    logp = lp[action] if alive[action] else torch.tensor(-math.inf, dtype=torch.float64)
    r = torch.exp(logp - old)
    loss = torch.maximum(-r * adv, -torch.clamp(r, 1 - lo, 1 + hi) * adv) + klc * kl - entc * ent
    return loss, logp, kl, ent
