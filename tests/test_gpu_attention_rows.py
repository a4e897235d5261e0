"""Gradients of the attention operator row by row, with bounds as tight as its
roundings: rows that see few keys, alone and beside long sequences."""
import math

import numpy as np
import pytest

import op_reference as ref
from test_gpu_attention_op import LONG, POISON, Problem

pytestmark = pytest.mark.gpu

# Delta from P dP: rows of sequences of 32 tokens at most, of windows of 4 at most, and
# rows that see 5 keys at most.
SHORT, NARROW, FEW = 32, 4, 5


def bounds(p, q, k, v, scale, out, lse, prob, u, t0, dout, grads):
    """Elementwise bounds on dq, dk, dv, by counting roundings.

    Scores, probabilities and out as in op_reference.attention_bounds. dP: 64
    products summed in f32, 70 * 2^-24 of sum |dO V|. delta: for rows of short
    sequences or with few keys the f32 sum of P dP over at most 32 keys (40
    roundings of it), so off by what its terms are off; else the sum of dO and
    the 16-bit out, off by what out is off. dS = P (dP - delta) in f32, rounded
    once to 16 bits (u, and t0 among the subnormals); the products' sums in f32
    (a rounding each); the result's own rounding."""
    import torch
    hq, hk = q.shape[1], k.shape[1]
    rep, n = hq // hk, q.shape[0]
    F = ref.F32
    kk, vv = k.repeat_interleave(rep, 1).abs(), v.repeat_interleave(rep, 1).abs()
    es = 80 * F * scale * torch.einsum("ihd,jhd->hij", q.abs(), kk)
    seen = (prob > 0).double()
    es = (es * seen).amax(-1)
    ep = (2 * es + 2.0 ** -20 + 2.0 ** -22 * lse.t().abs())[..., None]
    d_out, flushed = dout.abs(), 2.0 ** -126
    dp = torch.einsum("ihd,jhd->hij", dout, v.repeat_interleave(rep, 1))
    dp_abs = torch.einsum("ihd,jhd->hij", d_out, vv)
    delta = (dout * out).sum(-1).t()[..., None]
    b_out = ref.attention_bounds(q, k, v, scale, prob, out, lse, u, t0)["out"]
    from_out = (d_out * (b_out + 70 * F * out.abs())).sum(-1).t()[..., None]
    from_keys = (prob * (ep * dp.abs() + 70 * F * dp_abs + 40 * F * dp.abs()) + flushed * seen * dp.abs()).sum(
        -1, keepdim=True)
    few = (seen.sum(-1, keepdim=True) <= FEW) | (p.length <= SHORT) | (0 <= p.window <= NARROW)
    e_delta = torch.where(few, from_keys, from_out)
    ds = (prob * (dp - delta)).abs()
    e_ds = prob * (ep * (dp - delta).abs() + 70 * F * dp_abs + e_delta) + flushed * seen * (dp - delta).abs()
    e_ds = e_ds * (1 + u) + u * ds + t0 * seen
    sums = (n * rep + 20) * F

    def shared(x):
        return x.reshape(n, hk, rep, 64).sum(2)

    gq, gk, gv = grads
    total = e_ds + sums * ds
    e_p = (u + ep * (1 + u) + sums) * prob + (t0 + flushed) * seen
    return {"dq": scale * torch.einsum("hij,jhd->ihd", total, kk) * (1 + u) + (u + 2 * F) * gq.abs() + t0,
            "dk": scale * shared(torch.einsum("hij,ihd->jhd", total, q.abs())) * (1 + u) + (u + 2 * F) * gk.abs() + t0,
            "dv": shared(torch.einsum("hij,ihd->jhd", e_p, d_out)) * (1 + u) + (u + 2 * F) * gv.abs() + t0}


class Sequence:
    def __init__(self, length, window):
        self.length, self.window = length, window


def check(p):
    """Every sequence's gradients within the bounds."""
    import torch
    from laya_zig_b200 import gpu
    gpu.op_status(p.status.data_ptr())
    hq, hk = p.hq, p.hk
    u, t0 = ref.half_step(p.dtype), ref.tiny(p.dtype)
    start, worst = POISON, {}
    for n in p.lens:
        rows = torch.arange(start, start + n, device="cuda")
        start += n
        rows = rows[p.here[rows]]
        m = rows.numel()
        if m == 0:
            continue
        W = (hq + 2 * hk) * 64
        x = p.qkv[rows][:, :W].double().reshape(m, hq + 2 * hk, 64)
        q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
        do = p.dout[rows][:, :hq * 64].double().reshape(m, hq, 64)
        out, lse, grads, prob = ref.attention(q, k, v, p.scale, p.window, rows, do)
        b = bounds(Sequence(n, p.window), q, k, v, p.scale, out, lse, prob, u, t0, do, grads)
        dx = p.dqkv[rows][:, :W].double().reshape(m, hq + 2 * hk, 64)
        got = {"dq": dx[:, :hq], "dk": dx[:, hq:hq + hk], "dv": dx[:, hq + hk:]}
        for name, want in zip(("dq", "dk", "dv"), grads):
            worst[name] = max(worst.get(name, 0.0), ((got[name] - want).abs() / b[name]).max().item())
    for name, off in worst.items():
        assert off <= 1.0, (name, off)


MIXED = [2] * 30 + [1, 180, 3, 9, 10, 31, 32, 33, 2, 64, 65]
kernels = pytest.mark.parametrize("max_len", [None, LONG], ids=["small", "large"])


@kernels
@pytest.mark.parametrize("dtype", ["BF16", "F16"])
@pytest.mark.parametrize("hq,hk", [(3, 3), (4, 2)])
@pytest.mark.parametrize("lens", [[2] * 20, [31, 5], MIXED, [300, 2, 200]], ids=["pairs", "short", "mixed", "long"])
def test_short_sequences_beside_long_ones(lens, hq, hk, dtype, max_len):
    p = Problem(lens, hq=hq, hk=hk, dtype=dtype, max_len=max_len)
    p.run()
    check(p)
    p.check()


@kernels
@pytest.mark.parametrize("window", [0, 1, 4, 5, 8, 9, 40])
def test_rows_near_an_end_of_a_window(window, max_len):
    p = Problem(MIXED + [300], hq=2, hk=1, window=window, max_len=max_len)
    p.run()
    check(p)
    p.check()


def _sparse(step, dense_from):
    def f(n):
        i = np.arange(n)
        return ((i % step == 3) | (i >= dense_from)).astype(np.uint8)
    return f


@kernels
@pytest.mark.parametrize("window", [-1, 70, 6])
@pytest.mark.parametrize("step", [40, 61, 97])
def test_long_sequences_with_few_tokens_left(step, window, max_len):
    """300 tokens of which 8, 5 or 4 are there, beside others that are whole."""
    p = Problem([300, 40, 200], hq=4, hk=2, window=window, mask=_sparse(step, 300), max_len=max_len)
    p.run()
    check(p)
    p.check()


@pytest.mark.parametrize("hq", [1, 5, 40, 130])
def test_heads_that_no_block_ends_with(hq):
    """Delta's blocks take 128 (token, head) pairs: a token's heads in two of
    them, many tokens in one."""
    p = Problem([3, 150, 1, 20], hq=hq, hk=1, max_len=LONG)
    p.run()
    check(p)
    p.check()


def test_one_bound_for_all_batches():
    """The same two-token sequences alone and behind a long one."""
    import torch
    a = Problem([2] * 16, hq=2, hk=2, seed=3)
    b = Problem([180] + [2] * 16, hq=2, hk=2, seed=4)
    b.qkv[POISON + 180:POISON + 212] = a.qkv[POISON:POISON + 32]
    b.dout[POISON + 180:POISON + 212] = a.dout[POISON:POISON + 32]
    for p in (a, b):
        p.run()
        check(p)
    # dS and its rounding are the same but for the order of f32 sums
    x = a.dqkv[POISON:POISON + 32, :384].double()
    y = b.dqkv[POISON + 180:POISON + 212, :384].double()
    assert ((x - y).norm() / x.norm()).item() <= 2.0 ** -9 * 2
    assert math.isfinite(x.sum().item()) and torch.isfinite(y).all()
