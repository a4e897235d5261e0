"""The training-step operators' host side and index arithmetic, without a
GPU: refused arguments, the rotary plan, and the block-to-tile search of
csrc/operators.cuh restated and checked on good and on broken offset tables
(every row an accepted tile names lies in the buffers)."""
import math
import random
from fractions import Fraction

import numpy as np
import pytest

from laya_zig_b200 import gpu

A = 1 << 20  # an address that is never read: what refuses the call comes first


def _shape(**kw):
    d = dict(cu_seqlens_ptr=A, n_seqs=2, n_tokens=100, max_len=60, n_heads=12, n_kv_heads=12, status_ptr=A)
    d.update(kw)
    return gpu.AttentionShape(**d)


def _fwd(shape, **kw):
    d = dict(q_ptr=A, q_stride=2304, k_ptr=A + 1536, k_stride=2304, v_ptr=A + 2 * 1536, v_stride=2304,
             out_ptr=A + (1 << 24), out_stride=768, lse_ptr=A + (1 << 25))
    d.update(kw)
    gpu.attention(shape, **d)


def _bwd(shape, **kw):
    far = A + (1 << 26)
    d = dict(q_ptr=A, q_stride=2304, k_ptr=A + 1536, k_stride=2304, v_ptr=A + 2 * 1536, v_stride=2304,
             out_ptr=A + (1 << 24), out_stride=768, lse_ptr=A + (1 << 25), dout_ptr=A + (1 << 23), dout_stride=768,
             dq_ptr=far, dq_stride=2304, dk_ptr=far + 1536, dk_stride=2304, dv_ptr=far + 2 * 1536, dv_stride=2304,
             workspace_ptr=A + (1 << 27), workspace_bytes=1 << 20)
    d.update(kw)
    gpu.attention_backward(shape, **d)


def _code(f, *a, **kw):
    with pytest.raises(gpu.LayaError) as e:
        f(*a, **kw)
    return e.value.code


@pytest.mark.parametrize("kw", [dict(n_heads=0), dict(n_kv_heads=0), dict(n_heads=12, n_kv_heads=5),
                                dict(n_heads=70000, n_kv_heads=1), dict(scale=0.0), dict(scale=-1.0),
                                dict(scale=math.inf), dict(scale=math.nan), dict(scale=3e38),
                                dict(cu_seqlens_ptr=A + 2), dict(status_ptr=A + 1), dict(n_tokens=(1 << 30) + 1), dict(n_tokens=1 << 30),
                                dict(cu_seqlens_ptr=0), dict(status_ptr=0)])
def test_attention_refuses_shapes(kw):
    assert _code(_fwd, _shape(**kw)) == gpu.ERR_ARG
    assert _code(_bwd, _shape(**kw)) == gpu.ERR_ARG


def test_attention_refuses_f32():
    assert _code(_fwd, _shape(dtype="F32")) == gpu.ERR_DTYPE
    assert _code(gpu.attention_backward_workspace, _shape(dtype="F32")) == gpu.ERR_ARG


@pytest.mark.parametrize("kw", [dict(q_ptr=0), dict(k_ptr=0), dict(v_ptr=0), dict(out_ptr=0), dict(q_ptr=A + 8),
                                dict(q_stride=760), dict(k_stride=2300), dict(out_stride=769),
                                dict(out_ptr=A), dict(out_ptr=A + 2 * 1536, out_stride=2304), dict(lse_ptr=A + 4096),
                                dict(out_ptr=A + 2 * 1536 + 16, out_stride=2304), dict(lse_ptr=A + (1 << 25) + 2)])
def test_attention_refuses_rows(kw):
    assert _code(_fwd, _shape(), **kw) == gpu.ERR_ARG


@pytest.mark.parametrize("kw", [dict(lse_ptr=0), dict(dout_ptr=0), dict(dq_ptr=0), dict(dk_ptr=0), dict(dv_ptr=0),
                                dict(workspace_ptr=0), dict(workspace_bytes=12 * 100 * 4 - 1),
                                dict(workspace_ptr=A + (1 << 27) + 8), dict(dq_ptr=A), dict(dk_ptr=A + 1536),
                                dict(dv_ptr=A + (1 << 26) + 1536), dict(dq_ptr=A + (1 << 23), dq_stride=768),
                                dict(workspace_ptr=A + (1 << 25)), dict(dout_stride=800 + 4)])
def test_attention_backward_refuses(kw):
    assert _code(_bwd, _shape(), **kw) == gpu.ERR_ARG


def test_columns_of_one_packed_array_do_not_overlap():
    """q, k, v and, behind them, out in one row array: accepted as far as the
    host can tell (this host has no GPU, or the address is no device memory)."""
    code = _code(_fwd, _shape(), q_stride=3080, k_stride=3080, v_stride=3080, out_ptr=A + 4608,
                 out_stride=3080)
    import torch
    assert code == (gpu.ERR_ARG if torch.cuda.is_available() else gpu.ERR_NODEV)


def test_nothing_to_do():
    _fwd(_shape(n_tokens=0))
    _fwd(_shape(n_seqs=0))
    _bwd(_shape(n_seqs=0))
    assert gpu.attention_backward_workspace(_shape(n_tokens=0)) == 0
    assert gpu.attention_backward_workspace(_shape()) >= 12 * 100 * 4
    gpu.rope(gpu.RopePlan(), 0, 768, 0, 768, 0, 12, 0, cu_seqlens_ptr=A, n_seqs=1)
    gpu.policy_loss(gpu.PolicyBatch(0, 0, 0, 0, 0), 0, 0, 0, 0, 0)


@pytest.mark.parametrize("kw", [dict(head_dim=0), dict(head_dim=63, rot_dim=32), dict(head_dim=258), dict(rot_dim=66),
                                dict(rot_dim=0), dict(rot_dim=31), dict(theta=1.0), dict(theta=math.nan),
                                dict(factor=0.5), dict(factor=math.inf), dict(magnitude=math.inf),
                                dict(layout="other"), dict(original_len=8, beta_fast=1.0, beta_slow=1.0),
                                dict(original_len=8, beta_slow=-1.0)])
def test_rope_plan_refuses(kw):
    assert _code(gpu.RopePlan, **kw) == gpu.ERR_ARG


@pytest.mark.parametrize("kw", [dict(x_ptr=0), dict(y_ptr=0), dict(status_ptr=0), dict(x_stride=767),
                                dict(y_stride=700), dict(cu_seqlens_ptr=0), dict(positions_ptr=A),
                                dict(y_ptr=A + 2), dict(x_ptr=A + 1), dict(y_ptr=A, y_stride=776)])
def test_rope_refuses(kw):
    d = dict(x_ptr=A, x_stride=768, y_ptr=A + (1 << 22), y_stride=768, n_tokens=10, heads=12, status_ptr=A,
             cu_seqlens_ptr=A, n_seqs=1)
    d.update(kw)
    assert _code(gpu.rope, gpu.RopePlan(), **d) == gpu.ERR_ARG


@pytest.mark.parametrize("kw,args", [(dict(clip_low=-0.1), {}), (dict(clip_low=1.5), {}), (dict(clip_high=-1.0), {}),
                                     (dict(clip_high=math.inf), {}), (dict(kl_coef=math.nan), {}),
                                     (dict(entropy_coef=math.inf), {}), (dict(temperature=(1.0, math.nan, 1.0)), {}),
                                     (dict(cu_options_ptr=0), {}), (dict(status_ptr=0), {}),
                                     ({}, dict(logits_ptr=0)), ({}, dict(actions_ptr=0)), ({}, dict(advantages_ptr=0)),
                                     ({}, dict(old_logp_ptr=0)), ({}, dict(dlogits_ptr=A)),
                                     ({}, dict(dlogits_ptr=A + 4)), ({}, dict(logits_ptr=A + 2)),
                                     ({}, dict(loss_ptr=A + 8192)), ({}, dict(actions_ptr=A + 8194)), ({}, dict(kl_ptr=A + (1 << 18) + 1)),
                                     (dict(cu_options_ptr=A + 1), {}), (dict(qtypes_ptr=A + 2), {}), ({}, dict(kl_ptr=A + (1 << 16)))])
def test_policy_refuses(kw, args):
    b = dict(cu_options_ptr=A, n_decisions=8, n_options=64, max_options=8, status_ptr=A)
    b.update(kw)
    d = dict(logits_ptr=A, ref_logits_ptr=A + 4096, actions_ptr=A + 8192, advantages_ptr=A + 12288,
             old_logp_ptr=A + 16384, loss_ptr=A + (1 << 16), dlogits_ptr=A + (1 << 17))
    d.update(args)
    assert _code(gpu.policy_loss, gpu.PolicyBatch(**b), **d) == gpu.ERR_ARG


def test_status_word_refused():
    assert _code(gpu.op_status, 0) == gpu.ERR_ARG


# ------------------------------------------------------------------ rotary plan

@pytest.mark.parametrize("kw", [dict(), dict(rot_dim=32), dict(theta=10000.0, factor=4.0),
                                dict(factor=4.0, original_len=8192), dict(head_dim=256, theta=1e6),
                                dict(factor=8.0, original_len=512, beta_fast=16.0, beta_slow=2.0)])
def test_plan_turns(kw):
    """turn[i] against the frequency's definition in exact fractions of 64-bit
    arithmetic: what is left is the 64-bit floating error of this side,
    2^-50 of the frequency, which at position 2^20 is 2^-30 turns."""
    p = gpu.RopePlan(**kw)
    d = kw.get("rot_dim") or kw.get("head_dim", 64)
    theta, factor = kw.get("theta", 160000.0), kw.get("factor", 1.0)
    for i in range(d // 2):
        f = theta ** (-2.0 * i / d)
        if kw.get("original_len"):
            hi, lo = kw.get("beta_fast", 32.0), kw.get("beta_slow", 1.0)
            g = min(1.0, max(0.0, (kw["original_len"] * f / (2 * math.pi) - lo) / (hi - lo)))
            f = f * (g + (1 - g) / factor)
        else:
            f /= factor
        got = Fraction(p.c.turn[i], 1 << 64)
        want = Fraction(f) / Fraction(2 * math.pi)
        assert abs(got - want) <= want * Fraction(1, 1 << 46) + Fraction(1, 1 << 63), i
    assert all(p.c.turn[i] == 0 for i in range(d // 2, 128))


def test_fixed_point_angle():
    """pos * turn modulo 2^64, top 32 bits as a signed f32 of half turns
    (csrc/rope.cu), against the angle in 64 bits, at positions of either sign
    out to the ends of 32 bits: the f32 fraction is off by 2^-25 half turns at
    most and the 32-bit cut by 2^-31, the 64-bit comparison by pos * 2^-52."""
    p = gpu.RopePlan()
    for pos in [0, 1, -1, 2, 7, 8191, 32767, -32768, 1 << 20, (1 << 31) - 1, -(1 << 31)]:
        for i in range(32):
            t = (pos * p.c.turn[i]) & ((1 << 64) - 1)
            hi = t >> 32
            frac = np.float32(hi - (1 << 32) if hi >= 1 << 31 else hi) * np.float32(2.0 ** -31)
            exact = Fraction(pos) * Fraction(p.c.turn[i], 1 << 63)  # half turns
            d = (Fraction(float(frac)) - exact + 1) % 2 - 1
            assert abs(d) <= Fraction(1, 1 << 25) + Fraction(1, 1 << 30)


# ------------------------------------------------------------------ block -> tile

def warp_search(n, key, x):
    lo, first = 0, True
    while n > 1 or first:
        step = (n + 31) // 32
        le = [lane * step < n and key(lo + lane * step) <= x for lane in range(32)]
        c = sum(le)
        if c == 0:
            return -1 if first else lo
        lo += (c - 1) * step
        n = min(step, n - (c - 1) * step)
        first = False
    return lo


def find_tile(cu, n_seqs, n_tokens, max_len, rows, x):
    s = warp_search(n_seqs, lambda i: max(cu[i], 0) // rows + i, x)
    if s < 0:
        return None
    start, end = cu[s], cu[s + 1]
    if not (start >= 0 and end >= start and end <= n_tokens and end - start <= max_len):
        return None
    tile = x - (start // rows + s)
    if tile < 0 or tile * rows >= end - start:
        return None
    return s, start, end - start, tile * rows


def walk_find(cu, n_seqs, n_tokens, max_len, rows, x):
    """The search of csrc/attention_op_tc.cu's Walk: the first round's keys
    kept, the second round's entries handed among the lanes."""
    if n_seqs > 1024:
        return find_tile(cu, n_seqs, n_tokens, max_len, rows, x)

    def key(start, s):
        return max(start, 0) // rows + s
    step = (n_seqs + 31) // 32
    c = sum(lane * step < n_seqs and key(cu[lane * step], lane * step) <= x for lane in range(32))
    if c == 0:
        return None
    lo = (c - 1) * step
    m = min(step, n_seqs - lo)
    at = [cu[min(lo + lane, n_seqs)] for lane in range(32)]
    c1 = sum(lane < m and key(at[lane], lo + lane) <= x for lane in range(32))
    if c1 == 0:
        return None
    s = lo + c1 - 1
    start, end = at[c1 - 1], at[c1] if c1 < 32 else cu[s + 1]
    if not (start >= 0 and end >= start and end <= n_tokens and end - start <= max_len):
        return None
    tile = x - key(start, s)
    if tile < 0 or tile * rows >= end - start:
        return None
    return s, start, end - start, tile * rows


@pytest.mark.parametrize("find", [find_tile, walk_find])
@pytest.mark.parametrize("rows", [64, 128, 256])
@pytest.mark.parametrize("seed", range(12))
def test_every_tile_has_one_block(rows, seed, find):
    r = random.Random(seed * 7 + rows)
    n = r.choice([1, 2, 31, 32, 33, 64, 200, 1023, 1024, 1025])
    lens = [r.choice([0, 1, rows - 1, rows, rows + 1, r.randint(0, 700)]) for _ in range(n)]
    cu = [r.choice([0, 5, 300])]
    for v in lens:
        cu.append(cu[-1] + v)
    T = cu[-1] + r.choice([0, 17])
    want = {(s, row0) for s, v in enumerate(lens) for row0 in range(0, v, rows)}
    got = [find(cu, n, T, max(lens), rows, x) for x in range(T // rows + n)]
    got = [(g[0], g[3]) for g in got if g]
    assert len(got) == len(set(got)) and set(got) == want


@pytest.mark.parametrize("seed", range(12))
def test_no_tile_lies_past_the_slots_in_use(seed):
    """Walk::slots: a table that ends in unused entries is not walked to its
    end, and nothing before them is left out."""
    r, rows = random.Random(seed), 128
    n = r.choice([0, 1, 2, 31, 33, 200, 1024])
    cu = [r.choice([0, 5, 300])]
    for _ in range(n):
        cu.append(cu[-1] + r.choice([0, 1, rows - 1, rows, rows + 1, r.randint(0, 700)]))
    used, T = max([s + 1 for s in range(n) if cu[s] < cu[n]], default=0), cu[-1] + r.choice([0, 17, 5000])
    cu += [cu[-1]] * r.choice([1, 3, 900])
    n = len(cu) - 1
    end = cu[n] // rows + warp_search(n, lambda i: cu[i], cu[n] - 1) + 1
    assert end == cu[n] // rows + used
    assert not any(walk_find(cu, n, T, 700, rows, x) for x in range(end, T // rows + n))


@pytest.mark.parametrize("find,rows", [(find_tile, 64), (walk_find, 128)])
@pytest.mark.parametrize("seed", range(30))
def test_broken_tables_name_no_row_outside(seed, find, rows):
    """Unsorted, negative and overlong entries: an accepted tile's rows stay
    inside [0, n_tokens)."""
    r = random.Random(seed)
    n, T = r.choice([1, 5, 40, 300]), 1000
    cu = [r.randint(-50, 1100) for _ in range(n + 1)]
    if r.random() < 0.5:
        cu.sort()
    for x in range(T // rows + n):
        g = find(cu, n, T, 400, rows, x)
        if g:
            s, start, L, row0 = g
            assert 0 <= s < n and 0 <= start and start + L <= T and 0 <= row0 < L <= 400
    for t in range(T):  # rope's search: token -> sequence
        s = warp_search(n, lambda i: cu[i], t)
        assert -1 <= s < n
