"""Whole numbers that do not fit the C interface are refused, not wrapped."""
import pytest

from laya_zig_b200 import gpu

A = 1 << 20  # an address that is never read


def _refused(f, *a, **kw):
    with pytest.raises(gpu.LayaError) as e:
        f(*a, **kw)
    return e.value.code == gpu.ERR_ARG


@pytest.mark.parametrize("kw", [dict(window=(1 << 32) + 5), dict(window=1 << 31), dict(window=-(1 << 31) - 1),
                                dict(n_tokens=1 << 32), dict(n_seqs=-1), dict(max_len=(1 << 32) + 60),
                                dict(n_heads=(1 << 32) + 12), dict(n_kv_heads=(1 << 33) + 12)])
def test_attention(kw):
    d = dict(cu_seqlens_ptr=A, n_seqs=2, n_tokens=100, max_len=60, n_heads=12, n_kv_heads=12, status_ptr=A)
    d.update(kw)
    assert _refused(gpu.AttentionShape, **d)


@pytest.mark.parametrize("kw", [dict(n_tokens=1 << 32), dict(heads=(1 << 32) + 2), dict(n_seqs=1 << 32), dict(n_tokens=-1)])
def test_rope(kw):
    d = dict(x_ptr=A, x_stride=768, y_ptr=A + (1 << 22), y_stride=768, n_tokens=10, heads=12, status_ptr=A,
             cu_seqlens_ptr=A, n_seqs=1)
    d.update(kw)
    assert _refused(gpu.rope, gpu.RopePlan(), **d)


@pytest.mark.parametrize("kw", [dict(head_dim=(1 << 32) + 64), dict(rot_dim=(1 << 32) + 32), dict(original_len=1 << 32),
                                dict(original_len=-1)])
def test_rope_plan(kw):
    assert _refused(gpu.RopePlan, **kw)


@pytest.mark.parametrize("kw", [dict(n_decisions=1 << 32), dict(n_options=(1 << 32) + 8), dict(max_options=-1)])
def test_policy(kw):
    d = dict(cu_options_ptr=A, n_decisions=8, n_options=64, max_options=8, status_ptr=A)
    d.update(kw)
    assert _refused(gpu.PolicyBatch, **d)


def test_the_ends_of_the_range_pass():
    gpu.AttentionShape(A, 2, 100, (1 << 32) - 1, 12, 12, A, window=(1 << 31) - 1)
    gpu.AttentionShape(A, 2, 100, 60, 12, 12, A, window=-(1 << 31))
    gpu.PolicyBatch(A, 8, 64, (1 << 32) - 1, A)
    gpu.RopePlan(original_len=(1 << 32) - 1)
