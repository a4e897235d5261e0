"""laya_gpu_rope against the rotation by complex numbers in 64 bits."""
import numpy as np
import pytest

import op_reference as ref

pytestmark = pytest.mark.gpu


def _bound(x, r, layout, u, t0, magnitude):
    """Per element: cos and sin off by at most 2^-22 (angle 2^-25 turns and
    sincospif's rounding, times magnitude), two products and a sum in f32, one
    rounding to the type: (u + 2^-20) of |a| + |b| covers all of it."""
    import torch
    pair = torch.zeros_like(x)
    h = x[..., :r].abs()
    if layout == "half":
        s = h[..., :r // 2] + h[..., r // 2:]
        pair[..., :r] = torch.cat([s, s], -1)
    else:
        pair[..., :r] = (h[..., 0::2] + h[..., 1::2]).repeat_interleave(2, -1)
    return (u + 2.0 ** -20) * magnitude * pair + t0


def _run(lens=None, positions=None, heads=3, hd=64, rot=64, layout="half", dtype="BF16", inverse=False, pad=8,
         in_place=False, shift=0, seed=0, **plan):
    import torch
    from laya_zig_b200 import gpu
    dt = ref.DT[dtype]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lead = 3
    T = (sum(lens) if lens is not None else len(positions)) + (2 * lead if lens is not None else 0)
    ld = heads * hd + pad
    store = torch.randn((T * ld + shift,), generator=g, device="cuda").to(dt)
    x = store[shift:].view(T, ld)
    x0 = x.clone()
    y = x if in_place else torch.full((T, heads * hd + 2 * pad), 7.0, dtype=dt, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    p = gpu.RopePlan(head_dim=hd, rot_dim=rot, layout=layout, **plan)
    if lens is not None:
        cu = torch.tensor([lead] + (np.cumsum(lens) + lead).tolist(), dtype=torch.int32, device="cuda")
        gpu.rope(p, x.data_ptr(), ld, y.data_ptr(), y.stride(0), T, heads, status.data_ptr(),
                 cu_seqlens_ptr=cu.data_ptr(), n_seqs=len(lens), inverse=inverse, dtype=dtype)
        pos = torch.cat([torch.arange(n) for n in lens]).cuda()
        rows = slice(lead, T - lead)
    else:
        pt = torch.tensor(positions, dtype=torch.int32, device="cuda")
        gpu.rope(p, x.data_ptr(), ld, y.data_ptr(), y.stride(0), T, heads, status.data_ptr(),
                 positions_ptr=pt.data_ptr(), inverse=inverse, dtype=dtype)
        pos, rows = pt, slice(0, T)
    gpu.op_status(status.data_ptr())
    f = ref.rope_frequencies(rot, plan.get("theta", 160000.0), plan.get("factor", 1.0), plan.get("original_len", 0),
                             plan.get("beta_fast", 32.0), plan.get("beta_slow", 1.0))
    mag = plan.get("magnitude", 1.0)
    xs = x0[rows][:, :heads * hd].double().reshape(-1, heads, hd)
    want = ref.rope(xs, pos, f, layout, mag, inverse)
    got = y[rows][:, :heads * hd].double().reshape(-1, heads, hd)
    b = _bound(xs, rot, layout, ref.half_step(dtype), ref.tiny(dtype), mag)
    assert ((got - want).abs() <= b).all()
    assert torch.equal(got[..., rot:], xs[..., rot:])
    # what belongs to no head or no sequence
    other = x0 if in_place else torch.full_like(y, 7.0)
    assert torch.equal(y[:, heads * hd:], other[:, heads * hd:])
    if lens is not None:
        for edge in (slice(0, lead), slice(T - lead, T)):
            assert torch.equal(y[edge], other[edge])
    if not in_place:
        assert torch.equal(x, x0)


@pytest.mark.parametrize("dtype", ["BF16", "F16", "F32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [64, 48, 32, 20, 2])
def test_layouts_and_parts(layout, rot, dtype):
    _run([1, 0, 64, 5, 130], layout=layout, rot=rot, dtype=dtype)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("kw", [dict(in_place=True), dict(inverse=True), dict(in_place=True, inverse=True, rot=32),
                                dict(pad=3, dtype="F32"), dict(pad=1), dict(shift=1), dict(heads=1, hd=128, rot=128),
                                dict(hd=256, rot=256, dtype="F32"), dict(heads=24), dict(hd=40, rot=24),
                                dict(magnitude=1.3), dict(magnitude=0.0)])
def test_forms(layout, kw):
    _run([17, 64, 1, 200], layout=layout, **kw)


@pytest.mark.parametrize("kw", [dict(factor=4.0), dict(factor=4.0, original_len=8192), dict(theta=1e6),
                                dict(factor=2.0, original_len=64, beta_fast=4.0, beta_slow=0.5, magnitude=1.07)])
def test_scaled(kw):
    _run([32768, 3], heads=2, dtype="F32", **kw)


@pytest.mark.parametrize("dtype", ["F32", "F16"])
def test_far_and_negative_positions(dtype):
    """Angles of far positions keep their accuracy. Against 64-bit angles,
    which at 2^31 radians are themselves off by 2^-22 (the bound's 2^-20 holds
    that)."""
    _run(positions=[0, 5, 5, -1, 32767, 131071, -70000, 1 << 20, (1 << 31) - 1, -(1 << 31), 3], heads=2, dtype=dtype)


def test_many_sequences():
    rng = np.random.default_rng(0)
    _run(rng.integers(0, 7, 3000).tolist(), heads=1)


def test_inverse_undoes():
    """Forward then inverse in f32 returns x within two roundings of the pair."""
    import torch
    from laya_zig_b200 import gpu
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = torch.randn((500, 128), generator=g, device="cuda")
    y = x.clone()
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 500], dtype=torch.int32, device="cuda")
    p = gpu.RopePlan(rot_dim=64)
    for inv in (False, True):
        gpu.rope(p, y.data_ptr(), 128, y.data_ptr(), 128, 500, 2, st.data_ptr(), cu_seqlens_ptr=cu.data_ptr(),
                 n_seqs=1, inverse=inv, dtype="F32")
    h = x.reshape(500, 2, 2, 32)
    bound = (2.0 ** -19 * (h[:, :, :1].abs() + h[:, :, 1:].abs())).expand_as(h).reshape(500, 128)
    assert ((x - y).abs() <= bound).all()


@pytest.mark.parametrize("table", [[0, 50, 40, 100], [-3, 20, 60, 100], [0, 30, 60, 500]])
def test_broken_offsets_are_recorded(table):
    import torch
    from laya_zig_b200 import gpu
    x = torch.zeros((100, 64), device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor(table, dtype=torch.int32, device="cuda")
    gpu.rope(gpu.RopePlan(), x.data_ptr(), 64, x.data_ptr(), 64, 100, 1, st.data_ptr(), cu_seqlens_ptr=cu.data_ptr(),
             n_seqs=3, dtype="F32")
    with pytest.raises(gpu.LayaError) as e:
        gpu.op_status(st.data_ptr())
    assert e.value.code == gpu.ERR_ARG


def test_captured_between_streams_that_join():
    """Behind a join of two streams in a captured graph, ahead of one and behind
    a copy: the kernel waits for all that comes before it, and what follows waits
    for the kernel."""
    import torch
    from laya_zig_b200 import gpu
    x = torch.randn((64, 2304), device="cuda").to(torch.bfloat16)
    y, z = torch.zeros_like(x), torch.zeros_like(x)
    cu = torch.tensor([0, 64], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    slow = torch.zeros(1 << 24, device="cuda")
    plan = gpu.RopePlan()
    s, other = torch.cuda.Stream(), torch.cuda.Stream()

    def rope():
        gpu.rope(plan, z.data_ptr(), 2304, y.data_ptr(), 2304, 64, 24, status.data_ptr(), cu_seqlens_ptr=cu.data_ptr(),
                 n_seqs=1, stream=s.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        z.copy_(x)
        rope()
    torch.cuda.synchronize()
    want = y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        other.wait_stream(s)
        with torch.cuda.stream(other):
            slow.add_(1)
            z.copy_(x)
        y.zero_()
        s.wait_stream(other)
        rope()
        first = y.clone()
        other.wait_stream(s)
        with torch.cuda.stream(other):
            slow.add_(1)
            z.zero_()
        s.wait_stream(other)
        rope()
        second = y.clone()
        z.copy_(x)
        rope()
    for _ in range(3):
        y.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(first, want) and (second[:, :24 * 64] == 0).all() and torch.equal(y, want)
    gpu.op_status(status.data_ptr())
