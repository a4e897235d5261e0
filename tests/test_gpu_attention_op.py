"""laya_gpu_attention and laya_gpu_attention_backward against the definition
in 64 bits (op_reference.py), within elementwise bounds that count the 16-bit
roundings of the operands and results."""
import math

import numpy as np
import pytest

import op_reference as ref

pytestmark = pytest.mark.gpu

POISON = 4  # rows of NaN before the first and behind the last sequence

# Short sequences and few tokens go to one set of kernels, the rest to another;
# a longest length that no sequence reaches asks for the second.
LONG = 5000
kernels = pytest.mark.parametrize("max_len", [None, LONG], ids=["small", "large"])


class Problem:
    """Packed rows with columns to spare, NaN wherever no present token is."""

    def __init__(self, lens, hq=2, hk=2, window=-1, dtype="BF16", mask=None, seed=0, scale=0.125, pad=8, spread=1.0,
                 max_len=None):
        import torch
        from laya_zig_b200 import gpu
        self.lens, self.hq, self.hk, self.window, self.dtype, self.scale = lens, hq, hk, window, dtype, scale
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        dt = ref.DT[dtype]
        T = sum(lens) + 2 * POISON
        self.T = T
        self.ld = (hq + 2 * hk) * 64 + pad
        self.cu = torch.tensor([POISON] + (np.cumsum(lens) + POISON).tolist(), dtype=torch.int32, device="cuda")
        self.here = torch.zeros(T, dtype=torch.bool, device="cuda")
        self.here[POISON:T - POISON] = True
        self.mask = None
        if mask is not None:
            m = torch.ones(T, dtype=torch.uint8, device="cuda")
            m[POISON:T - POISON] = torch.as_tensor(mask(sum(lens)), dtype=torch.uint8, device="cuda")
            self.mask, self.here = m, self.here & (m != 0)
        self.qkv = (spread * torch.randn((T, self.ld), generator=g, device="cuda")).to(dt)
        self.dout = torch.randn((T, hq * 64 + pad), generator=g, device="cuda").to(dt)
        self.qkv[~self.here] = math.nan
        self.dout[~self.here] = math.nan
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.shape = gpu.AttentionShape(self.cu.data_ptr(), len(lens), T, max_len or max(lens), hq, hk,
                                        self.status.data_ptr(), window=window, scale=scale, dtype=dtype,
                                        token_mask_ptr=0 if self.mask is None else self.mask.data_ptr())
        self.buffers()

    def buffers(self):
        import torch
        from laya_zig_b200 import gpu
        dt = ref.DT[self.dtype]
        self.out = torch.full((self.T, self.hq * 64 + 16), 7.0, dtype=dt, device="cuda")
        self.lse = torch.full((self.hq, self.T), 7.0, dtype=torch.float32, device="cuda")
        self.dqkv = torch.full((self.T, self.ld), 7.0, dtype=dt, device="cuda")
        self.ws = torch.full((gpu.attention_backward_workspace(self.shape),), 255, dtype=torch.uint8, device="cuda")

    def forward(self, stream=0):
        from laya_zig_b200 import gpu
        e, q = 2, self.qkv.data_ptr()
        self.q3 = (q, q + self.hq * 64 * e, q + (self.hq + self.hk) * 64 * e)
        gpu.attention(self.shape, self.q3[0], self.ld, self.q3[1], self.ld, self.q3[2], self.ld, self.out.data_ptr(),
                      self.out.stride(0), self.lse.data_ptr(), stream)

    def backward(self, stream=0):
        from laya_zig_b200 import gpu
        d = self.dqkv.data_ptr()
        gpu.attention_backward(self.shape, self.q3[0], self.ld, self.q3[1], self.ld, self.q3[2], self.ld,
                               self.out.data_ptr(), self.out.stride(0), self.lse.data_ptr(), self.dout.data_ptr(),
                               self.dout.stride(0), d, self.ld, d + self.hq * 128, self.ld,
                               d + (self.hq + self.hk) * 128, self.ld, self.ws.data_ptr(), self.ws.numel(), stream)

    def run(self, stream=0):
        self.forward(stream)
        self.backward(stream)

    def check(self):
        import torch
        from laya_zig_b200 import gpu
        gpu.op_status(self.status.data_ptr())
        hq, hk = self.hq, self.hk
        u, t0 = ref.half_step(self.dtype), ref.tiny(self.dtype)
        W = (hq + 2 * hk) * 64
        start = POISON
        worst = {}
        for n in self.lens:
            rows = torch.arange(start, start + n, device="cuda")
            start += n
            there = self.here[rows]
            gone = rows[~there]
            # absent tokens
            assert (self.out[gone][:, :hq * 64] == 0).all() and (self.lse[:, gone] == -math.inf).all()
            assert (self.dqkv[gone][:, :W] == 0).all()
            rows = rows[there]
            m = rows.numel()
            if m == 0:
                continue
            x = self.qkv[rows][:, :W].double().reshape(m, hq + 2 * hk, 64)
            q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
            do = self.dout[rows][:, :hq * 64].double().reshape(m, hq, 64)
            out, lse, grads, p = ref.attention(q, k, v, self.scale, self.window, rows, do)
            b = ref.attention_bounds(q, k, v, self.scale, p, out, lse, u, t0, do, grads)
            dx = self.dqkv[rows][:, :W].double().reshape(m, hq + 2 * hk, 64)
            got = {"out": self.out[rows][:, :hq * 64].double().reshape(m, hq, 64), "lse": self.lse[:, rows].t().double(),
                   "dq": dx[:, :hq], "dk": dx[:, hq:hq + hk], "dv": dx[:, hq + hk:]}
            want = {"out": out, "lse": lse, "dq": grads[0], "dk": grads[1], "dv": grads[2]}
            for name in got:
                off = ((got[name] - want[name]).abs() / b[name]).max().item()
                worst[name] = max(worst.get(name, 0.0), off)
        for name, off in worst.items():
            assert off <= 1.0, (name, off)  # NaN fails too
        # rows of no sequence, and the columns between rows, are as they were
        edge = torch.ones(self.T, dtype=torch.bool, device="cuda")
        edge[POISON:self.T - POISON] = False
        for t in (self.out, self.dqkv):
            assert (t[edge] == 7).all()
        assert (self.out[:, hq * 64:] == 7).all() and (self.dqkv[:, W:] == 7).all()
        assert (self.lse[:, edge] == 7).all()


LENGTHS = {"one": [1], "tile": [64], "tile+1": [65], "edges": [1, 63, 64, 65, 0, 2, 127, 128, 129, 0, 191, 193],
           "batch": [175, 176, 180, 178], "long": [700, 33]}


@pytest.mark.parametrize("dtype", ["BF16", "F16"])
@pytest.mark.parametrize("window", [-1, 0, 1, 64, 1000])
@pytest.mark.parametrize("lens", list(LENGTHS))
@kernels
def test_lengths_and_windows(lens, window, dtype, max_len):
    p = Problem(LENGTHS[lens], window=window, dtype=dtype, max_len=max_len)
    p.run()
    p.check()


@pytest.mark.parametrize("hq,hk", [(1, 1), (3, 1), (6, 2), (12, 12), (12, 4)])
@pytest.mark.parametrize("window", [-1, 17, 3])
@kernels
def test_head_groups(hq, hk, window, max_len):
    p = Problem([70, 129], hq=hq, hk=hk, window=window, seed=hq, max_len=max_len)
    p.run()
    p.check()


def _every(step):
    return lambda n: (np.arange(n) % step != 0).astype(np.uint8)


def _only(*kept):
    def f(n):
        m = np.zeros(n, np.uint8)
        m[[i for i in kept if i < n]] = 3
        return m
    return f


@pytest.mark.parametrize("dtype", ["BF16", "F16"])
@pytest.mark.parametrize("mask", [_every(2), _every(3), _only(), _only(0), _only(130, 131), _only(63, 64, 200)],
                         ids=["half", "third", "none", "first", "tile2", "across"])
@pytest.mark.parametrize("window", [-1, 5])
@kernels
def test_absent_tokens(mask, window, dtype, max_len):
    """NaN in every absent token's rows; sequences with no token left."""
    p = Problem([66, 1, 190, 64], window=window, mask=mask, dtype=dtype, hq=2, hk=1, max_len=max_len)
    p.run()
    p.check()


@kernels
def test_large_scores(max_len):
    """Scores of some hundreds: rows that put all weight on one key, and keys
    no query gives any."""
    p = Problem([200, 31], spread=8.0, dtype="BF16", scale=0.5, max_len=max_len)
    p.run()
    p.check()


@kernels
def test_scale_and_padded_rows(max_len):
    p = Problem([130], scale=0.7, pad=64, dtype="F16", hq=4, hk=2, max_len=max_len)
    p.run()
    p.check()


@kernels
@pytest.mark.parametrize("n", [700, 1500])
def test_many_short_sequences(n, max_len):
    """More than 1,024 of them: the search for a tile takes another round."""
    rng = np.random.default_rng(5)
    p = Problem(rng.integers(0, 9, n).tolist() + [1], hq=2, hk=1, window=3, max_len=max_len)
    p.run()
    p.check()


@pytest.mark.parametrize("lens", [[200, 77, 180], [300, 77, 180], [1200, 700]])
def test_same_bits_every_time(lens):
    a = Problem(lens, hq=6, hk=2, mask=_every(5))
    a.run()
    first = (a.out.clone(), a.lse.clone(), a.dqkv.clone())
    import torch
    for _ in range(3):
        a.buffers()
        a.run()
        for x, y in zip(first, (a.out, a.lse, a.dqkv)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@kernels
def test_gradient_against_differences(max_len):
    """sum(out * dout) of the definition, moved both ways along random
    directions, against the kernel's gradients: they agree within the
    gradients' own bounds plus the differences' h^2 term."""
    import torch
    p = Problem([90], hq=2, hk=1, window=40, dtype="F16", seed=3, max_len=max_len)
    p.run()
    rows = torch.arange(POISON, POISON + 90, device="cuda")
    x = p.qkv[rows][:, :256].double().reshape(90, 4, 64)
    do = p.dout[rows][:, :128].double().reshape(90, 2, 64)

    def f(y):
        return (ref.attention(y[:, :2], y[:, 2:3], y[:, 3:], p.scale, 40, rows)[0] * do).sum()

    out, lse, grads, pr = ref.attention(x[:, :2], x[:, 2:3], x[:, 3:], p.scale, 40, rows, do)
    b = ref.attention_bounds(x[:, :2], x[:, 2:3], x[:, 3:], p.scale, pr, out, lse, ref.half_step("F16"),
                             ref.tiny("F16"), do, grads)
    bound = torch.cat([b["dq"], b["dk"], b["dv"]], 1)
    g = p.dqkv[rows][:, :256].double().reshape(90, 4, 64)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    for _ in range(4):
        d = torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float64)
        d1 = (f(x + 1e-4 * d) - f(x - 1e-4 * d)) / 2e-4
        d2 = (f(x + 2e-4 * d) - f(x - 2e-4 * d)) / 4e-4
        assert abs((g * d).sum() - d1) <= (bound * d.abs()).sum() + 2 * (d2 - d1).abs()


@kernels
def test_forward_without_statistics(max_len):
    import torch
    from laya_zig_b200 import gpu
    p = Problem([100, 3], max_len=max_len)
    p.forward()
    want = p.out.clone()
    p.out.fill_(7.0)
    gpu.attention(p.shape, p.q3[0], p.ld, p.q3[1], p.ld, p.q3[2], p.ld, p.out.data_ptr(), p.out.stride(0))
    assert torch.equal(want, p.out)


@pytest.mark.parametrize("hq,hk", [(2, 2), (6, 2), (5, 1), (64, 64)])
@pytest.mark.parametrize("window", [-1, 0, 2, 40])
@pytest.mark.parametrize("masked", [False, True])
def test_more_short_sequences_than_blocks(hq, hk, window, masked):
    """At most 64 tokens each, more of them than blocks; a third of the tokens
    and every seventh sequence absent."""
    lens = ([1, 16, 17, 33, 0, 64, 48, 2, 31, 63, 15] * (4 if hq > 8 else 60))[:-3]
    owner = np.repeat(np.arange(len(lens)), lens)

    def mask(n):
        return (np.arange(n) % 3 != 1) & (owner % 7 != 3)
    p = Problem(lens, hq=hq, hk=hk, window=window, mask=mask if masked else None, dtype="F16" if masked else "BF16")
    p.run()
    p.check()


@pytest.mark.parametrize("lens", [[1] * 50 + [9, 64, 30], [20, 3], [200, 70, 1], [500] * 4])
@pytest.mark.parametrize("dtype", ["BF16", "F16"])
def test_one_key_has_no_gradient_through_its_score(dtype, lens):
    """A query that sees one key has P = 1 whatever the score: dQ and dK are 0
    but for what exp(S - lse) is off 1. delta = P dP, so dS = P dP (1 - P);
    |1 - P| <= 2^-18 (S and lse below 2^3 in f32, each off by a few 2^-21), and
    |dP| <= 64 |dO| |V| < 64 * 25: |dQ| <= 0.125 * 1600 * 2^-18 * 5 < 2^-8."""
    p = Problem(lens, hq=3, hk=3, window=0, dtype=dtype)
    p.run()
    assert (p.dqkv[POISON:p.T - POISON, :2 * 3 * 64].abs() < 2.0 ** -8).all()
    p.check()


@kernels
@pytest.mark.parametrize("lens", [[180, 33] + [0] * 900, [0, 70, 0, 300] + [0] * 1500, [0] * 40 + [130] + [0] * 5])
def test_tables_with_unused_entries(lens, max_len):
    """Entries behind the last sequence are passed over, and still checked."""
    from laya_zig_b200 import gpu
    p = Problem(lens, max_len=max_len)
    p.run()
    p.check()
    p.cu[len(lens) - 2] += 1
    p.forward()
    with pytest.raises(gpu.LayaError) as e:
        gpu.op_status(p.status.data_ptr())
    assert e.value.code == gpu.ERR_ARG
    p.run()
    with pytest.raises(gpu.LayaError):
        gpu.op_status(p.status.data_ptr())


@pytest.mark.parametrize("table,max_len", [([0, 50, 40, 100], 60), ([-3, 20, 60, 100], 60), ([0, 30, 60, 5000], 60),
                                           ([90, 60, 30, 0], 60), ([0, 10, 20, 100], 60), ([0, 50, 40, 100], LONG),
                                           ([-3, 20, 60, 100], LONG), ([0, 30, 60, 5000], LONG),
                                           ([90, 60, 30, 0], LONG), ([-70, -60, 30, 0], LONG)])
def test_broken_offsets_are_recorded(table, max_len):
    """Decreasing, negative, too far, and a run longer than max_len."""
    import torch
    from laya_zig_b200 import gpu
    p = Problem([30, 30, 40], max_len=max_len)
    p.forward()  # sets the pointers
    gpu.op_status(p.status.data_ptr())
    p.cu.copy_(torch.tensor(table, dtype=torch.int32))
    p.run()
    with pytest.raises(gpu.LayaError) as e:
        gpu.op_status(p.status.data_ptr())
    assert e.value.code == gpu.ERR_ARG
    gpu.op_status(p.status.data_ptr())  # cleared


def test_host_memory_is_refused():
    from laya_zig_b200 import gpu
    p = Problem([30])
    a = np.zeros(1 << 16, np.uint8)
    at = (a.ctypes.data + 15) & ~15
    with pytest.raises(gpu.LayaError) as e:
        gpu.attention(p.shape, at, p.ld, p.qkv.data_ptr(), p.ld, p.qkv.data_ptr(), p.ld, p.out.data_ptr(),
                      p.out.stride(0))
    assert e.value.code == gpu.ERR_ARG and "device memory" in str(e.value)


@pytest.mark.parametrize("max_len", [200, LONG])
def test_captured_and_replayed_on_new_inputs(max_len):
    """Forward and backward in one CUDA graph, replayed after the inputs and
    the offsets changed, give what eager calls give."""
    import torch
    a = Problem([100, 60, 30], hq=4, hk=2, seed=1, max_len=max_len)
    b = Problem([20, 160, 10], hq=4, hk=2, seed=2, max_len=max_len)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a.run(s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        a.run(s.cuda_stream)
    a.qkv.copy_(b.qkv)
    a.dout.copy_(b.dout)
    a.cu.copy_(b.cu)
    a.lens, a.here = b.lens, b.here
    g.replay()
    torch.cuda.synchronize()
    b.run()
    a.check()
    assert torch.equal(a.dqkv, b.dqkv) and torch.equal(a.out, b.out)


@pytest.mark.parametrize("lens", [[100, 30], [400, 300]])
def test_two_streams_at_once(lens):
    import torch
    ps = [Problem(lens, seed=i) for i in range(2)]
    for p in ps:
        p.run()
    want = [p.dqkv.clone() for p in ps]
    streams = [torch.cuda.Stream() for _ in ps]
    torch.cuda.synchronize()
    for _ in range(5):
        for p, s in zip(ps, streams):
            p.run(s.cuda_stream)
    torch.cuda.synchronize()
    for p, w in zip(ps, want):
        assert torch.equal(p.dqkv, w)


@pytest.mark.parametrize("hq,hk", [(4, 4), (6, 2)])
def test_calls_in_a_row_share_a_workspace(hq, hk):
    """Backward passes back to back on one stream with one workspace, each
    followed at once by a kernel that overwrites its results: eager, and as two
    graphs replayed in turn."""
    import torch
    ps = [Problem(lens, hq=hq, hk=hk, seed=i) for i, lens in enumerate([[700, 900, 33], [2000], [300] * 20])]
    for p in ps:
        p.run()
    torch.cuda.synchronize()
    want = [p.dqkv.clone() for p in ps]
    ws = max((p.ws for p in ps), key=lambda w: w.numel())
    s = torch.cuda.Stream()
    kept = [torch.empty_like(w) for w in want]

    def go(i):
        p = ps[i]
        p.ws = ws
        p.backward(s.cuda_stream)
        kept[i].copy_(p.dqkv)
        p.dqkv.fill_(7.0)

    def check():
        torch.cuda.synchronize()
        for i, p in enumerate(ps):
            assert torch.equal(kept[i], want[i]) and (p.dqkv == 7).all()
            kept[i].zero_()
    with torch.cuda.stream(s):
        for _ in range(3):
            for i in range(3):
                go(i)
    check()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g, order in zip(graphs, [(0, 2, 1), (1, 0, 2)]):
        with torch.cuda.graph(g, stream=s):
            for i in order:
                go(i)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(4):
            for g in graphs:
                g.replay()
    check()
