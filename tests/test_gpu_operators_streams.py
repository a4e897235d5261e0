"""Rotary positions and the policy loss on two streams at once, and in place."""
import pytest

import op_reference as ref

pytestmark = pytest.mark.gpu


def test_rope_on_two_streams():
    """Different rows, one plan, each stream's calls one after the other in place:
    a quarter turn's worth of calls forward and as many back."""
    import torch
    from laya_zig_b200 import gpu
    plan = gpu.RopePlan()
    cu = [torch.tensor([0, n], dtype=torch.int32, device="cuda") for n in (3000, 2500)]
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    x = [torch.randn((int(c[1]), 768), generator=g, device="cuda").to(torch.bfloat16) for c in cu]

    def turn(y, i, stream, inverse=False):
        gpu.rope(plan, y.data_ptr(), 768, y.data_ptr(), 768, y.shape[0], 12, status[i:].data_ptr(),
                 cu_seqlens_ptr=cu[i].data_ptr(), n_seqs=1, inverse=inverse, stream=stream)
    want = []
    for i in range(2):
        y = x[i].clone()
        for _ in range(4):
            turn(y, i, 0)
        turn(y, i, 0, inverse=True)
        want.append(y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [t.clone() for t in x]
    torch.cuda.synchronize()
    for _ in range(4):
        for i in range(2):
            turn(got[i], i, streams[i].cuda_stream)
    for i in range(2):
        turn(got[i], i, streams[i].cuda_stream, inverse=True)
    for i in range(2):
        gpu.op_status(status[i:].data_ptr(), streams[i].cuda_stream)
        assert torch.equal(got[i], want[i])
    # and the first call's result is the rotation
    y = x[0].clone()
    turn(y, 0, 0)
    gpu.op_status(status.data_ptr())
    xs = x[0].double().reshape(-1, 12, 64)
    exact = ref.rope(xs, torch.arange(3000, device="cuda"), ref.rope_frequencies(64))
    pair = xs[..., :32].abs() + xs[..., 32:].abs()
    bound = (ref.half_step("BF16") + 2.0 ** -20) * torch.cat([pair, pair], -1) + ref.tiny("BF16")
    assert ((y.double().reshape(-1, 12, 64) - exact).abs() <= bound).all()


@pytest.mark.parametrize("k", [16, 64, 1024, 3000])
def test_policy_on_two_streams(k):
    """Two batches, each with its own outputs and status word, over and over; one
    of them has a bad action, which the other's status does not show."""
    import torch
    from laya_zig_b200 import gpu
    n = 500
    g = torch.Generator(device="cuda")
    g.manual_seed(k)
    cu = torch.arange(n + 1, dtype=torch.int32, device="cuda") * k
    status = torch.zeros(2, dtype=torch.int32, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    sides = []
    for i in range(2):
        d = dict(z=torch.randn(n * k, generator=g, device="cuda"), r=torch.randn(n * k, generator=g, device="cuda"),
                 a=torch.randint(0, k, (n,), generator=g, device="cuda").to(torch.int32),
                 adv=torch.randn(n, generator=g, device="cuda"), old=torch.zeros(n, device="cuda"),
                 loss=torch.zeros(n, device="cuda"), d=torch.zeros(n * k, device="cuda"))
        d["b"] = gpu.PolicyBatch(cu.data_ptr(), n, n * k, k, status[i:].data_ptr(), kl_coef=0.1, entropy_coef=0.01)
        sides.append(d)
    sides[1]["a"][7] = k

    def call(s, stream):
        gpu.policy_loss(s["b"], s["z"].data_ptr(), s["r"].data_ptr(), s["a"].data_ptr(), s["adv"].data_ptr(),
                        s["old"].data_ptr(), loss_ptr=s["loss"].data_ptr(), dlogits_ptr=s["d"].data_ptr(), stream=stream)
    want = []
    for s in sides:
        call(s, 0)
        want.append((s["loss"].clone(), s["d"].clone()))
        s["loss"].fill_(7.0)
        s["d"].fill_(7.0)
    status.zero_()
    torch.cuda.synchronize()
    for _ in range(10):
        for i, s in enumerate(sides):
            call(s, streams[i].cuda_stream)
    gpu.op_status(status.data_ptr(), streams[0].cuda_stream)
    with pytest.raises(gpu.LayaError):
        gpu.op_status(status[1:].data_ptr(), streams[1].cuda_stream)
    for s, (loss, d) in zip(sides, want):
        assert torch.equal(s["loss"], loss) and torch.equal(s["d"], d)
    assert want[1][0][7] == 0 and (want[1][1][7 * k:8 * k] == 0).all() and (want[0][0] != 0).any()
