"""The digits that the policy loss keeps where 32 bits are few: logits far from
0, decisions that are nearly certain."""
import math

import numpy as np
import pytest

import op_reference as ref
from test_gpu_policy import TEMP, _call, _make

pytestmark = pytest.mark.gpu

SHAPES = {"to16": [4, 16, 1, 7, 2], "to32": [17, 32, 5], "to64": [33, 64], "to128": [65, 128, 3], "to256": [129, 256],
          "to512": [257, 512], "to1024": [1000, 1024, 3], "wider": [1025, 3, 4000]}
NAMES = ("loss", "logp", "kl", "entropy", "dlogits")
# whole multiples of the first number up to the second in size, moved by the third:
# still exact in the type
STEPS = {"F32": [(2.0 ** -10, 4.0, 100.0), (2.0 ** -10, 4.0, -8192.0), (2.0 ** -3, 4.0, 2.0 ** 20)],
         "F16": [(2.0 ** -6, 4.0, 24.0)], "BF16": [(2.0 ** -3, 2.0, -16.0)]}


def _steps(t, step, most):
    return (t.float().clamp(-most, most) / step).round() * step


@pytest.mark.parametrize("lens", list(SHAPES))
@pytest.mark.parametrize("dtype,which", [("F32", 0), ("F32", 1), ("F32", 2), ("F16", 0), ("BF16", 0)])
def test_a_shift_of_all_logits_changes_nothing(lens, dtype, which):
    """Only differences of a decision's logits matter, and these are the same:
    so is every output, to the last bit. And log p is right: x - max is exact,
    times the scale 2^-23 of |z|, a sum of exponentials of 2^-22 each (its tree
    and the errors of z, weighted, beside that), a logarithm of 2^-22, two
    products: within 2^-21 (2 + |z| + sum p |z|) in all."""
    import torch
    from laya_zig_b200 import gpu
    step, most, shift = STEPS[dtype][which]
    z, zr, act, q, adv, old, grad = _make(SHAPES[lens], dtype, seed=which)
    z, zr = _steps(z, step, most), _steps(zr, step, most)
    ref_dt = ref.DT[dtype]
    assert torch.equal((z + shift).to(ref_dt).double(), z.double() + shift)
    a, sa = _call(SHAPES[lens], z, zr, act, q, adv, old, grad, dtype)
    b, sb = _call(SHAPES[lens], z + shift, zr - shift, act, q, adv, old, grad, dtype)
    for s in (sa, sb):
        gpu.op_status(s.data_ptr())
    for name in NAMES:
        assert torch.equal(a[name].view(torch.uint8), b[name].view(torch.uint8)), name
    at = 0
    for i, k in enumerate(SHAPES[lens]):
        zi = z[at:at + k].double() / float(np.float32(TEMP[int(q[i])]))
        at += k
        lp = torch.log_softmax(zi, 0)
        far = (zi - zi.max()).abs()
        want = lp[int(act[i])].item()
        bound = 2.0 ** -21 * (2 + far[int(act[i])].item() + (lp.exp() * far).sum().item())
        assert abs(b["logp"][i].item() - want) <= bound and math.isfinite(want)


def _certain(lens, seed):
    """Logits 8 to 12 below the decision's best option, which was taken; old log
    probabilities near the present ones."""
    import torch
    g = torch.Generator()
    g.manual_seed(seed)
    z, act, old = [], [], []
    for k in lens:
        x = -8 - 4 * torch.rand(k, generator=g)
        a = int(torch.randint(0, k, (1,), generator=g))
        x[a] = 0.0
        z.append(x + 3.0)
        act.append(a)
        old.append(0.1 * (torch.rand((), generator=g).item() - 0.5))
    n = len(lens)
    q = torch.randint(0, 3, (n,), generator=g).to(torch.int32)
    return (torch.cat(z), torch.tensor(act, dtype=torch.int32), q, torch.rand(n, generator=g) + 0.5,
            torch.tensor(old), torch.ones(n))


@pytest.mark.parametrize("lens", ["to16", "to32", "to64", "to128", "to256", "to512", "to1024", "wider"])
def test_certain_decisions_keep_their_digits(lens):
    """1 - p near 1e-4 a rival: log p, the entropy and the gradients, relative to
    themselves. In units of 2^-23: a rival's e^z is off by |z| (z's rounding) and 2
    (ex2.approx), their sum by 20 (39 roundings at most), the logarithm by 12 (of
    1/8 and more, where lg2.approx's 2^-22 is that part of it; less below), its
    products by 4: R = |z| + 38 for log p and 1 - p. The ratio: exp of log p - old,
    both at most 1 in size and off by R |log p| + 2^-24: 2^-20. The entropy's terms
    are p times log p, products of values off by R and 2^-23 (1 + |z|)."""
    import torch
    from laya_zig_b200 import gpu
    shape = SHAPES[lens]
    z, act, q, adv, old, grad = _certain(shape, 7)
    out, status = _call(shape, z, None, act, q, adv, old, grad, klc=0.0, entc=0.0, lead=2)
    gpu.op_status(status.data_ptr())
    at = 0
    for i, k in enumerate(shape):
        t = float(np.float32(TEMP[int(q[i])]))
        zi = (z[at:at + k].double()).requires_grad_(True)
        got = out["dlogits"][2 + at:2 + at + k].cpu().double()
        at += k
        loss, logp, _, ent = ref.policy(zi, None, int(act[i]), float(adv[i]), float(old[i]), t, float(np.float32(0.2)),
                                        float(np.float32(0.3)), 0.0, 0.0)
        want = torch.autograd.grad(loss, zi)[0]
        if k == 1:
            assert out["logp"][i] == 0 and out["entropy"][i] == 0 and got[0] == 0
            continue
        R = 2.0 ** -23 * (12 / t + 38)
        assert abs(out["logp"][i].item() / logp.item() - 1) <= R
        assert abs(out["entropy"][i].item() / ent.item() - 1) <= 2 * R
        assert ((got - want).abs() <= (2 * R + 2.0 ** -20) * want.abs()).all()
        assert abs(got.sum().item()) <= (2 * R + 2.0 ** -20) * got.abs().sum().item()


@pytest.mark.parametrize("lens", ["to16", "to32", "to64", "to128", "to256", "to512", "to1024", "wider"])
@pytest.mark.parametrize("every", [1, 2, 3])
def test_ties_at_the_maximum(lens, every):
    """All options, or every second or third, at the maximum, the others ruled out:
    the sum is the whole number n, log p its logarithm within 2^-21 (of two or
    more: lg2.approx 2^-22 of 1 at least, two products), 1 / n and 1 - 1 / n right
    to 2^-20, and the gradients, -1/n of the difference, to 2^-19."""
    import torch
    from laya_zig_b200 import gpu
    shape = [k for k in SHAPES[lens] if k >= 3]
    z = torch.full((sum(shape),), -math.inf)
    at, act = 0, []
    for k in shape:
        z[at:at + k:every] = 1.5
        act.append((k - 1) // every * every)
        at += k
    n = len(shape)
    act = torch.tensor(act, dtype=torch.int32)
    adv, old = torch.ones(n), torch.zeros(n)
    out, status = _call(shape, z, z, act, None, adv, old, torch.ones(n), klc=0.0, entc=0.0)
    gpu.op_status(status.data_ptr())
    at = 0
    for i, k in enumerate(shape):
        m = len(range(0, k, every))
        d = out["dlogits"][2 + at:2 + at + k].cpu().double()
        at += k
        assert abs(out["logp"][i].item() + math.log(m)) <= 2.0 ** -21 * math.log(m)
        assert abs(out["entropy"][i].item() - math.log(m)) <= 2.0 ** -20 * math.log(m)
        assert out["kl"][i].item() == 0
        if m == 1:
            assert (d == 0).all()
            continue
        want = torch.zeros(k, dtype=torch.float64)
        want[::every] = 1.0 / m
        want[int(act[i])] -= 1.0
        want /= m  # the ratio: old is 0; below the clip's range min keeps r A
        assert ((d - want).abs() <= 2.0 ** -19 * want.abs()).all()


@pytest.mark.parametrize("lens", ["to16", "to64", "to512", "to1024", "wider"])
def test_a_reference_that_rules_options_out(lens):
    """An option that only the reference rules out makes the divergence infinite.
    With kl_coef 0 it is reported and nothing else: loss and gradients are those
    without a reference."""
    import torch
    from laya_zig_b200 import gpu
    shape = SHAPES[lens]
    z, zr, act, q, adv, old, grad = _make(shape, seed=3)
    zr = zr.clone()
    at = 0
    for k in shape:
        if k > 1:
            zr[at + k // 2] = -math.inf
        at += k
    a, sa = _call(shape, z, zr, act, q, adv, old, grad, klc=0.0)
    b, sb = _call(shape, z, None, act, q, adv, old, grad, klc=0.0)
    for s in (sa, sb):
        gpu.op_status(s.data_ptr())
    for i, k in enumerate(shape):
        assert a["kl"][i].item() == (math.inf if k > 1 else 0.0)
    for name in ("loss", "logp", "entropy", "dlogits"):
        assert torch.isfinite(b[name]).all() and torch.equal(a[name], b[name]), name
