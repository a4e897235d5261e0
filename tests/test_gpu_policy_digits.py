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
