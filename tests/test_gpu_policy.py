"""laya_gpu_policy_loss against its definition, differentiated in 64 bits."""
import math

import numpy as np
import pytest

import op_reference as ref

pytestmark = pytest.mark.gpu

TEMP = (1.0, 0.7, 1.6)


def _make(lens, dtype="F32", seed=0, ruled_out=0.0, spread=1.5, moved=0.3):
    import torch
    g = torch.Generator()
    g.manual_seed(seed)
    G, n = sum(lens), len(lens)
    zr = (spread * torch.randn(G, generator=g)).to(ref.DT[dtype])
    z = (zr.float() + moved * torch.randn(G, generator=g)).to(ref.DT[dtype])
    act = torch.tensor([int(torch.randint(0, max(k, 1), (1,), generator=g)) for k in lens], dtype=torch.int32)
    if ruled_out:
        out = torch.rand(G, generator=g) < ruled_out
        at = 0
        for k, a in zip(lens, act.tolist()):
            if k:
                out[at + a] = False
            at += k
        z[out] = -math.inf
        zr[out] = -math.inf
    q = torch.randint(0, 3, (n,), generator=g).to(torch.int32)
    adv = torch.randn(n, generator=g)
    old = torch.tensor([-math.log(max(k, 1)) for k in lens]) + 0.5 * torch.randn(n, generator=g)
    grad = torch.rand(n, generator=g) + 0.5
    return z, zr, act, q, adv, old, grad


def _call(lens, z, zr, act, q, adv, old, grad, dtype="F32", want=("loss", "logp", "kl", "entropy", "dlogits"),
          klc=0.1, entc=0.03, lead=2, max_options=None):
    import torch
    from laya_zig_b200 import gpu
    n, G = len(lens), sum(lens)
    dt = ref.DT[dtype]

    def padded(t):
        return None if t is None else torch.cat([torch.full((lead,), math.nan), t.float(),
                                                 torch.full((lead,), math.nan)]).to(dt).cuda()
    zp, zrp = padded(z), padded(zr)
    cu = torch.tensor([lead] + (np.cumsum(lens) + lead).tolist(), dtype=torch.int32, device="cuda")
    dev = {k: None if t is None else t.cuda() for k, t in dict(act=act, q=q, adv=adv, old=old, grad=grad).items()}
    out = {k: torch.full((n,), 7.0, device="cuda") for k in ("loss", "logp", "kl", "entropy")}
    out["dlogits"] = torch.full((G + 2 * lead,), 7.0, dtype=dt, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    b = gpu.PolicyBatch(cu.data_ptr(), n, G + 2 * lead, max_options or max(max(lens), 1), status.data_ptr(),
                        qtypes_ptr=0 if q is None else dev["q"].data_ptr(), temperature=TEMP, clip_low=0.2,
                        clip_high=0.3, kl_coef=klc, entropy_coef=entc, dtype=dtype)
    p = {k: out[k].data_ptr() if k in want else 0 for k in out}
    gpu.policy_loss(b, zp.data_ptr(), 0 if zrp is None else zrp.data_ptr(), dev["act"].data_ptr(),
                    dev["adv"].data_ptr(), dev["old"].data_ptr(), 0 if grad is None else dev["grad"].data_ptr(),
                    p["loss"], p["logp"], p["kl"], p["entropy"], p["dlogits"])
    return out, status


def _check(lens, dtype="F32", klc=0.1, entc=0.03, use_ref=True, use_q=True, use_grad=True, lead=2, max_options=None,
           **kw):
    import torch
    from laya_zig_b200 import gpu
    z, zr, act, q, adv, old, grad = _make(lens, dtype, **kw)
    if not use_ref:
        zr = None
    out, status = _call(lens, z, zr, act, q if use_q else None, adv, old, grad if use_grad else None, dtype,
                        klc=klc, entc=entc, lead=lead, max_options=max_options)
    gpu.op_status(status.data_ptr())
    got = {k: v.cpu().double() for k, v in out.items()}
    assert (got["dlogits"][:lead] == 7).all() and (got["dlogits"][len(z) + lead:] == 7).all()
    u, t0 = ref.half_step(dtype), ref.tiny(dtype)
    at = 0
    for i, k in enumerate(lens):
        w = float(grad[i]) if use_grad else 1.0
        d = got["dlogits"][lead + at:lead + at + k]
        zi = z[at:at + k].double()
        zri = None if zr is None else zr[at:at + k].double()
        at += k
        vals = [got[x][i].item() for x in ("loss", "logp", "kl", "entropy")]
        if k == 0 or not (zi > -math.inf).any():
            assert vals == [0.0] * 4 and (d == 0).all()
            continue
        zi.requires_grad_(True)
        t = TEMP[int(q[i])] if use_q else TEMP[0]
        t = float(np.float32(t))
        args = (zi, zri, int(act[i]), float(adv[i]), float(old[i]), t, float(np.float32(0.2)), float(np.float32(0.3)),
                float(np.float32(klc)), float(np.float32(entc)))
        loss, logp, kl, ent = ref.policy(*args)
        g = torch.autograd.grad(loss, zi)[0] * w
        g = torch.where(zi > -math.inf, g, 0.0)
        # z = logit / t carries two roundings; lse a sum of exponentials
        # (2 ulp each, a tree of at most 5 + K / 32 sums) and a logarithm: every
        # log probability is off by at most
        top = zi.detach()[zi > -math.inf].abs().max().item() / t
        if zri is not None:
            top = max(top, zri[zri > -math.inf].abs().max().item() / t)
        e = 2.0 ** -24 * (6 * top + 3 * abs(logp.item()) + 2 * math.log(k + 1) + 16 + k / 16)
        lp = torch.log_softmax(zi.detach() / t, 0)
        lp = torch.where(zi.detach() > -math.inf, lp, 0.0)
        size = lp.abs().max().item()
        if zri is not None:
            lr = torch.log_softmax(zri / t, 0)
            size = max(size, lr[lr > -math.inf].abs().max().item())
        ee = e * (4 + 2 * size) + 2.0 ** -22 * (1 + size)  # of sums of p times log probabilities
        assert abs(vals[1] - logp.item()) <= e + 2.0 ** -23 * abs(logp.item())
        assert abs(vals[3] - ent.item()) <= ee
        assert abs(vals[2] - kl.item()) <= ee
        r = math.exp(logp.item() - float(old[i]))
        ra = r * abs(float(adv[i]))
        el = 2 * (e + 2.0 ** -22 * (2 + abs(float(old[i])) + abs(logp.item()))) * ra
        assert abs(vals[0] - loss.item()) <= el + (klc + entc) * 2 * ee + 2.0 ** -22 * abs(loss.item())
        near = min(abs(r - 0.8), abs(r - 1.3)) < 1e-5  # 32 bits do not say on which side of the edge
        if not near:
            p = torch.exp(lp) * (zi.detach() > -math.inf)
            own = torch.zeros(k, dtype=torch.float64)
            own[int(act[i])] = 1
            eg = el * (own + p) * 2 + (klc + entc) * p * (6 * ee + 4 * e * size)
            # ex2.approx.ftz gives 0 below 2^-126: an absolute error of 2^-126
            # for a probability, which is multiplied by r A, by kl_coef (d -
            # KL) and by entropy_coef (lp + H), whose factors do not pass 2
            # size
            eg = eg + 2.0 ** -126 * (ra + (abs(klc) + abs(entc)) * 2 * size + 1)
            assert ((d - g).abs() <= w / t * eg + (u + 2.0 ** -20) * g.abs() + t0 +
                    2.0 ** -22 * w / t * ra * (own + p)).all(), (i, k)
    return got


SHAPES = {"one": [1], "four": [4] * 9, "mixed": [4, 16, 1, 0, 7, 9, 16, 2], "to32": [17, 32, 5, 31, 1, 0],
          "to64": [33, 64, 2, 0, 63, 8], "to128": [17, 65, 5, 31, 128, 1, 0], "to256": [129, 256, 1, 32, 33],
          "to512": [257, 512, 31, 0, 4], "wide": [129, 1000, 1024, 3], "wider": [1025, 3, 4000, 0]}


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("lens", list(SHAPES))
def test_shapes(lens, dtype):
    _check(SHAPES[lens], dtype)


@pytest.mark.parametrize("lens", ["mixed", "to32", "to64", "to128", "to256", "to512", "wide", "wider"])
@pytest.mark.parametrize("kw", [dict(ruled_out=0.4), dict(use_ref=False), dict(use_q=False), dict(use_grad=False),
                                dict(klc=0.0, entc=0.0), dict(spread=30.0), dict(klc=3.0, entc=-1.0, seed=9)])
def test_forms(lens, kw):
    _check(SHAPES[lens], **kw)


def test_all_ruled_out():
    z, zr, act, q, adv, old, grad = _make([5, 3, 4])
    z[5:8] = -math.inf
    zr[5:8] = -math.inf
    out, status = _call([5, 3, 4], z, zr, act, q, adv, old, grad)
    from laya_zig_b200 import gpu
    gpu.op_status(status.data_ptr())
    for k in ("loss", "logp", "kl", "entropy"):
        assert out[k][1] == 0 and out[k][0] != 0 and out[k][2] != 0
    assert (out["dlogits"][2 + 5:2 + 8] == 0).all()


def test_small_kl_keeps_its_digits():
    """A policy moved by 1e-3 from its reference: KL near 5e-7, right to a
    percent (the plain difference of two logarithms would be off by 1e-7)."""
    lens = [6] * 50
    got = _check(lens, moved=1e-3)
    z, zr, act, q, adv, old, grad = _make(lens, moved=1e-3)
    for i in range(50):
        t = float(np.float32(TEMP[int(q[i])]))
        kl = ref.policy(z[6 * i:6 * i + 6].double(), zr[6 * i:6 * i + 6].double(), int(act[i]), 0.0, 0.0, t, .2, .3,
                        0, 0)[2].item()
        assert abs(got["kl"][i].item() - kl) <= 1e-2 * kl + 1e-10


def test_gradient_against_differences():
    """Losses of moved logits, in the kernel's own f32: central differences
    with h = 2^-6, whose third-order term is at most h^2 and whose rounding is
    2^-22 |loss| / h."""
    import torch
    lens = [5, 3]
    z, zr, act, q, adv, old, grad = _make(lens, seed=2)
    old = old + 2.0  # ratios far below the clip's edge
    adv = -adv.abs()
    grad = torch.ones(2)
    base = _call(lens, z, zr, act, None, adv, old, grad, klc=0.5, entc=0.2)[0]
    d = base["dlogits"].cpu()[2:10]
    h = 2.0 ** -6
    for j in range(8):
        f = []
        for s in (h, -h):
            zz = z.clone()
            zz[j] += s
            f.append(_call(lens, zz, zr, act, None, adv, old, grad, klc=0.5, entc=0.2)[0]["loss"].cpu().double())
        i = 0 if j < 5 else 1
        diff = ((f[0] - f[1]) / (2 * h))[i].item()
        size = 2 * base["loss"].abs().max().item() + 4
        assert abs(diff - d[j].item()) <= h * h * size + 2.0 ** -21 * size / h


def test_outputs_are_optional():
    import torch
    lens = [4, 9, 2]
    data = _make(lens)
    full, _ = _call(lens, *data)
    for name in full:
        part, _ = _call(lens, *data, want=(name,))
        for k in part:
            assert torch.equal(part[k], full[k]) if k == name else (part[k] == 7).all()


@pytest.mark.parametrize("max_options", [16, 32, 64, 128, 256, 512, 1024, 5000])
def test_bad_indices_are_recorded(max_options):
    """An action outside its decision, a question type above 2: the decision's
    outputs are 0, the others' untouched by it."""
    import torch
    from laya_zig_b200 import gpu
    lens = [4, 5, 6]
    z, zr, act, q, adv, old, grad = _make(lens)
    good, _ = _call(lens, z, zr, act, q, adv, old, grad, max_options=max_options)
    for bad in ("act", "neg", "q"):
        a2, q2 = act.clone(), q.clone()
        if bad == "q":
            q2[1] = 3
        else:
            a2[1] = 5 if bad == "act" else -1
        out, status = _call(lens, z, zr, a2, q2, adv, old, grad, max_options=max_options)
        with pytest.raises(gpu.LayaError) as e:
            gpu.op_status(status.data_ptr())
        assert e.value.code == gpu.ERR_ARG
        assert out["loss"][1] == 0 and (out["dlogits"][6:11] == 0).all()
        for i in (0, 2):
            assert out["loss"][i] == good["loss"][i]
        assert torch.equal(out["dlogits"][11:17], good["dlogits"][11:17])


@pytest.mark.parametrize("table", [[2, 1, 6, 17], [-4, 3, 6, 17], [2, 6, 10, 4000]])
def test_broken_offsets_are_recorded(table):
    import torch
    from laya_zig_b200 import gpu
    z = torch.zeros(17, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    f = torch.zeros(3, device="cuda")
    d = torch.full((17,), 7.0, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    cu = torch.tensor(table, dtype=torch.int32, device="cuda")
    b = gpu.PolicyBatch(cu.data_ptr(), 3, 17, 16, st.data_ptr())
    gpu.policy_loss(b, z.data_ptr(), 0, i.data_ptr(), f.data_ptr(), f.data_ptr(), dlogits_ptr=d.data_ptr())
    with pytest.raises(gpu.LayaError):
        gpu.op_status(st.data_ptr())


def test_nan_stays_in_its_decision():
    import torch
    lens = [4, 4, 4]
    z, zr, act, q, adv, old, grad = _make(lens)
    good, _ = _call(lens, z, zr, act, q, adv, old, grad)
    z[5] = math.nan
    out, _ = _call(lens, z, zr, act, q, adv, old, grad)
    assert torch.isnan(out["loss"][1]) and torch.isnan(out["dlogits"][6:10]).all()
    for i in (0, 2):
        assert out["loss"][i] == good["loss"][i]
        assert torch.equal(out["dlogits"][2 + 4 * i:6 + 4 * i], good["dlogits"][2 + 4 * i:6 + 4 * i])
