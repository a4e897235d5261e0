"""Workloads of the training-step operators: rotary positions, packed
attention with its backward pass, and the clipped policy loss over a
decision's options. `listed()` names the cases, `draw()` makes more of the
same ranges, `prepare()` makes the inputs on the GPU, `run()` makes one pass
(in plain torch operations, or through the framework's entry points where
`own` is true), `exact()` gives the same outputs from the definitions in 64
bits, and `work()` the bytes and operations a pass cannot do without.
"""
import math
import random

import torch

own = False

HEAD_DIM = 64
THETA = 160000.0  # the encoder's rotary base
DTYPES = {"BF16": torch.bfloat16, "F16": torch.float16, "F32": torch.float32}
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
KL_COEF, ENTROPY_COEF = 0.05, 0.01
TEMPERATURE = (1.0, 0.8, 1.25)


# ---------------------------------------------------------------- the cases

def _rope(name, n_seqs, min_len, max_len, **kw):
    c = {"name": name, "op": "rope", "n_seqs": n_seqs, "min_len": min_len, "max_len": max_len, "len_seed": 1,
         "heads": 24, "layout": "half", "rot_dim": 64, "factor": 1.0, "original_len": 0, "inverse": False,
         "dtype": "BF16", "positions": False}
    c.update(kw)
    return c


def _attn(name, n_seqs, min_len, max_len, **kw):
    c = {"name": name, "op": "attention", "n_seqs": n_seqs, "min_len": min_len, "max_len": max_len, "len_seed": 1,
         "n_heads": 12, "n_kv_heads": 12, "window": -1, "dtype": "BF16", "mask": False, "backward": True}
    c.update(kw)
    return c


def _policy(name, n, min_k, max_k, **kw):
    c = {"name": name, "op": "policy", "n": n, "min_k": min_k, "max_k": max_k, "len_seed": 1, "dtype": "F32",
         "ref": True, "masked": False}
    c.update(kw)
    return c


def listed():
    return [
        # one short decision: launch latency
        _rope("rope_decision", 1, 64, 64),
        # the headline batch: 64 decisions of 175-180 tokens, queries and keys of one layer
        _rope("rope_batch", 64, 175, 180),
        # gradient of a long scaled sequence: pairs side by side, half of each head rotated
        _rope("rope_long_scaled", 1, 32768, 32768, layout="interleaved", rot_dim=32, factor=4.0, original_len=8192,
              inverse=True, dtype="F16"),
        # one short decision, forward and backward: latency
        _attn("attention_decision", 1, 64, 64),
        # a global layer of the headline batch, forward and backward
        _attn("attention_batch_global", 64, 175, 180),
        # a sliding layer (64 keys to either side) of the same batch
        _attn("attention_batch_window", 64, 175, 180, window=64, dtype="F16"),
        # ragged lengths down to one token, a padded batch's absent tokens, key heads shared by three query heads
        _attn("attention_ragged_grouped", 128, 1, 512, n_kv_heads=4, mask=True),
        # one decision of 8,192 tokens, a global layer, forward and backward
        _attn("attention_long", 1, 8192, 8192),
        # scoring two long sequences on a sliding layer: the forward alone, with its statistics
        _attn("attention_long_window_forward", 2, 16000, 16384, window=64, backward=False),
        # one batch of decisions with four options each: latency
        _policy("policy_batch", 64, 4, 4),
        # a sweep's worth of decisions, some options masked out
        _policy("policy_sweep", 65536, 4, 16, masked=True),
        # many options to a decision, up to the most the model scores, 16-bit logits
        _policy("policy_wide", 16384, 1, 1024, dtype="BF16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attention", "attention", "policy"])
    if op == "rope":
        hi = _log_int(rng, 1, 8192)
        n = _log_int(rng, 1, max(1, 32768 // hi))
        c = _rope("", n, rng.randint(max(1, hi // 3), hi), hi, layout=rng.choice(["half", "interleaved"]),
                  rot_dim=rng.choice([64, 48, 32, 16]), heads=rng.choice([24, 16, 13, 2]),
                  factor=rng.choice([1.0, 1.0, 2.0, 4.0]), original_len=rng.choice([0, 8192]),
                  inverse=rng.random() < 0.5, dtype=rng.choice(["BF16", "F16", "F32"]), positions=rng.random() < 0.3)
    elif op == "attention":
        hi = _log_int(rng, 1, 6000)
        window = rng.choice([-1, -1, 64, 64, _log_int(rng, 1, 200)])
        most = max(1, min(20000 // hi, 30_000_000 // (hi * hi)))
        n = min(300, _log_int(rng, 1, most))
        heads, kv = rng.choice([(12, 12), (12, 12), (12, 4), (8, 2), (5, 1)])
        c = _attn("", n, rng.randint(max(1, hi // 4), hi), hi, n_heads=heads, n_kv_heads=kv, window=window,
                  dtype=rng.choice(["BF16", "F16"]), mask=rng.random() < 0.3, backward=rng.random() < 0.75)
    else:
        hi = _log_int(rng, 2, 1024)
        n = _log_int(rng, 1, min(200000, 8_000_000 // hi))
        c = _policy("", n, rng.randint(1, hi), hi, dtype=rng.choice(["F32", "F32", "BF16", "F16"]),
                    ref=rng.random() < 0.75, masked=rng.random() < 0.5)
    c["len_seed"] = rng.randrange(1 << 30)
    del c["name"]
    return c


def _lengths(n, lo, hi, seed):
    """n whole numbers of [lo, hi], the largest among them."""
    r = random.Random(seed)
    v = [r.randint(lo, hi) for _ in range(n)]
    v[r.randrange(n)] = hi
    return v


# ---------------------------------------------------------------- the inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed & 0x7FFFFFFFFFFF)
    return g


def _offsets(lens):
    return torch.tensor([0] + torch.tensor(lens, dtype=torch.int64).cumsum(0).tolist(), dtype=torch.int32,
                        device="cuda")


def _inputs_rope(case, seed):
    g = _gen(seed)
    lens = _lengths(case["n_seqs"], case["min_len"], case["max_len"], case["len_seed"])
    T, W = sum(lens), case["heads"] * HEAD_DIM
    # queries and keys inside the projection's row of queries, keys and values
    row = torch.randn((T, W + W // 2), generator=g, device="cuda").to(DTYPES[case["dtype"]])
    st = {"x": row[:, :W], "y": torch.zeros((T, W), dtype=row.dtype, device="cuda"), "cu": _offsets(lens),
          "positions": None, "T": T, "row": row}
    if case["positions"]:
        # tokens taken out of a longer text: their places in it, in order
        st["positions"] = torch.randint(0, 4 * case["max_len"], (T,), generator=g, device="cuda").to(torch.int32)
    return st


def _inputs_attention(case, seed):
    g = _gen(seed)
    lens = _lengths(case["n_seqs"], case["min_len"], case["max_len"], case["len_seed"])
    dt = DTYPES[case["dtype"]]
    T, hq, hk = sum(lens), case["n_heads"], case["n_kv_heads"]
    width = (hq + 2 * hk) * HEAD_DIM
    qkv = torch.randn((T, width), generator=g, device="cuda").to(dt)
    st = {"qkv": qkv, "cu": _offsets(lens), "T": T, "lens": lens, "mask": None,
          "out": torch.zeros((T, hq * HEAD_DIM), dtype=dt, device="cuda"),
          "lse": torch.zeros((hq, T), dtype=torch.float32, device="cuda")}
    if case["mask"]:
        # an absent token in five, and now and then a whole sequence
        keep = torch.rand((T,), generator=g, device="cuda") > 0.2
        gone = torch.rand((len(lens),), generator=g, device="cuda") > 0.05
        keep &= torch.repeat_interleave(gone, torch.tensor(lens, device="cuda"))
        st["mask"] = keep.to(torch.uint8)
    if case["backward"]:
        st["dout"] = torch.randn((T, hq * HEAD_DIM), generator=g, device="cuda").to(dt)
        st["dqkv"] = torch.zeros_like(qkv)
    return st


def _off_the_edge(old, logits, qtypes, cu, at, k):
    """`old` moved where the ratio falls within 1e-5 of the clip's edges: the
    gradient steps there, and 32 bits do not say on which side it falls."""
    n = k.numel()
    owner = torch.repeat_interleave(torch.arange(n, device="cuda"), k)
    t = torch.tensor(TEMPERATURE, dtype=torch.float64, device="cuda")[qtypes.to(torch.int64)]
    z = logits.double() / t[owner]
    total = torch.zeros((n,), dtype=torch.float64, device="cuda").index_add_(0, owner, torch.exp(z))
    ratio = torch.exp(z[at] - torch.log(total) - old.double())
    close = ((ratio - (1.0 - CLIP_LOW)).abs() < 1e-5) | ((ratio - (1.0 + CLIP_HIGH)).abs() < 1e-5)
    return torch.where(close, old + 1e-3, old)


def _inputs_policy(case, seed):
    g = _gen(seed)
    n, dt = case["n"], DTYPES[case["dtype"]]
    lens = _lengths(n, case["min_k"], case["max_k"], case["len_seed"])
    cu = _offsets(lens)
    k = (cu[1:] - cu[:-1]).to(torch.int64)
    G = int(cu[-1])
    ref = 1.5 * torch.randn((G,), generator=g, device="cuda")
    logits = ref + 0.3 * torch.randn((G,), generator=g, device="cuda")
    pick = torch.rand((n,), generator=g, device="cuda")
    actions = torch.minimum((pick * k).to(torch.int64), k - 1)
    at = cu[:-1].to(torch.int64) + actions
    if case["masked"]:
        # options the caller rules out: -inf in both, never the one that was taken
        out = torch.rand((G,), generator=g, device="cuda") < 0.15
        out[at] = False
        logits[out] = -math.inf
        ref[out] = -math.inf
    logits, ref = logits.to(dt), ref.to(dt)
    qtypes = torch.randint(0, 3, (n,), generator=g, device="cuda").to(torch.int32)
    # the behaviour policy's log probability of the taken option: near the present one
    near = -torch.log(k.to(torch.float32)) + 0.4 * torch.randn((n,), generator=g, device="cuda")
    near = _off_the_edge(near, logits, qtypes, cu, at, k)
    return {"logits": logits, "ref": ref if case["ref"] else None, "cu": cu, "G": G,
            "actions": actions.to(torch.int32), "qtypes": qtypes, "old": near,
            "advantages": torch.randn((n,), generator=g, device="cuda"),
            "grad": torch.full((n,), 1.0 / n, device="cuda"),
            "loss": torch.zeros((n,), device="cuda"), "logp": torch.zeros((n,), device="cuda"),
            "kl": torch.zeros((n,), device="cuda"), "entropy": torch.zeros((n,), device="cuda"),
            "dlogits": torch.zeros((G,), dtype=dt, device="cuda")}


_INPUTS = {"rope": _inputs_rope, "attention": _inputs_attention, "policy": _inputs_policy}


def prepare(case, seed):
    st = _INPUTS[case["op"]](case, seed)
    st["case"] = case
    if own:
        from laya_zig_b200 import gpu
        st["status"] = torch.zeros((1,), dtype=torch.int32, device="cuda")
        status = st["status"].data_ptr()
        if case["op"] == "rope":
            st["plan"] = gpu.RopePlan(head_dim=HEAD_DIM, rot_dim=case["rot_dim"], theta=THETA, layout=case["layout"],
                                      factor=case["factor"], original_len=case["original_len"])
        elif case["op"] == "attention":
            mask = 0 if st["mask"] is None else st["mask"].data_ptr()
            st["shape"] = gpu.AttentionShape(st["cu"].data_ptr(), case["n_seqs"], st["T"], case["max_len"],
                                             case["n_heads"], case["n_kv_heads"], status, window=case["window"],
                                             scale=HEAD_DIM ** -0.5, dtype=case["dtype"], token_mask_ptr=mask)
            if case["backward"]:
                nbytes = gpu.attention_backward_workspace(st["shape"])
                st["workspace"] = torch.empty((max(nbytes, 1),), dtype=torch.uint8, device="cuda")
        else:
            st["batch"] = gpu.PolicyBatch(st["cu"].data_ptr(), case["n"], st["G"], case["max_k"], status,
                                          qtypes_ptr=st["qtypes"].data_ptr(), temperature=TEMPERATURE,
                                          clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF,
                                          entropy_coef=ENTROPY_COEF, dtype=case["dtype"])
    return st


# ---------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "attention": _own_attention, "policy": _own_policy}[op](state)
    return {"rope": _plain_rope, "attention": _plain_attention, "policy": _plain_policy}[op](state)


def _own_rope(st):
    from laya_zig_b200 import gpu
    c = st["case"]
    by_row = st["positions"] is not None
    gpu.rope(st["plan"], st["x"].data_ptr(), st["x"].stride(0), st["y"].data_ptr(), st["y"].stride(0), st["T"],
             c["heads"], st["status"].data_ptr(), cu_seqlens_ptr=0 if by_row else st["cu"].data_ptr(),
             n_seqs=0 if by_row else c["n_seqs"], positions_ptr=st["positions"].data_ptr() if by_row else 0,
             inverse=c["inverse"], dtype=c["dtype"], stream=torch.cuda.current_stream().cuda_stream)
    return st["y"]


def _own_attention(st):
    from laya_zig_b200 import gpu
    c = st["case"]
    hq, hk = c["n_heads"], c["n_kv_heads"]
    stream = torch.cuda.current_stream().cuda_stream
    e = st["qkv"].element_size()
    ld, old = st["qkv"].stride(0), st["out"].stride(0)
    q = st["qkv"].data_ptr()
    k, v = q + hq * HEAD_DIM * e, q + (hq + hk) * HEAD_DIM * e
    gpu.attention(st["shape"], q, ld, k, ld, v, ld, st["out"].data_ptr(), old, st["lse"].data_ptr(), stream)
    if not c["backward"]:
        return {"out": st["out"], "lse": st["lse"]}
    dq = st["dqkv"].data_ptr()
    dk, dv = dq + hq * HEAD_DIM * e, dq + (hq + hk) * HEAD_DIM * e
    gpu.attention_backward(st["shape"], q, ld, k, ld, v, ld, st["out"].data_ptr(), old, st["lse"].data_ptr(),
                           st["dout"].data_ptr(), st["dout"].stride(0), dq, ld, dk, ld, dv, ld,
                           st["workspace"].data_ptr(), st["workspace"].numel(), stream)
    return {"out": st["out"], "lse": st["lse"], "dqkv": st["dqkv"]}


def _own_policy(st):
    from laya_zig_b200 import gpu
    gpu.policy_loss(st["batch"], st["logits"].data_ptr(), 0 if st["ref"] is None else st["ref"].data_ptr(),
                    st["actions"].data_ptr(), st["advantages"].data_ptr(), st["old"].data_ptr(),
                    st["grad"].data_ptr(), st["loss"].data_ptr(), st["logp"].data_ptr(), st["kl"].data_ptr(),
                    st["entropy"].data_ptr(), st["dlogits"].data_ptr(), torch.cuda.current_stream().cuda_stream)
    return {k: st[k] for k in ("loss", "logp", "kl", "entropy", "dlogits")}


def _frequencies(case):
    """Radians a position for each pair, in 64 bits. With original_len, pairs
    that turn often within it keep their frequency, those that hardly turn
    are stretched by `factor`, with a ramp between (32 turns and 1)."""
    r = case["rot_dim"]
    f = THETA ** (-torch.arange(0, r, 2, dtype=torch.float64, device="cuda") / r)
    if case["original_len"] == 0:
        return f / case["factor"]
    turns = case["original_len"] * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return f * keep + f / case["factor"] * (1.0 - keep)


def _positions(st):
    if st["positions"] is not None:
        return st["positions"].to(torch.int64)
    cu = st["cu"].to(torch.int64)
    t = torch.arange(st["T"], device="cuda")
    return t - cu[torch.searchsorted(cu, t, right=True) - 1]


def _plain_rope(st):
    c = st["case"]
    angle = _positions(st).to(torch.float64)[:, None] * _frequencies(c)[None, :]
    cos, sin = torch.cos(angle).float()[:, None, :], torch.sin(angle).float()[:, None, :]
    if c["inverse"]:
        sin = -sin
    r = c["rot_dim"]
    x = st["x"].reshape(st["T"], c["heads"], HEAD_DIM).float()
    y = x.clone()
    if c["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2] = a * cos - b * sin
        y[..., r // 2:r] = a * sin + b * cos
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2] = a * cos - b * sin
        y[..., 1:r:2] = a * sin + b * cos
    st["y"].copy_(y.reshape(st["T"], -1))
    return st["y"]


def _groups(lens, limit):
    """Runs of sequences to pad together: (first, count, longest)."""
    i = 0
    while i < len(lens):
        n, longest = 0, 0
        while i + n < len(lens):
            most = max(longest, lens[i + n])
            if n and (n + 1) * most * most > limit:
                break
            longest, n = most, n + 1
        yield i, n, longest
        i += n


def _plain_attention(st):
    c = st["case"]
    hq, hk, w = c["n_heads"], c["n_kv_heads"], c["window"]
    rep, scale, T = hq // hk, HEAD_DIM ** -0.5, st["T"]
    out = torch.zeros((T, hq * HEAD_DIM), device="cuda")
    lse_all = torch.full((T, hq), -math.inf, device="cuda")
    cu = st["cu"].to(torch.int64)
    grads = torch.zeros((T, (hq + 2 * hk) * HEAD_DIM), device="cuda") if c["backward"] else None
    for first, n, L in _groups(st["lens"], 8_000_000):
        at = cu[first:first + n, None] + torch.arange(L, device="cuda")[None, :]
        here = at < cu[first + 1:first + n + 1, None]
        at = at.clamp(max=T - 1)
        if st["mask"] is not None:
            here = here & (st["mask"][at] != 0)
        x = torch.where(here[..., None], st["qkv"][at].float(), 0.0).reshape(n, L, hq + 2 * hk, HEAD_DIM)
        x = x.transpose(1, 2)
        q = x[:, :hq].reshape(n, hk, rep, L, HEAD_DIM)
        k, v = x[:, hq:hq + hk, None], x[:, hq + hk:, None]
        if grads is not None:
            do = torch.where(here[..., None], st["dout"][at].float(), 0.0).reshape(n, L, hk, rep, HEAD_DIM)
            do = do.permute(0, 2, 3, 1, 4)
            dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        o, lse = torch.zeros_like(q), torch.full(q.shape[:-1], -math.inf, device="cuda")
        step = 1024
        for a in range(0, L, step):
            b = min(L, a + step)
            lo, hi = (0, L) if w < 0 else (max(0, a - w), min(L, b + w))
            see = here[:, a:b, None] & here[:, None, lo:hi]
            if w >= 0:
                i = torch.arange(a, b, device="cuda")[:, None]
                j = torch.arange(lo, hi, device="cuda")[None, :]
                see = see & ((i - j).abs() <= w)
            see = see[:, None, None]
            s = torch.matmul(q[..., a:b, :], k[..., lo:hi, :].transpose(-1, -2)) * scale
            s = torch.where(see, s, -math.inf)
            top = s.amax(-1, keepdim=True)
            top = torch.where(top > -math.inf, top, 0.0)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            o[..., a:b, :] = torch.matmul(p, v[..., lo:hi, :])
            lse[..., a:b] = (top + torch.log(total))[..., 0]
            if grads is not None:
                d = do[..., a:b, :]
                dp = torch.matmul(d, v[..., lo:hi, :].transpose(-1, -2))
                ds = p * (dp - (d * o[..., a:b, :]).sum(-1, keepdim=True)) * scale
                dq[..., a:b, :] = torch.matmul(ds, k[..., lo:hi, :])
                dk[..., lo:hi, :] += torch.matmul(ds.transpose(-1, -2), q[..., a:b, :]).sum(2, keepdim=True)
                dv[..., lo:hi, :] += torch.matmul(p.transpose(-1, -2), d).sum(2, keepdim=True)
        rows = at[here]
        out[rows] = o.reshape(n, hq, L, HEAD_DIM).transpose(1, 2).reshape(n, L, -1)[here]
        lse_all[rows] = lse.reshape(n, hq, L).transpose(1, 2)[here]
        if grads is not None:
            dx = torch.cat([dq.reshape(n, hq, L, HEAD_DIM), dk[:, :, 0], dv[:, :, 0]], 1)
            grads[rows] = dx.transpose(1, 2).reshape(n, L, -1)[here]
    st["out"].copy_(out)
    st["lse"].copy_(lse_all.t())
    if grads is None:
        return {"out": st["out"], "lse": st["lse"]}
    st["dqkv"].copy_(grads)
    return {"out": st["out"], "lse": st["lse"], "dqkv": st["dqkv"]}


def _plain_policy(st):
    c = st["case"]
    n, K = c["n"], c["max_k"]
    cu = st["cu"].to(torch.int64)
    col = torch.arange(K, device="cuda")[None, :]
    at = cu[:-1, None] + col
    here = at < cu[1:, None]
    at = at.clamp(max=st["G"] - 1)
    t = torch.tensor(TEMPERATURE, device="cuda")[st["qtypes"].to(torch.int64)][:, None]

    def log_probs(x):
        z = torch.where(here, x[at].float() / t, -math.inf)
        z = z - z.amax(-1, keepdim=True)
        return z - torch.log(torch.exp(z).sum(-1, keepdim=True))

    lp = log_probs(st["logits"])
    p = torch.exp(lp)
    lp0 = torch.where(p > 0, lp, 0.0)
    ent = -(p * lp0).sum(-1)
    if st["ref"] is not None:
        d = torch.where(p > 0, lp0 - log_probs(st["ref"]), 0.0)
        kl = (p * d).sum(-1)
    else:
        d, kl = torch.zeros_like(p), torch.zeros((n,), device="cuda")
    act = st["actions"].to(torch.int64)[:, None]
    logp = lp.gather(1, act)[:, 0]
    adv = st["advantages"]
    ratio = torch.exp(logp - st["old"])
    free, held = ratio * adv, ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv
    st["loss"].copy_(-torch.minimum(free, held) + KL_COEF * kl - ENTROPY_COEF * ent)
    st["logp"].copy_(logp)
    st["kl"].copy_(kl)
    st["entropy"].copy_(ent)
    g = torch.where(free <= held, -free, 0.0)[:, None]
    dz = g * ((col == act).float() - p)
    dz = dz + KL_COEF * p * (d - kl[:, None]) + ENTROPY_COEF * p * (lp0 + ent[:, None])
    dz = dz * st["grad"][:, None] / t
    st["dlogits"].copy_(dz[here])
    return {k: st[k] for k in ("loss", "logp", "kl", "entropy", "dlogits")}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    st = _INPUTS[case["op"]](case, seed)
    st["case"] = case
    return {"rope": _exact_rope, "attention": _exact_attention, "policy": _exact_policy}[case["op"]](st)


def _exact_rope(st):
    """Each pair as a complex number times e^(i angle)."""
    c = st["case"]
    r, parts = c["rot_dim"], []
    for i in range(r // 2):
        f = math.pow(THETA, -2.0 * i / r)
        if c["original_len"]:
            m = min(1.0, max(0.0, (c["original_len"] * f / (2 * math.pi) - 1.0) / 31.0))
            f = f * (m + (1.0 - m) / c["factor"])
        else:
            f = f / c["factor"]
        parts.append(-f if c["inverse"] else f)
    if st["positions"] is not None:
        pos = st["positions"].double()
    else:
        lens = (st["cu"][1:] - st["cu"][:-1]).tolist()
        pos = torch.cat([torch.arange(n, dtype=torch.float64, device="cuda") for n in lens])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.outer(pos, torch.tensor(parts, dtype=torch.float64, device="cuda")))[:, None, :]
    x = st["x"].double().reshape(st["T"], c["heads"], HEAD_DIM)
    head = x[..., :r]
    if c["layout"] == "half":
        z = torch.complex(head[..., :r // 2].contiguous(), head[..., r // 2:].contiguous()) * turn
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(head.reshape(st["T"], c["heads"], r // 2, 2).contiguous()) * turn
        head = torch.view_as_real(z).reshape(st["T"], c["heads"], r)
    return torch.cat([head, x[..., r:]], -1).reshape(st["T"], -1)


def _exact_attention(st):
    """Sequence by sequence over the tokens that are present, the gradients by
    differentiating the definition."""
    c = st["case"]
    hq, hk, w, T = c["n_heads"], c["n_kv_heads"], c["window"], st["T"]
    out = torch.zeros((T, hq * HEAD_DIM), dtype=torch.float64, device="cuda")
    lse = torch.full((hq, T), -math.inf, dtype=torch.float64, device="cuda")
    dqkv = torch.zeros((T, (hq + 2 * hk) * HEAD_DIM), dtype=torch.float64, device="cuda")
    start = 0
    for n in st["lens"]:
        rows = torch.arange(start, start + n, device="cuda")
        start += n
        if st["mask"] is not None:
            rows = rows[st["mask"][rows] != 0]
        m = rows.numel()
        if m == 0:
            continue
        x = st["qkv"][rows].double().reshape(m, hq + 2 * hk, HEAD_DIM).transpose(0, 1).contiguous()
        x.requires_grad_(c["backward"])
        gx = torch.zeros_like(x)
        step = 2048 if w < 0 else 512
        for a in range(0, m, step):
            b = min(m, a + step)
            pos = rows[a:b, None]
            near = torch.ones((b - a, m), dtype=torch.bool, device="cuda")
            lo, hi = 0, m
            if w >= 0:
                lo = int(torch.searchsorted(rows, rows[a] - w))
                hi = int(torch.searchsorted(rows, rows[b - 1] + w, right=True))
                near = (pos - rows[None, lo:hi]).abs() <= w
            k = x[hq:hq + hk, lo:hi].repeat_interleave(hq // hk, 0)
            v = x[hq + hk:, lo:hi].repeat_interleave(hq // hk, 0)
            s = torch.einsum("hid,hjd->hij", x[:hq, a:b], k) / math.sqrt(HEAD_DIM)
            s = s.masked_fill(~near, -math.inf)
            z = torch.logsumexp(s, -1)
            o = torch.einsum("hij,hjd->ihd", torch.exp(s - z[..., None]), v).reshape(b - a, -1)
            out[rows[a:b]] = o.detach()
            lse[:, rows[a:b]] = z.detach()
            if c["backward"]:
                gx += torch.autograd.grad(o, x, st["dout"][rows[a:b]].double())[0]
        if c["backward"]:
            dqkv[rows] = gx.transpose(0, 1).reshape(m, -1)
    if not c["backward"]:
        return {"out": out, "lse": lse}
    return {"out": out, "lse": lse, "dqkv": dqkv}


def _exact_policy(st):
    """The loss from its definition, its gradient by differentiating it."""
    cu = st["cu"].to(torch.int64)
    n = cu.numel() - 1
    owner = torch.repeat_interleave(torch.arange(n, device="cuda"), cu[1:] - cu[:-1])
    t = torch.tensor(TEMPERATURE, dtype=torch.float64, device="cuda")[st["qtypes"].to(torch.int64)]

    def total(v):
        return torch.zeros((n,), dtype=torch.float64, device="cuda").index_add(0, owner, v)

    def log_p(z):
        top = torch.full((n,), -math.inf, dtype=torch.float64, device="cuda")
        top = top.scatter_reduce(0, owner, z.detach(), "amax")
        return z - (top + torch.log(total(torch.exp(z - top[owner]))))[owner]

    alive = st["logits"] > -math.inf
    x = torch.where(alive, st["logits"].double(), -1e4).requires_grad_(True)
    lp = log_p(x / t[owner])
    p = torch.where(alive, torch.exp(lp), 0.0)
    ent = -total(p * lp)
    kl = torch.zeros((n,), dtype=torch.float64, device="cuda")
    if st["ref"] is not None:
        r = torch.where(alive, st["ref"].double(), -1e4)
        kl = total(p * (lp - log_p(r / t[owner])))
    logp = lp[cu[:-1] + st["actions"].to(torch.int64)]
    adv = st["advantages"].double()
    ratio = torch.exp(logp - st["old"].double())
    clipped = torch.clamp(ratio, 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH)
    loss = torch.maximum(-adv * ratio, -adv * clipped) + KL_COEF * kl - ENTROPY_COEF * ent
    dx = torch.autograd.grad((loss * st["grad"].double()).sum(), x)[0]
    return {"loss": loss.detach(), "logp": logp.detach(), "kl": kl.detach(), "entropy": ent.detach(), "dlogits": dx}


# ---------------------------------------------------------------- the work

def _pairs(case):
    """(query, key) pairs that see one another, absent tokens not deducted."""
    w, total = case["window"], 0
    for n in _lengths(case["n_seqs"], case["min_len"], case["max_len"], case["len_seed"]):
        if w < 0 or w >= n:
            total += n * n
        else:
            total += n * (2 * w + 1) - w * (w + 1)
    return total


def work(case):
    e = 4 if case["dtype"] == "F32" else 2
    if case["op"] == "rope":
        T = sum(_lengths(case["n_seqs"], case["min_len"], case["max_len"], case["len_seed"]))
        width = case["heads"] * HEAD_DIM
        return {"bytes": 2 * T * width * e + 4 * (T if case["positions"] else case["n_seqs"] + 1),
                "flops": 3 * T * case["heads"] * case["rot_dim"]}
    if case["op"] == "attention":
        T = sum(_lengths(case["n_seqs"], case["min_len"], case["max_len"], case["len_seed"]))
        hq, hk = case["n_heads"], case["n_kv_heads"]
        qkv, o, lse = T * (hq + 2 * hk) * HEAD_DIM * e, T * hq * HEAD_DIM * e, T * hq * 4
        small = 4 * (case["n_seqs"] + 1) + (T if case["mask"] else 0)
        product = 2 * HEAD_DIM * hq * _pairs(case)
        if not case["backward"]:
            return {"bytes": qkv + o + lse + small, "flops": 2 * product}
        return {"bytes": 2 * qkv + 2 * o + lse + small, "flops": 7 * product}
    n = case["n"]
    G = sum(_lengths(n, case["min_k"], case["max_k"], case["len_seed"]))
    return {"bytes": G * e * (3 if case["ref"] else 2) + n * (5 * 4 + 4 * 4) + 4 * (n + 1), "flops": 20 * G}
