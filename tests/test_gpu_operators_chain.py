"""The training-step operators one after the other, as a fine-tuning step uses
them on one layer and the option scorer: project, rotate, attend, score the
option markers, take the policy loss, and go back to the projection's output.
The middle (a linear scorer over the attention's output rows) is torch, the
rest is the library; the gradients are compared with the same chain
differentiated in 64 bits."""
import math

import numpy as np
import pytest

import op_reference as ref

pytestmark = pytest.mark.gpu

H, D = 12, 768


class Step:
    """Buffers of one step over a packed batch, and the calls it makes."""

    def __init__(self, lens, options, window, seed):
        import torch
        from laya_zig_b200 import gpu
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        bf = torch.bfloat16

        def rand(*s, scale=1.0):
            return scale * torch.randn(s, generator=g, device="cuda")
        self.lens, self.options, self.window = lens, options, window
        self.T, self.n, self.G = sum(lens), len(lens), sum(options)
        self.x, self.w = rand(self.T, D).to(bf), rand(3 * D, D, scale=0.05).to(bf)
        self.score_w = rand(D, scale=0.1)
        self.cu = torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32, device="cuda")
        self.cu_opt = torch.tensor([0] + np.cumsum(options).tolist(), dtype=torch.int32, device="cuda")
        r = np.random.default_rng(seed)
        rows = [s + r.choice(n, k, replace=False) for s, n, k in zip(np.cumsum([0] + lens[:-1]), lens, options)]
        self.markers = torch.tensor(np.concatenate(rows), device="cuda")
        self.actions = torch.tensor([r.integers(0, k) for k in options], dtype=torch.int32, device="cuda")
        self.adv = rand(self.n)
        self.old = torch.tensor([-math.log(k) for k in options], dtype=torch.float32, device="cuda")
        self.grad = torch.full((self.n,), 1.0, device="cuda")
        self.ref_logits = rand(self.G)
        z = dict(device="cuda")
        self.qkv32 = torch.zeros((self.T, 3 * D), **z)
        self.qkv = torch.zeros((self.T, 3 * D), dtype=bf, **z)
        self.out = torch.zeros((self.T, D), dtype=bf, **z)
        self.lse = torch.zeros((H, self.T), **z)
        self.logits, self.dlogits = torch.zeros(self.G, **z), torch.zeros(self.G, **z)
        self.loss = torch.zeros(self.n, **z)
        self.dout = torch.zeros((self.T, D), dtype=bf, **z)
        self.dqkv = torch.zeros((self.T, 3 * D), dtype=bf, **z)
        self.status = torch.zeros(1, dtype=torch.int32, **z)
        st = self.status.data_ptr()
        self.plan = gpu.RopePlan()
        self.shape = gpu.AttentionShape(self.cu.data_ptr(), self.n, self.T, max(lens), H, H, st, window=window)
        self.ws = torch.zeros(gpu.attention_backward_workspace(self.shape), dtype=torch.uint8, **z)
        self.batch = gpu.PolicyBatch(self.cu_opt.data_ptr(), self.n, self.G, max(options), st, kl_coef=0.1,
                                     entropy_coef=0.02)

    def run(self):
        import torch
        from laya_zig_b200 import gpu
        s = torch.cuda.current_stream().cuda_stream
        st, ld = self.status.data_ptr(), 3 * D
        gpu.linear(self.x.data_ptr(), self.w.data_ptr(), 0, self.qkv32.data_ptr(), self.T, 3 * D, D, "BF16", s)
        self.qkv.copy_(self.qkv32)
        q = self.qkv.data_ptr()
        # queries and keys lie side by side: 24 heads, in place
        gpu.rope(self.plan, q, ld, q, ld, self.T, 2 * H, st, cu_seqlens_ptr=self.cu.data_ptr(), n_seqs=self.n, stream=s)
        k, v = q + D * 2, q + 2 * D * 2
        gpu.attention(self.shape, q, ld, k, ld, v, ld, self.out.data_ptr(), D, self.lse.data_ptr(), s)
        self.logits.copy_(self.out[self.markers].float() @ self.score_w)
        gpu.policy_loss(self.batch, self.logits.data_ptr(), self.ref_logits.data_ptr(), self.actions.data_ptr(),
                        self.adv.data_ptr(), self.old.data_ptr(), self.grad.data_ptr(), self.loss.data_ptr(), 0, 0, 0,
                        self.dlogits.data_ptr(), s)
        self.dout.zero_()
        self.dout.index_copy_(0, self.markers, (self.dlogits[:, None] * self.score_w[None, :]).to(torch.bfloat16))
        d = self.dqkv.data_ptr()
        gpu.attention_backward(self.shape, q, ld, k, ld, v, ld, self.out.data_ptr(), D, self.lse.data_ptr(),
                               self.dout.data_ptr(), D, d, ld, d + D * 2, ld, d + 2 * D * 2, ld, self.ws.data_ptr(),
                               self.ws.numel(), s)
        gpu.rope(self.plan, d, ld, d, ld, self.T, 2 * H, st, cu_seqlens_ptr=self.cu.data_ptr(), n_seqs=self.n,
                 inverse=True, stream=s)

    def exact(self):
        """Loss and its gradient at the projection's output, in 64 bits."""
        import torch
        qkv = (self.x.double() @ self.w.double().t()).requires_grad_(True)
        pos = torch.cat([torch.arange(n, device="cuda") for n in self.lens])
        heads = qkv.reshape(self.T, 3 * H, 64)
        qk = ref.rope(heads[:, :2 * H], pos, ref.rope_frequencies(64))
        rows, at = [], 0
        for n in self.lens:
            sl = slice(at, at + n)
            at += n
            s = torch.einsum("ihd,jhd->hij", qk[sl, :H], qk[sl, H:]) / 8
            if self.window >= 0:
                i = torch.arange(n, device="cuda")
                s = s.masked_fill((i[:, None] - i[None, :]).abs() > self.window, -math.inf)
            rows.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), heads[sl, 2 * H:]).reshape(n, D))
        logits = torch.cat(rows)[self.markers] @ self.score_w.double()
        loss, at = [], 0
        for i, k in enumerate(self.options):
            loss.append(ref.policy(logits[at:at + k].cpu(), self.ref_logits[at:at + k].double().cpu(),
                                   int(self.actions[i]), float(self.adv[i]), float(self.old[i]), 1.0, 0.2, 0.2, 0.1,
                                   0.02)[0])
            at += k
        total = torch.stack(loss)
        return total.detach().cuda(), torch.autograd.grad(total.sum(), qkv)[0]


def _close(step):
    """The chain rounds eight times to bf16 on its way (projection, rotation, P,
    out, dout, dS, gradient, its rotation), each half a step of 2^-8 relative to
    what it rounds; a rounding early in the chain reaches the gradient through
    scores of magnitude ~1 (their error times P: a factor of at most 2). So the
    gradient's 2-norm is within 16 half steps, the losses (of logits near 1)
    within 16 half steps of their size plus 1."""
    import torch
    from laya_zig_b200 import gpu
    gpu.op_status(step.status.data_ptr())
    loss, g = step.exact()
    u = ref.half_step("BF16")
    assert ((step.loss.double() - loss).abs() <= 16 * u * (1 + loss.abs())).all()
    d = step.dqkv.double()
    assert torch.isfinite(d).all()
    assert ((d - g).norm() / g.norm()).item() <= 16 * u


@pytest.mark.parametrize("window", [-1, 64])
@pytest.mark.parametrize("lens,options", [([64], [4]), ([175, 180, 177], [4, 9, 3]), ([130, 1, 400, 67], [16, 1, 5, 2])])
def test_step(lens, options, window):
    s = Step(lens, options, window, seed=len(lens))
    s.run()
    _close(s)


def test_step_captured_and_replayed():
    """The whole step in one CUDA graph, replayed after its inputs changed:
    the same bits as the calls made one by one."""
    import torch
    lens, options = [175, 180, 177], [4, 9, 3]
    a, b = Step(lens, options, 64, seed=1), Step(lens, options, 64, seed=2)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        a.run()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        a.run()
    for name in ("x", "w", "score_w", "markers", "actions", "adv", "ref_logits"):
        getattr(a, name).copy_(getattr(b, name))
    g.replay()
    torch.cuda.synchronize()
    b.run()
    torch.cuda.synchronize()
    for name in ("loss", "dlogits", "out", "dqkv"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    _close(a)
