"""What the attention operator's backward pass reads of its own workspace is
complete before it reads it: one kernel that waits for the one before it, and
calls that share a workspace give what they give alone."""
import ctypes

import pytest

from test_gpu_attention_op import Problem

pytestmark = pytest.mark.gpu


def _nodes(graph):
    """Node types of a captured graph (CUgraphNodeType: 0 is a kernel)."""
    cuda = ctypes.CDLL("libcuda.so.1")
    n = ctypes.c_size_t(0)
    assert cuda.cuGraphGetNodes(ctypes.c_void_p(graph), None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert cuda.cuGraphGetNodes(ctypes.c_void_p(graph), nodes, ctypes.byref(n)) == 0
    types = []
    for x in nodes:
        t = ctypes.c_int(-1)
        assert cuda.cuGraphNodeGetType(ctypes.c_void_p(x), ctypes.byref(t)) == 0
        types.append(t.value)
    return types


@pytest.mark.parametrize("hq,hk", [(4, 4), (6, 2)])
def test_long_backward_is_delta_and_one_kernel(hq, hk):
    """dQ and dK/dV are one launch, which waits for delta by the stream's own
    order (griddepcontrol.wait): no kernel reads what a kernel two places before
    it wrote without such a wait."""
    import torch
    p = Problem([700, 33, 300], hq=hq, hk=hk)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        p.run(s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g, stream=s):
        p.backward(s.cuda_stream)
    assert _nodes(g.raw_cuda_graph()) == [0, 0]
    p.dqkv.fill_(7.0)
    p.ws.fill_(255)
    g.replay()
    torch.cuda.synchronize()
    p.check()


@pytest.mark.parametrize("hq,hk", [(4, 4), (6, 2)])
def test_workspace_of_the_call_before(hq, hk):
    """Two problems of the same shape in turn on one workspace, so that every
    word of delta has a plausible old value, back to back many times."""
    import torch
    ps = [Problem([260, 700, 31, 180], hq=hq, hk=hk, seed=i) for i in range(2)]
    for p in ps:
        p.run()
        p.check()
    want = [p.dqkv.clone() for p in ps]
    ps[1].ws = ps[0].ws
    kept = [torch.empty_like(w) for w in want]
    for _ in range(40):
        for p, k in zip(ps, kept):
            p.backward()
            k.copy_(p.dqkv)
            p.dqkv.fill_(7.0)
        torch.cuda.synchronize()
        for k, w in zip(kept, want):
            assert torch.equal(k, w)


@pytest.mark.parametrize("lens,window", [([64], 2), ([33, 40, 64], 0), ([50] * 5, 4)])
def test_short_sequences_in_a_narrow_window_are_one_launch(lens, window):
    """Their blocks have all of delta at hand."""
    import torch
    p = Problem(lens, window=window)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        p.run(s.cuda_stream)
    s.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g, stream=s):
        p.backward(s.cuda_stream)
    assert _nodes(g.raw_cuda_graph()) == [0]
    torch.cuda.synchronize()
    p.check()
