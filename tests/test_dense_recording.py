"""Recording dpc_amd.dense.linear_fp8 into a graph beside a living eager autograd graph of the same leaf is refused, whatever the
leaf's strides."""
import pytest
import torch

from test_dense import bind, draw


@pytest.fixture(params=["compiled"])
def gpu(request, monkeypatch):
    import dpc_amd
    bind(monkeypatch, request.param)
    prev = dpc_amd._dense_capi.set_library(None)
    yield torch.device("cuda")
    dpc_amd._dense_capi.set_library(prev)


@pytest.mark.gpu
def test_recording_beside_a_living_eager_graph_is_refused_for_strided_leaves(gpu):
    import dpc_amd
    x, w, dy = (draw(s, i, torch.float32, gpu) for i, s in enumerate(((5, 24), (70, 24), (5, 70))))
    bias = draw((140,), 9, torch.float32, gpu)[::2]              # a strided leaf
    for t in (w, bias):
        t.requires_grad_()
    eager = dpc_amd.dense.linear_fp8(x, w, bias)
    want = torch.autograd.grad(eager, (w, bias), dy, retain_graph=True)
    only_bias = dpc_amd.dense.linear_fp8(x, w.detach(), bias)
    torch.cuda.synchronize()
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="earlier eager call of the same leaf"):
            dpc_amd.dense.linear_fp8(x, w, bias)
        with pytest.raises(RuntimeError, match="earlier eager call of the same leaf"):
            dpc_amd.dense.linear_fp8(x, w.detach(), bias)
        with torch.no_grad():
            z = dpc_amd.dense.linear_fp8(x, w, bias)
    refused.replay()
    assert torch.equal(z, eager)
    del eager, only_bias
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = dpc_amd.dense.linear_fp8(x, w, bias)
        y2 = dpc_amd.dense.linear_fp8(x, w, bias)
        got = torch.autograd.grad(y + 0 * y2, (w, bias), dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
