"""Recording dpc_amd.dense.linear_fp8 into a graph beside a living eager autograd graph of the same leaf is refused by both bindings; the
ctypes binding's question is tried on the CPU with a stream that only pretends to record."""
import pytest
import torch

from test_dense import bind, draw, emulated, dense_emulation  # noqa: F401  (fixtures)


@pytest.fixture(params=["compiled", "ctypes"])
def gpu(request, monkeypatch):
    import dpc_amd
    bind(monkeypatch, request.param)
    prev = dpc_amd._dense_capi.set_library(None)
    yield torch.device("cuda")
    dpc_amd._dense_capi.set_library(prev)


def test_a_living_graph_is_seen_through_its_accumulator(dense_emulation, monkeypatch):
    import dpc_amd
    bind(monkeypatch, "ctypes")
    prev = dpc_amd._dense_capi.set_library(dense_emulation)
    try:
        dense = dpc_amd.dense
        x, w, bias = draw((5, 24), 1, torch.float32, "cpu"), draw((7, 24), 2, torch.float32, "cpu"), draw((14,), 3, torch.float32, "cpu")[::2]
        for t in (x, w, bias):
            t.requires_grad_()
        call = lambda: dense.linear_fp8(x, w, bias)
        want = call().detach()
        stream = [None]
        monkeypatch.setattr(dense, "_recording_stream", lambda lib, device: stream[0], raising=False)
        for alive in (lambda: call(), lambda: w * 2, lambda: bias.sum(), lambda: torch.nn.functional.linear(x, w)):
            stream[0] = None
            eager = alive()
            stream[0] = 7
            for _ in range(2):                                   # asking leaves nothing behind that would let the next call pass
                with pytest.raises(RuntimeError, match="earlier eager call of the same leaf"):
                    call()
            with torch.no_grad():
                assert torch.equal(call(), want)
            del eager
            first = call()
            second = call()                                      # the leaves' graph lives, but this recording made it
            assert torch.equal(first, want) and torch.equal(second, want)
            stream[0] = 9                                        # another recording, the first one's graph still alive
            with pytest.raises(RuntimeError, match="earlier eager call of the same leaf"):
                call()
            del first, second
            grads = torch.autograd.grad(call(), (x, w, bias), torch.ones(5, 7))
            assert all(g.shape == t.shape for g, t in zip(grads, (x, w, bias)))
    finally:
        dpc_amd._dense_capi.set_library(prev)


@pytest.mark.gpu
def test_recording_beside_a_living_eager_graph_is_refused_by_both_bindings(gpu):
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


@pytest.mark.gpu
@pytest.mark.parametrize("gather", ["none", "accumulate", "copy"])
def test_a_recorded_training_step_through_either_binding(gpu, gather):
    """8-bit layers, gradient buckets and Muon in one graph: nothing of an eager step is alive, so nothing is refused"""
    import dpc_amd
    from test_dense import toy
    finals = []
    for recorded in (False, True):
        net, x = toy(dpc_amd, gpu), draw((5, 24), 1, torch.float32, gpu)
        opt = dpc_amd.optim.Muon([net[0].weight, net[2].weight], lr=torch.full((1,), 0.02, device=gpu))
        red = dpc_amd.distributed.GradBuckets(net.parameters(), bucket_mb=0.001, gather=gather) if gather != "none" else None

        def step():
            if red is None:
                opt.zero_grad()
            loss = net(x).square().sum()
            loss.backward()
            if red is not None:
                red.finish()
            opt.step()
            if red is not None:
                red.zero_()
            return loss.detach()
        if recorded:
            run = dpc_amd.graphs.RecordedStep(step, device=gpu, warmup=3)
        else:
            run = step
            for _ in range(3):
                step()
        losses = []
        for _ in range(3):
            losses.append(run().clone())
            torch.cuda.synchronize()
        finals.append(losses + [p.detach().clone() for p in net.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*finals))
