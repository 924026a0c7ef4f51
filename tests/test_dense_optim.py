"""dpc_amd.optim as a training program uses it: under torch's learning-rate schedulers, saved and loaded, with parameters that it cannot step;
on the CPU through the emulation of the kernels and on the GPU (-m gpu)."""
import pytest
import torch

from test_dense import draw, toy
from test_dense import dense_emulation  # noqa: F401  (a fixture)
from test_dense_ranks import device  # noqa: F401  (a fixture)


SCHEDULERS = {
    "StepLR": lambda opt: torch.optim.lr_scheduler.StepLR(opt, 2, 0.5),
    "CosineAnnealingLR": lambda opt: torch.optim.lr_scheduler.CosineAnnealingLR(opt, 4),
    "OneCycleLR": lambda opt: torch.optim.lr_scheduler.OneCycleLR(opt, 0.05, total_steps=6),       # moves the momentum as well
    "LambdaLR": lambda opt: torch.optim.lr_scheduler.LambdaLR(opt, lambda i: 0.9 ** i),
}


@pytest.mark.parametrize("rate", ["number", "tensor"])
@pytest.mark.parametrize("name", sorted(SCHEDULERS))
def test_muon_under_schedulers(device, name, rate):
    """the steps are those of muon_update with the rate and the momentum that the scheduler has set"""
    import dpc_amd
    w = draw((8, 12), 1, torch.float32, device).requires_grad_()
    twin, mom = w.detach().clone(), torch.zeros(8, 12, device=device)
    opt = dpc_amd.optim.Muon([w], lr=0.02 if rate == "number" else torch.tensor(0.02, device=device), weight_decay=0.1)
    scheduler = SCHEDULERS[name](opt)
    rates = []
    for i in range(4):
        w.grad = draw((8, 12), 10 + i, torch.float32, device)
        group = opt.param_groups[0]
        rates.append(float(group["lr"]))
        dpc_amd.dense.muon_update([twin], [w.grad], [mom], lr=group["lr"], momentum=group["momentum"], weight_decay=0.1)
        opt.step()
        scheduler.step()
        assert torch.equal(w.detach(), twin)
    assert len(set(rates)) > 1


@pytest.mark.parametrize("binding", ["compiled", "ctypes"])
def test_a_refused_update_moves_nothing(dense_emulation, monkeypatch, binding):  # noqa: F811
    """a matrix that the library refuses, behind others that would run in an earlier call of it: more than 40, or of another type"""
    import dpc_amd
    from test_dense import bind
    bind(monkeypatch, binding)
    prev = dpc_amd._dense_capi.set_library(dense_emulation)
    try:
        long = (1, (1 << 20) + 1)
        for count, dtype in ((1, torch.bfloat16), (40, torch.float32)):
            w = [draw((4, 5), i, torch.float32, "cpu") for i in range(count)] + [torch.ones(long, dtype=dtype)]
            g, m = [torch.ones_like(t) for t in w], [torch.zeros(t.shape) for t in w]
            before, versions = [t.clone() for t in w], [t._version for t in w + m]
            with pytest.raises(dpc_amd.DpcError):
                dpc_amd.dense.muon_update(w, g, m, lr=0.1)
            assert all(torch.equal(a, b) for a, b in zip(w, before)) and not any(bool(t.any()) for t in m)
            assert [t._version for t in w + m] == versions          # graphs that hold them may still run backward
            with pytest.raises(dpc_amd.DpcError):
                dpc_amd.dense.newton_schulz(w)
        dpc_amd.dense.muon_update(w[:2], g[:2], m[:2], lr=0.1)
        assert not torch.equal(w[0], before[0])
    finally:
        dpc_amd._dense_capi.set_library(prev)


def test_parameters_that_no_step_takes_are_refused_at_once():
    from importlib import import_module
    Muon = import_module("differentiable-point-clouds_amd.optim").Muon
    P = torch.nn.Parameter
    good = P(torch.ones(4, 5))
    bad = [P(torch.ones(5)), P(torch.ones(5, 4).t()), P(torch.ones(2, 3, 4, 4, 4).to(memory_format=torch.channels_last_3d)),
           P(torch.ones(4, 5, dtype=torch.float64))]
    opt = Muon([good])
    for p in bad:
        with pytest.raises((TypeError, ValueError)):
            Muon([p])
        with pytest.raises((TypeError, ValueError)):
            opt.add_param_group({"params": [p]})
        assert len(opt.param_groups) == 1 and opt.param_groups[0]["params"] == [good]
    opt.add_param_group({"params": P(torch.ones(2, 3, 4, 4).to(memory_format=torch.channels_last)), "lr": 0.1})
    assert [g["lr"] for g in opt.param_groups] == [0.02, 0.1]


def test_loaded_state_takes_the_place_of_the_old(device):
    """momenta and a rate on the device keep their memory, which a recorded step reads and writes"""
    import dpc_amd
    make = lambda: draw((8, 12), 1, torch.float32, device).requires_grad_()
    w, other = make(), make()
    lr = torch.tensor([0.02], device=device)
    opt, fresh = dpc_amd.optim.Muon([w], lr=lr), dpc_amd.optim.Muon([other], lr=0.5)
    untouched = fresh.state_dict()
    for p, o in ((w, opt), (other, fresh)):
        p.grad = draw((8, 12), 2, torch.float32, device)
        o.step()
    where = opt.state[w]["momentum_buffer"].data_ptr()
    for saved, rate in ((fresh.state_dict(), 0.5), (opt.state_dict(), 0.5), (untouched, 0.5)):
        opt.load_state_dict(saved)
        assert opt.param_groups[0]["lr"] is lr and float(lr) == rate
        assert opt.state[w]["momentum_buffer"].data_ptr() == where
        want = fresh.state[other]["momentum_buffer"] if saved is not untouched else torch.zeros(8, 12, device=device)
        assert torch.equal(opt.state[w]["momentum_buffer"], want)
    fresh.load_state_dict(opt.state_dict())                    # a number takes the loaded rate as it comes
    assert float(fresh.param_groups[0]["lr"]) == 0.5


@pytest.mark.gpu
def test_recorded_steps_go_on_with_loaded_state(monkeypatch):
    import copy
    import dpc_amd
    from test_dense import bind
    bind(monkeypatch, "compiled")
    gpu = torch.device("cuda")
    prev = dpc_amd._dense_capi.set_library(None)
    try:
        net, x = toy(dpc_amd, gpu), draw((5, 24), 1, torch.float32, gpu)
        lr = torch.full((1,), 0.02, device=gpu)
        opt = dpc_amd.optim.Muon([net[0].weight, net[2].weight], lr=lr)

        def step():
            opt.zero_grad()
            loss = net(x).square().sum()
            loss.backward()
            opt.step()
            return loss.detach()
        recorded = dpc_amd.graphs.RecordedStep(step, device=gpu, warmup=3)
        recorded()
        torch.cuda.synchronize()
        weights, state = copy.deepcopy(net.state_dict()), copy.deepcopy(opt.state_dict())
        runs = []
        for _ in range(3):
            lr.fill_(0.7)                                      # what loading has to take back
            net.load_state_dict(weights)
            opt.load_state_dict(state)
            losses = [recorded().clone() for _ in range(3)]
            torch.cuda.synchronize()
            runs.append(losses + [p.detach().clone() for p in net.parameters()])
        for run in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(run, runs[0]))
    finally:
        dpc_amd._dense_capi.set_library(prev)
