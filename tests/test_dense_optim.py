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
