"""Optimisers for the networks around the projector, beside the gradient buckets of ``distributed`` and the recorded steps of
``graphs`` (the reference trains with stock Adam: dpc/run/train.py:91-92).

    opt = muon_with_adam(net, lr=0.02, adam_lr=1e-4)      # matrices by Muon, everything else by torch.optim.Adam
    loss.backward(); opt.step()"""
import torch

from . import dense


class Muon(torch.optim.Optimizer):
    """Momentum, orthogonalised by Newton-Schulz products, as the step of every matrix (``dense.muon_update``, whose arguments
    these are).  Parameters of two or more dimensions only: a convolution's filter counts as [out channels, the rest].  All
    matrices of a group step in the same launches; the momentum is float32 whatever the parameter's type.

    The step only enqueues work, so it can be recorded (``graphs.RecordedStep``): ``lr`` may be a one-element float32 tensor on
    the device, which a recorded step reads anew at each replay; the momenta must exist before the recording begins (one
    eager step makes them)."""

    # of a group, what the update takes; schedulers keep settings of their own there (initial_lr, max_momentum)
    _SETTINGS = ("lr", "momentum", "nesterov", "weight_decay", "steps", "coefficients", "eps", "adjust")

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=dense.COEFFICIENTS,
                 eps=1e-7, adjust="rms"):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps, adjust=adjust))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            for p in self.param_groups[-1]["params"]:
                dense._code(p, "a parameter")
                if p.dim() < 2:
                    raise ValueError("Muon takes matrices; a parameter of shape %s belongs to another optimiser" % (tuple(p.shape),))
                if dense._matrix_format(p) is None:
                    raise ValueError("Muon takes parameters that are contiguous or channels_last, got strides %s of shape %s"
                                     % (p.stride(), tuple(p.shape)))
        except (TypeError, ValueError):
            self.param_groups.pop()
            raise

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise ValueError("Muon does not take sparse gradients")
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon: the momenta must exist before a recording begins (run one step eagerly)")
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
                by_device.setdefault(p.device, []).append((p, p.grad, state["momentum_buffer"]))
            for entries in by_device.values():
                dense.muon_update(*zip(*entries), **{k: group[k] for k in self._SETTINGS if k in group})
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Momenta and rates that exist keep their memory, so that a recorded step goes on with what was loaded."""
        momenta = {p: s["momentum_buffer"] for p, s in self.state.items() if "momentum_buffer" in s}
        rates = [g["lr"] for g in self.param_groups]
        super().load_state_dict(state_dict)
        # the base class casts state to the parameter's type; momenta stay float32
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            saved, kept = state_dict["state"].get(i, {}).get("momentum_buffer"), momenta.get(p)
            if saved is None and kept is None:
                continue
            if kept is None:
                kept = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            self.state[p]["momentum_buffer"] = kept.zero_() if saved is None else kept.copy_(saved)
        for group, rate in zip(self.param_groups, rates):
            if isinstance(rate, torch.Tensor):
                group["lr"] = rate.copy_(torch.as_tensor(group["lr"]).reshape(rate.shape))


class Together(object):
    """Several optimisers over different parameters, stepped as one."""

    def __init__(self, *optimizers):
        self.optimizers = optimizers

    @property
    def param_groups(self):
        return [g for o in self.optimizers for g in o.param_groups]

    def step(self):
        for o in self.optimizers:
            o.step()

    def zero_grad(self, set_to_none=True):
        for o in self.optimizers:
            o.zero_grad(set_to_none=set_to_none)

    def state_dict(self):
        return {"optimizers": [o.state_dict() for o in self.optimizers]}

    def load_state_dict(self, state_dict):
        if len(state_dict["optimizers"]) != len(self.optimizers):
            raise ValueError("state of %d optimisers for %d" % (len(state_dict["optimizers"]), len(self.optimizers)))
        for o, s in zip(self.optimizers, state_dict["optimizers"]):
            o.load_state_dict(s)


def muon_with_adam(net, lr=0.02, adam_lr=1e-4, adam=None, **muon):
    """Muon over the matrices of ``net`` (filters of convolutions among them), torch.optim.Adam over its other parameters; ``adam``:
    further arguments of Adam (``capturable``, ``fused``), the rest goes to Muon."""
    params = [p for p in net.parameters() if p.requires_grad]
    matrices, others = [p for p in params if p.dim() >= 2], [p for p in params if p.dim() < 2]
    made = [Muon(matrices, lr=lr, **muon)] if matrices else []
    if others:
        made.append(torch.optim.Adam(others, lr=adam_lr, **(adam or {})))
    return Together(*made)
