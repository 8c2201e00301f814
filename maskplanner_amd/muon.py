"""Muon: momentum orthogonalised by Newton-Schulz products, for the weights that are matrices (csrc/muon.hip), and the pairing with DenseAdam
that drives a whole model: a convolution or Linear weight is a matrix (first axis by the rest), norms and biases are Adam's."""
import torch

from . import ops


class Muon(torch.optim.Optimizer):
    """m <- m + (1 - momentum)(g - m),  u = g + momentum (m - g) (nesterov) or m,  p <- (1 - lr weight_decay) p - lr s orthogonalize(u).

    scale: "original" s = sqrt(max(1, rows / columns)), "match_rms" s = 0.2 sqrt(max(rows, columns)) (an update of Adam's usual size), None 1.
    Parameters: contiguous HIP tensors of at least two axes, float32, float16 or bfloat16, gradients of the same type.  The momentum
    (`momentum_buffer`) is float32 whatever the parameter's type.  All parameters of one group and type go through each stage in one launch.
    The learning rate is fixed in a recorded graph; one step has to come before the recording."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, scale="original", steps=5, coefficients=ops.NEWTON_SCHULZ,
                 eps=1e-7):
        if not lr >= 0 or not 0 <= momentum < 1 or not weight_decay >= 0:
            raise ValueError("Muon: lr and weight_decay must not be negative, momentum lies in [0, 1)")
        if scale not in ops.MUON_SCALES:
            raise ValueError(f"Muon: scale is one of {list(ops.MUON_SCALES)}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, scale=scale, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.ndim < 2 or p.dtype not in ops._DTYPE or not p.is_contiguous():
                self.param_groups.pop()
                raise ValueError("Muon updates contiguous float32, float16 or bfloat16 parameters of at least two axes (give norms and biases to Adam)")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for g in self.param_groups:
            kinds = {}
            for p in g["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                st = self.state[p]
                if "momentum_buffer" not in st:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon: take one step before recording a graph (a momentum made inside it would be zeroed by every replay)")
                    st["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                kinds.setdefault((p.device, p.dtype), []).append((p, p.grad, st["momentum_buffer"]))
            for rows in kinds.values():
                ops.muon_step(*zip(*rows), lr=g["lr"], momentum=g["momentum"], nesterov=g["nesterov"], weight_decay=g["weight_decay"], scale=g["scale"],
                              steps=g["steps"], coefficients=g["coefficients"], eps=g["eps"])
        return loss

    def load_state_dict(self, state_dict):
        """torch.optim.Optimizer.load_state_dict casts floating-point state to the parameter's type: the momentum is taken again in float32."""
        super().load_state_dict(state_dict)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
            m = state_dict["state"].get(i, {}).get("momentum_buffer")
            if m is not None:
                self.state[p]["momentum_buffer"] = m.detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()


class MuonAdam:
    """Muon for `matrices`, factor_heads.DenseAdam for `others`, as one optimizer with DenseAdam's interface (`step_dev`, `state`,
    step(ticked)).  Like DenseAdam it has no param_groups and no state_dict: rates are scheduled and momenta saved on `muon`, which is a
    torch.optim.Optimizer; Adam's part is in `state` and `step_dev`."""

    def __init__(self, matrices, others, lr=1e-3, muon_lr=0.02, capturable=False, **muon):
        from .factor_heads import DenseAdam
        self.muon = Muon(list(matrices), lr=muon_lr, **muon)
        self.adam = DenseAdam(list(others), lr=lr, capturable=capturable)
        self.params = [p for g in self.muon.param_groups for p in g["params"]] + self.adam.params

    @property
    def step_dev(self):
        return self.adam.step_dev

    @property
    def state(self):
        return {**self.muon.state, **self.adam.state}

    def step(self, ticked=False):
        self.adam.step(ticked=ticked)
        self.muon.step()

    def zero_grad(self, set_to_none=True):
        self.muon.zero_grad(set_to_none)
        self.adam.zero_grad(set_to_none)
