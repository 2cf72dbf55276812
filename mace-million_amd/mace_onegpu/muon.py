"""Orthogonalised updates of weight blocks: Newton-Schulz iteration on hand-written kernels, and the Muon optimizer.

    X = m / (|m|_F + eps),   steps times:  A = X X^T,   X <- a X + (b A + c A A) X

on every matrix of m [..., rows, columns] (expert blocks [E, D, F] are a batch), on its shorter side.  With the usual
coefficients five steps bring the singular values of m into about 0.7 .. 1.2 and leave its singular vectors: the update
of a step then moves all directions alike.  float32, bfloat16 or float16; norms are summed in 64 bits, iterates are
carried in float32, products take float16 operands (of float32 and float16 matrices two parts of each, 22 bits).
Where entries of X, of A or of b X + c A X pass 16, or those of b A + c A A 64, the result is infinite or NaN (the usual
coefficients keep all of them below 3; others may make singular values grow past 2).  A matrix with infinite or NaN
entries gives NaN and leaves the others alone; a matrix of zeros stays one.  A matrix's result has the same bits
whatever stands beside it.  Runs on torch's current stream, can be captured into a HIP graph, and needs the GPU: there
is no CPU path.  The reference has no counterpart.
"""
import math

import torch

from ._ops import ops

COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # as published with this optimizer (K. Jordan and others, 2024)


def orthogonalize(m, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """m after `steps` Newton-Schulz steps (module docstring), of m's shape and type, contiguous.  coefficients: (a, b,
    c), or one such triple for every step.  Matrices up to 65536 x 65536.  No derivative: raises RuntimeError for a
    tensor that requires one."""
    steps = int(steps)
    if steps < 0:
        raise ValueError(f"steps must be at least 0, got {steps}")
    c = [float(v) for t in coefficients for v in (t if hasattr(t, "__len__") else (t,))]
    if len(c) == 3 and not hasattr(coefficients[0], "__len__"):
        c = c * steps
    if len(c) != 3 * steps:
        raise ValueError(f"coefficients must be (a, b, c) or a triple for each of the {steps} steps")
    return ops().orthogonalize(m, c, eps)


class Muon(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised, for parameters [..., rows, columns]: matrices and batches of blocks.

        buf <- momentum buf + grad,   u = grad + momentum buf (nesterov) or buf
        p <- (1 - lr weight_decay) p - lr 0.2 sqrt(max(rows, columns)) orthogonalize(u)

    The factor gives an update a root mean square of about 0.2, what Adam's has, so that learning rates carry over and
    neither axis has to be the input's.  buf is float32; so is u, but for bfloat16 parameters, to whose type it is rounded
    (of the same range; float16's would overflow, or lose small gradients).  Vectors and scalars belong to another
    optimizer.  A step may be captured into a HIP graph once every parameter has taken one (RuntimeError before); the
    graph keeps lr and the other numbers of its capture."""

    def __init__(self, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=COEFFICIENTS, eps=1e-7):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError(f"lr {lr} and weight_decay {weight_decay} must be >= 0, momentum {momentum} in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coefficients=coefficients, eps=eps))

    def add_param_group(self, group):
        super().add_param_group(group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                del self.param_groups[-1]
                raise ValueError(f"Muon takes matrices and batches of them, got a parameter {tuple(p.shape)}")

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # torch casts a state to its parameter's type, which would round the float32 buffers of 16-bit parameters
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, i in zip(group["params"], saved["params"]):
                buf = state_dict["state"].get(i, {}).get("momentum_buffer")
                if buf is not None:
                    self.state[p]["momentum_buffer"] = buf.detach().to(p.device, torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state and p.is_cuda and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("Muon takes a step before it is captured: a momentum made inside a graph would be "
                                       "cleared by every replay")
                g = p.grad.float()
                if not state:
                    state["momentum_buffer"] = torch.zeros_like(g)
                buf = state["momentum_buffer"]
                buf.mul_(group["momentum"]).add_(g)
                u = g.add(buf, alpha=group["momentum"]) if group["nesterov"] else buf
                u = u if p.dtype == torch.float16 else u.to(p.dtype)
                o = orthogonalize(u, group["steps"], group["coefficients"], group["eps"])
                if group["weight_decay"]:
                    p.mul_(1 - group["lr"] * group["weight_decay"])
                p.add_(o, alpha=-group["lr"] * 0.2 * math.sqrt(max(p.shape[-2:])))
        return loss
