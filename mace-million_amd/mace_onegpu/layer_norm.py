"""Layer norm over the last axis on hand-written kernels, forward and backward.

    y = (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias

x: float32, bfloat16 or float16, [..., D] with D up to 16384; rows may be strided (the scalar component h[:, 0, :] of
ir_mul features) and are read in place when the last axis is contiguous.  weight and bias: [D], of x's type or float32,
either may be None.  Means, variances and the gradients' sums are float32.  Backward gives dx, dweight (summed over the
rows in a fixed order: the same bits in every run) and dbias, once (no second derivative).  Runs on torch's current
stream, can be captured into a HIP graph, and needs the GPU: there is no CPU path.  The reference has no counterpart.
"""
import torch

from ._ops import ops


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x [..., D] over its last axis (module docstring); differentiable in x, weight and bias."""
    return ops().layer_norm(x, weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """layer_norm with learned weight (ones at first) and bias (zeros) over rows of dim values."""

    def __init__(self, dim, eps=1e-5, dtype=torch.float32, device=None):
        super().__init__()
        self.eps = float(eps)
        self.weight = torch.nn.Parameter(torch.ones(dim, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(dim, dtype=dtype, device=device))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
