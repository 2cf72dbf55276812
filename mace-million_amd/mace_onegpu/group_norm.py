"""Group norm with an activation over structures of atoms (batches of rows), channels last, forward and backward.

    h = (x - mean) / sqrt(mean((x - mean)^2) + eps),   y = act(h * weight + bias)

mean over the rows of a structure and the C / groups channels of a group.  x: float32, bfloat16 or float16, either
[structures, ..., C], every structure of the same number of rows, or [rows, C] with offsets [structures + 1] (int32 or
int64, ascending): structure s has the rows offsets[s] .. offsets[s + 1] - 1, possibly none; rows before the first and
behind the last structure give zeros and get zero gradients.  Rows may be strided and are read in place where the last
axis is contiguous.  weight and bias: [C], of x's type or float32, either may be None; activation: None, "silu" or "gelu"
(with erf).  Means, variances and the gradients' sums are float32, in a fixed order: the same bits in every run.  Groups
hold up to 16384 bytes of channels.  Differentiable once in x, weight and bias.  Runs on torch's current stream without
reading anything back (also of ragged structures), can be captured into a HIP graph, and needs the GPU: there is no CPU
path.  The reference has no counterpart.
"""
import torch

from ._ops import ops


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None, offsets=None):
    """Group norm of x [structures, ..., C], or [rows, C] with offsets, and an activation (module docstring)."""
    return ops().group_norm(x, groups, weight, bias, eps, activation, offsets)


class GroupNorm(torch.nn.Module):
    """group_norm with learned weight (ones at first) and bias (zeros)."""

    def __init__(self, groups, channels, eps=1e-5, activation=None, dtype=torch.float32, device=None):
        super().__init__()
        self.groups, self.eps, self.activation = int(groups), float(eps), activation
        self.weight = torch.nn.Parameter(torch.ones(channels, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(channels, dtype=dtype, device=device))

    def forward(self, x, offsets=None):
        return group_norm(x, self.groups, self.weight, self.bias, self.eps, self.activation, offsets)
