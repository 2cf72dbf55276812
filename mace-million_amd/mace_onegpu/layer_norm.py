"""Layer norm over the last axis on hand-written kernels, forward and backward.

    y = (x - mean) / sqrt(mean((x - mean)^2) + eps) * weight + bias

x: float32, bfloat16 or float16, [..., D] with D up to 16384; rows may be strided (the scalar component h[:, 0, :] of
ir_mul features) and are read in place when the last axis is contiguous.  weight and bias: [D], of x's type or float32,
either may be None.  Means, variances and the gradients' sums are float32.  Backward gives dx, dweight (summed over the
rows in a fixed order: the same bits in every run) and dbias.  Runs on torch's current stream, can be captured into a HIP
graph, and needs the GPU: there is no CPU path.  The reference has no counterpart.
"""
import ctypes

import torch

from ._lib import K, stream

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_DIM = 16384


def check_gpu(t, name):
    """t must be a float32 / bfloat16 / float16 tensor of the current GPU; its dtype code."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a GPU tensor")
    if t.dtype not in DTYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    return DTYPES[t.dtype]


def _rows(t):
    """(t or a copy of it as [rows, D] with a contiguous last axis, distance of rows)."""
    D = t.shape[-1]
    if t.dim() != 2:
        t = t.reshape(-1, D)
    if t.shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else D


def _check(x, weight, bias):
    code = check_gpu(x, "x")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., D] with D > 0, got {tuple(x.shape)}")
    if x.shape[-1] > MAX_DIM:
        raise ValueError(f"rows of more than {MAX_DIM} values are not supported, got {x.shape[-1]}")
    p_code = code
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        p_code = check_gpu(p, name)
        if p.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be {x.dtype} (as x) or float32, got {p.dtype}")
        if p.shape != x.shape[-1:]:
            raise ValueError(f"{name} must be [{x.shape[-1]}], got {tuple(p.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    return code, p_code


def _forward(x, weight, bias, eps, codes, stats):
    x2, ldx = _rows(x)
    rows, D = x2.shape
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    weight = weight.contiguous() if weight is not None else None
    bias = bias.contiguous() if bias is not None else None
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    K.mm_layernorm_fwd(x2, ldx, codes[0], rows, D, weight, bias, codes[1], eps, y, D, mean, rstd, stream())
    return y, x2, ldx, mean, rstd


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, codes):
        y, x2, ctx.ldx, mean, rstd = _forward(x, weight, bias, eps, codes, True)
        ctx.save_for_backward(x2, weight, bias, mean, rstd)
        ctx.codes, ctx.shape = codes, x.shape
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        nx, nw, nb = ctx.needs_input_grad[:3]
        rows, D = x.shape
        dy, lddy = _rows(dy)
        code, p_code = ctx.codes
        dx = torch.empty(ctx.shape, dtype=x.dtype, device=x.device) if nx else None
        dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if nw else None
        db = torch.empty_like(bias, memory_format=torch.contiguous_format) if nb else None
        ws = None
        if nw or nb:
            nbytes = ctypes.c_size_t(0)
            K.mm_layernorm_workspace(rows, D, code, ctypes.byref(nbytes))
            ws = torch.empty(nbytes.value // 4, dtype=torch.float32, device=x.device)
        K.mm_layernorm_bwd(dy, lddy, x, ctx.ldx, code, rows, D, weight.contiguous() if weight is not None else None,
                           p_code, mean, rstd, dx, D, dw, db, ws, stream())
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of x [..., D] over its last axis (module docstring); differentiable in x, weight and bias."""
    codes = _check(x, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNormFn.apply(x, weight, bias, float(eps), codes)
    return _forward(x, weight, bias, float(eps), codes, False)[0]


class LayerNorm(torch.nn.Module):
    """layer_norm with learned weight (ones at first) and bias (zeros) over rows of dim values."""

    def __init__(self, dim, eps=1e-5, dtype=torch.float32, device=None):
        super().__init__()
        self.eps = float(eps)
        self.weight = torch.nn.Parameter(torch.ones(dim, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(dim, dtype=dtype, device=device))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)
