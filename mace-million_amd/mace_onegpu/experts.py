"""Mixtures of expert weight blocks: routing of rows (atoms, tokens) to experts and the gated products with their blocks.

The species-block linears of the model multiply every node row by the block of its species.  Here a row gets k of E blocks
with gates that are learned:

    gates, experts = route(logits, k)                        # [T, E] -> float32 [T, k], int32 [T, k]
    plan = plan_experts(experts, E)                          # the (row, choice) slots sorted by expert
    y = expert_linear(x, weight, plan, gates)                # y[t] = sum_j gates[t, j] x[t] @ weight[experts[t, j]]

All three run hand-written kernels on torch's current stream without reading anything back, so that a chain of them can
be captured into a HIP graph; they need the GPU.  Results are the same bits in every run (no float atomics).  x and weight
(and the logits on their own) are float32, bfloat16 or float16; gates are float32, and sums are float32 whatever the type.
The reference has no counterpart; its nearest operation is SpeciesSkip (fast_layers.py:41-105).
"""
import ctypes

import torch

from ._lib import K, stream
from .layer_norm import check_gpu

MAX_EXPERTS = 1024
MAX_K = 32
MAX_GROUPS = 64
SCORING = {"softmax": 0, "sigmoid": 1}
INT32_MAX = 2 ** 31 - 1


# ------------------------------------------------------------------------------------------------ routing
class _RouteFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, args):
        gates, experts, logits = _route(logits, bias, args)
        ctx.save_for_backward(logits, gates, experts)
        ctx.args = args
        ctx.mark_non_differentiable(experts)
        return gates, experts

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dgates, _):
        logits, gates, experts = ctx.saved_tensors
        code, k, scoring, groups, top_groups, renormalize, scale = ctx.args
        T, E = logits.shape
        dlogits = torch.empty(T, E, dtype=logits.dtype, device=logits.device)
        K.mm_route_bwd(logits, logits.stride(0) if T > 1 else E, code, T, E, k, scoring, renormalize, scale, gates,
                       experts, dgates.contiguous(), dlogits, stream())
        return dlogits, None, None


def _route(logits, bias, args):
    code, k, scoring, groups, top_groups, renormalize, scale = args
    T, E = logits.shape
    if (E > 1 and logits.stride(1) != 1) or (T > 1 and logits.stride(0) < E):
        logits = logits.contiguous()
    gates = torch.empty(T, k, dtype=torch.float32, device=logits.device)
    experts = torch.empty(T, k, dtype=torch.int32, device=logits.device)
    K.mm_route_fwd(logits, logits.stride(0) if T > 1 else E, code, T, E, k, scoring, bias, groups, top_groups,
                   renormalize, scale, gates, experts, stream())
    return gates, experts, logits


def route(logits, k, scoring="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0):
    """(gates float32 [T, k], experts int32 [T, k]): the k experts of largest key = logit + bias of every row, in
    descending order of the key, ties to the lowest index.

    logits [T, E]: -inf closes an expert to a row; a slot without an open expert gets expert -1 and gate 0 (a row with
    nothing open: all slots).  A NaN logit is chosen first and makes the row's gates NaN.
    scoring: "softmax" (over the row's E logits) or "sigmoid" (of each).
    bias float32 [E]: moves the choice (balance of the experts' load) and not the gates; no gradient.  It is added to the
        logits, of which both scores are monotone functions.
    groups, top_groups: the E experts in `groups` equal runs, of which only the top_groups with the largest keys are open.
    renormalize: gates = scale * score / sum of the chosen scores, finite also where all scores underflow; else
        gates = scale * score.
    Differentiable in logits."""
    code = check_gpu(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [rows, experts], got {tuple(logits.shape)}")
    E, k, groups = logits.shape[1], int(k), int(groups)
    if E > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts are supported, got {E}")
    if not 1 <= k <= min(E, MAX_K):
        raise ValueError(f"k must be 1 .. {min(E, MAX_K)}, got {k}")
    if scoring not in SCORING:
        raise ValueError(f"scoring must be one of {sorted(SCORING)}, got {scoring!r}")
    if not 1 <= groups <= MAX_GROUPS or E % groups:
        raise ValueError(f"groups must divide the {E} experts and be at most {MAX_GROUPS}, got {groups}")
    top_groups = groups if top_groups is None else int(top_groups)
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top_groups must be 1 .. {groups}, got {top_groups}")
    scale = float(scale)
    if not 0 < abs(scale) < float("inf"):
        raise ValueError(f"scale must be finite and not 0, got {scale}")
    if bias is not None:
        check_gpu(bias, "bias")
        if bias.dtype != torch.float32:
            raise TypeError(f"bias must be float32, got {bias.dtype}")
        if bias.shape != (E,):
            raise ValueError(f"bias must be [{E}], got {tuple(bias.shape)}")
        bias = bias.detach().contiguous()
    args = (code, k, SCORING[scoring], groups, top_groups, int(bool(renormalize)), scale)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _RouteFn.apply(logits, bias, args)
    return _route(logits, bias, args)[:2]


# ------------------------------------------------------------------------------------------------ plan
class ExpertPlan:
    """The slots s = t k + j of experts [T, k] sorted by expert: those of expert e are order[offsets[e] : offsets[e + 1]],
    in ascending order.  Slots with an expert outside [0, n_experts) are in no list (order ends before them)."""

    def __init__(self, experts, n_experts, offsets, order):
        self.experts, self.n_experts, self.offsets, self.order = experts, n_experts, offsets, order

    @property
    def counts(self):
        """Slots of each expert, int32 [n_experts] (its load, for a balance bias)."""
        return self.offsets[1:] - self.offsets[:-1]


def plan_experts(experts, n_experts):
    """The ExpertPlan of experts [T, k] (int32 or int64; -1 for none): a stable counting sort on the GPU."""
    if not isinstance(experts, torch.Tensor) or not experts.is_cuda:
        raise TypeError("experts must be a GPU tensor")
    if experts.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"experts must be int32 or int64, got {experts.dtype}")
    if experts.device.index != torch.cuda.current_device():
        raise ValueError(f"experts is on {experts.device}, the current device is cuda:{torch.cuda.current_device()}")
    if experts.dim() != 2 or experts.shape[1] == 0:
        raise ValueError(f"experts must be [rows, k], got {tuple(experts.shape)}")
    E = int(n_experts)
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"n_experts must be 1 .. {MAX_EXPERTS}, got {n_experts}")
    S = experts.numel()
    if S > INT32_MAX:
        raise ValueError(f"more than 2^31 - 1 slots ({S})")
    if experts.dtype == torch.int64:       # values outside int32 must not wrap into the range of the experts
        experts = experts.clamp(-1, E).to(torch.int32)
    experts = experts.contiguous()
    n = ctypes.c_long(0)
    K.mm_expert_plan_scratch(S, E, ctypes.byref(n))
    buf = torch.empty(S + E + 1 + n.value, dtype=torch.int32, device=experts.device)
    offsets, order, scratch = buf[:E + 1], buf[E + 1:E + 1 + S], buf[E + 1 + S:]
    K.mm_expert_plan(experts, S, E, offsets, order, scratch if n.value else None, stream())
    return ExpertPlan(experts, E, offsets, order)


# ------------------------------------------------------------------------------------------------ products
def _strided(t):
    """(t with a contiguous last axis, distances of rows and components)."""
    if t.shape[2] > 1 and t.stride(2) != 1:
        t = t.contiguous()
    return t, t.stride(0), t.stride(1)


def _products(x, weight, gates, plan, code):
    T, M, D = x.shape
    E, _, F = weight.shape
    k = plan.experts.shape[1]
    y = torch.empty(T, M, F, dtype=x.dtype, device=x.device)
    rows = torch.empty(T * k, M, F, dtype=torch.float32, device=x.device)
    x, st, sm = _strided(x)
    K.mm_expert_rows(x, st, sm, code, T * k, k, M, D, F, weight, 0, E, plan.offsets, plan.order, rows, stream())
    K.mm_expert_combine(rows, gates, plan.experts, code, T, k, M, F, E, y, stream())
    return y


class _ExpertLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, gates, plan, code):
        weight = weight.contiguous()
        gates = gates.contiguous() if gates is not None else None
        ctx.save_for_backward(x, weight, gates)
        ctx.plan, ctx.code = plan, code
        return _products(x, weight, gates, plan, code)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, gates = ctx.saved_tensors
        plan, code = ctx.plan, ctx.code
        nx, nw, ng = ctx.needs_input_grad[:3]
        T, M, D = x.shape
        E, _, F = weight.shape
        k = plan.experts.shape[1]
        x, xt, xm = _strided(x)
        dy, yt, ym = _strided(dy)
        dx = torch.empty(T, M, D, dtype=x.dtype, device=x.device) if nx else None
        dg = torch.empty(T, k, dtype=torch.float32, device=x.device) if ng else None
        dw = torch.empty_like(weight) if nw else None
        if nx or ng:
            rows = torch.empty(T * k, M, D, dtype=torch.float32, device=x.device)
            K.mm_expert_rows(dy, yt, ym, code, T * k, k, M, F, D, weight, 1, E, plan.offsets, plan.order, rows,
                             stream())
            K.mm_expert_combine_bwd(rows, gates, plan.experts, x, xt, xm, code, T, k, M, D, E, dx, dg, stream())
        if nw:
            n = ctypes.c_size_t(0)
            K.mm_expert_wgrad_workspace(T * k, M, D, F, E, ctypes.byref(n))
            ws = torch.empty(n.value // 4, dtype=torch.float32, device=x.device) if n.value else None
            K.mm_expert_wgrad(x, xt, xm, dy, yt, ym, code, T * k, k, M, D, F, E, gates, plan.offsets, plan.order, dw,
                              ws, stream())
        return dx, dw, dg, None, None


def expert_linear(x, weight, plan, gates=None):
    """y[t, ...] = sum_j gates[t, j] x[t, ...] @ weight[plan.experts[t, j]]; slots without an expert add nothing.

    x [T, D], or [T, M, D]: M components of a row that share its experts (the 2 l + 1 components of an irrep; a slice of
    ir_mul features is read in place).  weight [E, D, F], of x's type; gates float32 [T, k] (None: ones).  Returns
    [T, (M,) F] of x's type.  Differentiable in x, weight and gates."""
    code = check_gpu(x, "x")
    if check_gpu(weight, "weight") != code:
        raise TypeError(f"weight must be {x.dtype} (as x), got {weight.dtype}")
    if not isinstance(plan, ExpertPlan):
        raise TypeError("plan must be an ExpertPlan (plan_experts)")
    if x.dim() not in (2, 3) or weight.dim() != 3:
        raise ValueError(f"x must be [rows, D] or [rows, components, D] and weight [experts, D, F], got "
                         f"{tuple(x.shape)} and {tuple(weight.shape)}")
    T, k = plan.experts.shape
    if x.shape[0] != T:
        raise ValueError(f"x has {x.shape[0]} rows, the plan {T}")
    if weight.shape[0] != plan.n_experts or weight.shape[1] != x.shape[-1] or 0 in weight.shape:
        raise ValueError(f"weight must be [{plan.n_experts}, {x.shape[-1]}, F], got {tuple(weight.shape)}")
    if x.dim() == 3 and x.shape[1] == 0:
        raise ValueError("x has no components")
    if gates is not None:
        check_gpu(gates, "gates")
        if gates.dtype != torch.float32:
            raise TypeError(f"gates must be float32, got {gates.dtype}")
        if gates.shape != (T, k):
            raise ValueError(f"gates must be {(T, k)}, got {tuple(gates.shape)}")
    if x.device != weight.device or x.device != plan.experts.device:
        raise ValueError("x, weight and the plan must be on one device")
    flat = x.dim() == 2
    if flat:
        x = x[:, None, :]
    if T * k * x.shape[1] > INT32_MAX - 128:
        raise ValueError(f"{T * k * x.shape[1]} rows: 2^31 or more are not supported")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, gates)):
        y = _ExpertLinearFn.apply(x, weight, gates, plan, code)
    else:
        y = _products(x, weight.contiguous(), gates.contiguous() if gates is not None else None, plan, code)
    return y[:, 0] if flat else y
