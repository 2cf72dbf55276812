"""Mixtures of expert weight blocks: routing of rows (atoms, tokens) to experts and the gated products with their
blocks.

The species-block linears of the model multiply every node row by the block of its species.  Here a row gets k of E
blocks with gates that are learned:

    gates, experts = route(logits, k)                        # [T, E] -> float32 [T, k], int32 [T, k]
    plan = plan_experts(experts, E)                          # the (row, choice) slots sorted by expert
    y = expert_linear(x, weight, plan, gates)                # y[t] = sum_j gates[t, j] x[t] @ weight[experts[t, j]]

All three run hand-written kernels on torch's current stream without reading anything back, so that a chain of them can
be captured into a HIP graph; they need the GPU.  Results are the same bits in every run (no float atomics).  x and
weight (and the logits on their own) are float32, bfloat16 or float16; gates are float32, and sums are float32 whatever
the type.  Gradients can be taken once (no second derivative).  The reference has no counterpart; its nearest operation
is SpeciesSkip (fast_layers.py:41-105).
"""
from ._ops import ops


def route(logits, k, scoring="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0):
    """(gates float32 [T, k], experts int32 [T, k]): the k experts of largest key = logit + bias of every row, in
    descending order of the key, ties to the lowest index.

    logits [T, E], E up to 1024, k up to 32: -inf closes an expert to a row; a slot without an open expert gets expert
        -1 and gate 0 (a row with nothing open: all slots).  A NaN logit is chosen first and makes the row's gates NaN
        (plain sigmoids: its own gate).
    scoring: "softmax" (over the row's E logits) or "sigmoid" (of each).
    bias float32 [E]: moves the choice (balance of the experts' load) and not the gates; no gradient.  It is added to
        the logits.  That is a rule of its own: a router whose bias was trained on the scores (score + bias, groups by
        the sum of their two best) chooses other experts here.
    groups, top_groups: the E experts in `groups` equal runs (64 at most), of which only the top_groups with the largest
        keys are open (None: all).
    renormalize: gates = scale * score / sum of the chosen scores, finite also where all scores underflow; else
        gates = scale * score.
    Differentiable in logits."""
    return ops().route(logits, k, scoring, bias, groups, top_groups, renormalize, scale)


def plan_experts(experts, n_experts):
    """The plan of experts [T, k] (int32 or int64; -1 for none), n_experts up to 1024, for expert_linear: a stable
    counting sort of the slots s = t k + j by expert.  A contiguous int32 tensor is not copied: it is read again by
    every product, and a plan whose experts were changed in place raises RuntimeError (under torch.inference_mode, where
    tensors carry no version, it cannot: leave them alone there).  Its fields (tensors are not to be changed: the
    kernels trust them):

    experts int32 [T, k], n_experts
    order int32 [T k], offsets int32 [n_experts + 1]: the slots of expert e are order[offsets[e] : offsets[e + 1]], in
        ascending order; slots with an expert outside [0, n_experts) come after them, from offsets[n_experts] on.
        Sorted when first needed on a stream (few rows need no order, rows of two choices may be sorted by pair of
        experts instead), except under graph capture, where it is recorded at once.  Outside that capture the plan's
        fields and products sort its experts as they are by then, after the last replay, at every use.
    counts int32 [n_experts]: slots of each expert (its load, for a balance bias)"""
    return ops().plan_experts(experts, n_experts)


def expert_linear(x, weight, plan, gates=None):
    """y[t, ...] = sum_j gates[t, j] x[t, ...] @ weight[plan.experts[t, j]]; slots without an expert add nothing.

    x [T, D], or [T, M, D]: M components of a row that share its experts (the 2 l + 1 components of an irrep; a slice of
    ir_mul features is read in place).  weight [E, D, F], of x's type; gates float32 [T, k] (None: ones).  Returns
    [T, (M,) F] of x's type.  Differentiable in x, weight and gates.  float32 products are taken from three bfloat16
    parts of each operand at float32 accuracy (as the model's linears do).  float32 operands that round to infinity in
    bfloat16 (from 3.396e38 on, infinity among them) give NaN in the results that they enter, for one row as for many;
    16-bit operands give infinity or NaN as their sums do.  In the gradient of weight the operand is gate times
    cotangent, of 16-bit types in two bfloat16 parts, and an infinite value gives infinity or NaN."""
    return ops().expert_linear(x, weight, gates, plan)
