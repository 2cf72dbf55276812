"""Cross entropy of a linear head over many classes, without keeping its logits.

    logits = x @ weight^T,   loss[t] = log sum_v exp(logits[t, v]) - logits[t, targets[t]]

x [..., D] and weight [classes, D]: float32, bfloat16 or float16, both of one type; rows of x may be strided and are read
in place where the last axis is contiguous.  targets [...]: int32 or int64 classes; rows whose target is ignore_index are
taken out (loss 0, zero gradient, whatever stands in them); any other target outside [0, classes) makes the row's loss
and the gradients NaN.  The logits live in registers alone: forward keeps two numbers a row, backward takes them again in
pieces of the classes.  Losses and gradients of rows that are certain of their class keep their digits: they come from the
sum over the other classes, which is never added to 1.  float32 products are taken from three bfloat16 parts of each
operand at float32 accuracy (values from 3.396e38 on, infinity among them, give NaN, for one row as for many; 16-bit
infinities give what their sums do); logits, exponentials and all sums are float32, in a fixed order: the same bits in
every run.
Sizes from 2^31 - 2^16 on are refused, and so are rows times classes, or their sum times D, from about 2^36 (6.8e10)
on: the launches' tiles of 64 x 64.  Runs on torch's current stream without reading anything back, can be captured into
a HIP graph, and needs the GPU: there is no CPU path.  The reference has no counterpart.
"""
from ._ops import ops


def linear_cross_entropy(x, weight, targets, ignore_index=-100, reduction="mean"):
    """The cross entropy of x @ weight^T against targets (module docstring), float32: "mean" over the rows that are not
    ignored (0 if there are none), "sum", or "none" for one loss a row (the score of single tokens or atoms).
    Differentiable once in x and weight."""
    return ops().linear_cross_entropy(x, weight, targets, ignore_index, reduction)
