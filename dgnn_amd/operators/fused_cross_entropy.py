"""Autograd operator of the cross entropy of a linear layer (new API surface; the reference's examples
form all logits and call nn.CrossEntropyLoss, script/train/train_gatconv.py)."""
import torch

from .._lib import DgnnError
from ..native import fused_cross_entropy
from ._autograd import differentiated

_REDUCTION = {"none": 0, "mean": 1, "sum": 2}


def LinearCrossEntropyFuse(feat, weight, label, ignore_index=-100, reduction="mean"):
    """cross_entropy(feat @ weight.T, label) without the [rows, classes] logits; float32.

    feat [rows, dim] and weight [classes, dim] of one type (float32, bfloat16 or float16), label int32 or
    int64.  Rows labelled ignore_index, or with a label outside [0, classes), have no loss and no
    gradient, whatever they hold.  reduction: "mean" over the labelled rows (0 if there are
    none), "sum", or "none" (one loss a row, 0 without a label).

    The gradient of the logits, rounded to feat's type, is rebuilt a piece of the classes at a
    time; both gradients are summed in float32 in a fixed order."""
    if reduction not in _REDUCTION:
        raise DgnnError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if not differentiated(feat, weight):
        return fused_cross_entropy.linear_ce_forward(feat.contiguous(), weight.contiguous(), label.contiguous(),
                                                     ignore_index, _REDUCTION[reduction])[0]
    return LinearCrossEntropyFunction.apply(feat, weight, label, ignore_index, _REDUCTION[reduction])


class LinearCrossEntropyFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, feat, weight, label, ignore_index, reduction):
        feat, weight, label = feat.contiguous(), weight.contiguous(), label.contiguous()
        loss, lse = fused_cross_entropy.linear_ce_forward(feat, weight, label, ignore_index, reduction)
        ctx.save_for_backward(feat, weight, label, lse)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_loss):
        feat, weight, label, lse = ctx.saved_tensors
        grad_feat, grad_weight = fused_cross_entropy.linear_ce_backward(
            feat, weight, label, ctx.ignore_index, ctx.reduction, lse, grad_loss.contiguous(),
            want_feat=ctx.needs_input_grad[0], want_weight=ctx.needs_input_grad[1])
        return grad_feat, grad_weight, None, None, None
