"""Softmax cross entropy of a linear classifier, without keeping its logits: what a network's head and its loss are in a training step.

The forward pass leaves a row's log-sum-exp and nothing of its logits; the backward pass computes them again, in pieces of the classes, and
turns them into the gradients of input, weight and bias.
"""
import torch
import torch.nn.functional as F

from . import _lib, fused
from .dwoconv1d import ordinary


def _composed(x, weight, bias, target, reduction, ignore_index, label_smoothing):
    """The same values from PyTorch ops, for any leading dimensions and none."""
    if target.shape != x.shape[:-1] or target.dtype != torch.int64:
        raise RuntimeError("target must be int64, one class for every row of x")
    logits = fused.linear_as(x, weight, bias).float()
    counts = target != ignore_index
    is_class = counts & (target >= 0) & (target < logits.shape[-1])
    # rows that are ignored may hold anything, and those whose target is no class are NaN, as are their gradients
    nothing = torch.where(counts & ~is_class, float("nan"), 0.0).to(logits.dtype)
    logits = torch.where(counts.unsqueeze(-1), logits, 0.0) + nothing.unsqueeze(-1)
    logs = F.log_softmax(logits, -1)
    loss = -logs.gather(-1, torch.where(is_class, target, 0).unsqueeze(-1)).squeeze(-1)
    if label_smoothing > 0:
        loss = (1 - label_smoothing) * loss - label_smoothing * logs.mean(-1)
    loss = torch.where(counts, loss, 0.0)
    if reduction == "none":
        return loss
    number = counts.sum()
    return torch.where(number > 0, loss.sum() / number.clamp(min=1), float("nan"))


def linear_cross_entropy(x, weight, bias, target, *, reduction="mean", ignore_index=-100, label_smoothing=0.0):
    """``F.cross_entropy(F.linear(x, weight, bias), target, ...)`` for ``x`` [..., C], ``weight`` [V, C], ``bias`` [V] or None and int64
    ``target`` [...], as fp32: the mean over the rows whose target is not ``ignore_index`` (NaN where there are none), or with reduction
    "none" a loss for every row, 0 where it is ignored.  A target that is no class gives NaN, in the loss and in the gradients.

    CUDA tensors of type float32, bfloat16 and float16; parameters may have another of these types and get gradients of their own.  Under
    autocast x and parameters are converted as for ``F.linear``.  Calls under compilation, tracing or torch.func transforms compose the
    same values from PyTorch ops; gradients of gradients are refused.

    Losses are computed in fp32.  In 16 bits the logits' gradients are rounded to the type of x for the products that read them; where rows *
    V * C is at most 2^28 they are held in two such values, so that a row's gradient may have other last bits in a small batch than in a
    large one, nearer to the formula."""
    if reduction not in ("mean", "none"):
        raise ValueError("reduction must be 'mean' or 'none'")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("label_smoothing must be between 0 and 1")
    if not ordinary(x, weight, bias, target):
        return _composed(x, weight, bias, target, reduction, ignore_index, label_smoothing)
    dtype = fused._autocast(x)
    return _lib.host(x.get_device()).head(x if dtype is None else x.to(dtype), weight, bias, target, reduction == "mean",
                                          int(ignore_index), float(label_smoothing))
