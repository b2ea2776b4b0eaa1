"""Softmax cross entropy of a linear classifier, without keeping its logits: what a network's head and its loss are in a training step.

The forward pass leaves a row's log-sum-exp and nothing of its logits; the backward pass computes them again, in pieces of the classes, and
turns them into the gradients of input, weight and bias.
"""
import torch.nn.functional as F

from . import _lib, fused
from .dwoconv1d import ordinary


def linear_cross_entropy(x, weight, bias, target, *, reduction="mean", ignore_index=-100, label_smoothing=0.0):
    """``F.cross_entropy(F.linear(x, weight, bias), target, ...)`` for ``x`` [..., C], ``weight`` [V, C], ``bias`` [V] or None and int64
    ``target`` [...], as fp32: the mean over the rows whose target is not ``ignore_index`` (NaN where there are none), or with reduction
    "none" a loss for every row, 0 where it is ignored.  A target that is no class gives NaN, in the loss and in the gradients.

    CUDA tensors of type float32, bfloat16 and float16; parameters may have another of these types and get gradients of their own.  Under
    autocast x and parameters are converted as for ``F.linear``.  Calls under compilation, tracing or torch.func transforms compose the
    same values from PyTorch ops; gradients of gradients are refused."""
    if reduction not in ("mean", "none"):
        raise ValueError("reduction must be 'mean' or 'none'")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("label_smoothing must be between 0 and 1")
    if not ordinary(x, weight, bias, target):
        logits = F.linear(x, weight, bias).float()
        loss = F.cross_entropy(logits.flatten(0, -2), target.flatten(), ignore_index=ignore_index, reduction=reduction,
                               label_smoothing=label_smoothing)
        return loss if reduction == "mean" else loss.unflatten(0, target.shape)
    dtype = fused._autocast(x)
    return _lib.host(x.get_device()).head(x if dtype is None else x.to(dtype), weight, bias, target, reduction == "mean",
                                          int(ignore_index), float(label_smoothing))
