"""Losses of a linear classifier, without keeping its logits: what a network's head and its loss are in a training step.

``linear_cross_entropy`` is softmax cross entropy against classes, ``linear_distillation`` that against a teacher's top logits, which
``top_logits`` takes of a row.  The forward pass leaves a row's log-sum-exp, and the few logits that the loss reads; the backward pass computes
them again, in pieces of the classes, and turns them into the gradients of input, weight and bias.
"""
import operator
from typing import NamedTuple

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


class TopLogits(NamedTuple):
    """The k largest logits of each row and their classes (int64), largest first."""
    values: torch.Tensor
    classes: torch.Tensor


def top_logits(logits, k):
    """The ``k`` largest of ``logits`` [..., V] and their classes as ``TopLogits``, [..., k] each, without their history: largest first, of equal
    ones the lowest class first.  NaN is above everything, and the zeros are equal.

    A CUDA tensor of type float32, bfloat16 or float16; V is at most 2^24, k at most 1024 and V.  Calls under compilation, tracing or torch.func
    transforms take the same from a stable sort."""
    k = operator.index(k)
    if logits.dim() < 1 or not 1 <= k <= min(logits.shape[-1], 1024):
        raise ValueError("k must be from 1 to 1024 and no more than there are classes")
    if not ordinary(logits):
        values, classes = torch.sort(logits.detach(), dim=-1, descending=True, stable=True)
        return TopLogits(values[..., :k], classes[..., :k])
    return TopLogits(*_lib.host(logits.get_device()).top(logits, k))


def _temperature(value):
    value = float(value)
    if not 1e-4 <= value <= 1e4:
        raise ValueError("temperature must be from 1e-4 to 1e4")
    return value


def _reduction(value):
    if value not in ("mean", "none"):
        raise ValueError("reduction must be 'mean' or 'none'")


def distillation_of(logits, teacher_logits, teacher_classes, temperature=1.0, reduction="mean"):
    """``linear_distillation`` of a classifier's own ``logits`` [..., V], from PyTorch ops: for any leading dimensions and none."""
    if teacher_logits.shape != teacher_classes.shape or teacher_logits.shape[:-1] != logits.shape[:-1] or teacher_classes.dtype != torch.int64:
        raise RuntimeError("teacher_classes must be int64, one class for every teacher logit, and both have entries for every row of x")
    _reduction(reduction)
    temperature = _temperature(temperature)
    if torch.is_grad_enabled() and teacher_logits.requires_grad:
        raise RuntimeError("the teacher's logits get no gradient: detach them")
    t = teacher_logits.float()
    classes = teacher_classes
    there = (classes != -1) & (t != float("-inf"))
    bad = there & ((classes < 0) | (classes >= logits.shape[-1]) | ~(t < float("inf")))
    there = there & ~bad
    bad, some = bad.any(-1), there.any(-1)
    counts = bad | some
    nothing = torch.where(bad, float("nan"), 0.0).to(torch.float32)
    # (rows that do not count may hold anything)
    own = torch.where(counts.unsqueeze(-1), logits.float(), 0.0) + nothing.unsqueeze(-1)
    logs = F.log_softmax(own / temperature, -1).gather(-1, torch.where(there, classes, 0))
    t = torch.where(there, t / temperature, float("-inf"))
    log_p = F.log_softmax(torch.where(some.unsqueeze(-1), t, 0.0), -1)
    p = torch.where(there, torch.exp(log_p), 0.0)
    loss = temperature * temperature * torch.where(p > 0, p * (log_p - logs), 0.0).sum(-1) + nothing
    loss = torch.where(counts, loss, 0.0)
    if reduction == "none":
        return loss
    number = counts.sum()
    return torch.where(number > 0, loss.sum() / number.clamp(min=1), float("nan"))


def linear_distillation(x, weight, bias, teacher_logits, teacher_classes, *, temperature=1.0, reduction="mean"):
    """The loss of a linear classifier, ``l = F.linear(x, weight, bias)`` for ``x`` [..., C], ``weight`` [V, C] and ``bias`` [V] or None, against the
    largest logits of a teacher, ``teacher_logits`` [..., k] and their int64 ``teacher_classes`` [..., k] (``top_logits``):
    ``temperature ** 2 * sum_j p_j (log p_j - log q_j)`` with ``p`` the softmax over the row's entries of ``teacher_logits / temperature`` and ``q_j``
    that of ``l / temperature`` over all classes at ``teacher_classes[j]``.  As fp32: the mean over the rows with entries (NaN where there are none),
    or with reduction "none" a loss for every row.

    An entry of class -1, or whose logit is -infinity, is absent, whatever else it holds; a row without entries has no loss (0), no gradient and
    does not count.  Another class that is none, or a teacher's logit that is NaN or infinite, gives NaN, in the row's loss and gradient.  Entries of the
    same class count each for itself.

    CUDA tensors of type float32, bfloat16 and float16; the teacher's logits and the parameters may have another of these types, the parameters get
    gradients of their own; teacher's logits that require one are refused.  k is at most 1024, the temperature from 1e-4 to 1e4.  Under autocast x
    and parameters are converted as for ``F.linear``.  Calls under compilation, tracing or torch.func transforms compose the same values from
    PyTorch ops; gradients of gradients are refused.  The loss and what goes into 16-bit products are computed and held as for ``linear_cross_entropy``."""
    _reduction(reduction)
    temperature = _temperature(temperature)
    if not ordinary(x, weight, bias, teacher_logits, teacher_classes):
        return distillation_of(fused.linear_as(x, weight, bias), teacher_logits, teacher_classes, temperature, reduction)
    dtype = fused._autocast(x)
    return _lib.host(x.get_device()).distill(x if dtype is None else x.to(dtype), weight, bias, teacher_logits, teacher_classes, temperature,
                                             reduction == "mean")
