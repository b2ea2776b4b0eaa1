"""Linear layers at inference as products of 8-bit integers, with a scale for each row and each output channel.

A row x with largest magnitude a is held as whole numbers ``q = round(127 x / a)``, ties to even, times ``a / 127``.  A layer's weight is held so
once, row by row (``quantize_rows``); ``linear_int8`` takes the rows of its input the same way, call by call, sums the products of whole numbers
exactly and scales the sums.  Weights take half the bytes of 16-bit ones; activations cross memory in their own type.

CUDA tensors of type float32, bfloat16 and float16.  There are no gradients: calls that would need them are refused, as are calls under compilation,
tracing and torch.func transforms.
"""
from typing import NamedTuple, Optional

import torch
import torch.nn as nn

from . import _lib, fused
from .checkpoint8 import activation_code, require_ordinary


class _CodesAndScales(NamedTuple):
    codes: torch.Tensor
    scales: torch.Tensor


class QuantizedRows(_CodesAndScales):
    """Rows in 8-bit integers: ``codes`` int8, rows filled up with zeros to a multiple of sixteen, and ``scales`` fp32, what a step of each row's
    codes stands for.  A tuple of these two.  ``channels`` is how many of a row's codes are values, or None where it is not known: zeros behind them and
    codes of zero look alike, and a layer checks its input's channels by it."""
    channels: Optional[int] = None

    def __new__(cls, codes, scales, channels=None):
        self = super().__new__(cls, codes, scales)
        self.channels = channels
        return self


def quantize_rows(x):
    """``x`` [..., C] in 8-bit integers, without its history: codes [..., C'] (C' the next multiple of sixteen) and scales [...].  A row with an
    infinity or NaN has codes of zero and a scale that is NaN."""
    require_ordinary("quantize_rows", x)
    return QuantizedRows(*_lib.host(x.get_device()).int8_rows(x), x.shape[-1])


def linear_int8(x, weight, bias=None, activation=None):
    """``act(F.linear(x, W, bias))`` for ``x`` [..., C], W the rows that ``weight``, the ``quantize_rows`` of a [D, C] matrix, holds, and x's rows held the
    same way; ``activation``: None, "gelu" (exact) or "silu".  The result has x's type and is rounded once.  A row or output channel that holds an
    infinity or NaN is NaN.  Under autocast x and bias are converted as for ``F.linear``.  C has to be ``weight.channels``; where that is None (codes
    and scales that were put together by hand) only its next multiple of sixteen is compared."""
    code = -1 if activation is None else activation_code(activation)
    require_ordinary("linear_int8", x, weight.codes, weight.scales, bias)
    channels = getattr(weight, "channels", None)
    if channels is not None and x.shape[-1:] != (channels,):
        raise RuntimeError("x must have the %d channels that the weight's rows were made of, and has the shape %s" % (channels, tuple(x.shape)))
    dtype = fused._autocast(x)
    return _lib.host(x.get_device()).int8_linear(x if dtype is None else x.to(dtype), weight.codes, weight.scales, bias, code)


class LinearInt8(nn.Module):
    """A linear layer for inference whose weight is held in 8-bit integers; ``of`` makes one of an ``nn.Linear``."""

    def __init__(self, weight: QuantizedRows, in_features: int, bias: Optional[torch.Tensor] = None):
        super().__init__()
        if weight.codes.dim() != 2 or weight.codes.shape[1] != -(-in_features // 16) * 16 or getattr(weight, "channels", None) not in (None, in_features):
            raise ValueError("the weight's rows must be those of a matrix of %d columns" % in_features)
        self.in_features, self.out_features = in_features, weight.codes.shape[0]
        self.register_buffer("codes", weight.codes)
        self.register_buffer("scales", weight.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().clone())

    @classmethod
    def of(cls, linear):
        return cls(quantize_rows(linear.weight), linear.in_features, linear.bias)

    def _apply(self, fn, recurse=True):
        # (the scales stay fp32 when a network goes to another type)
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:
            self.scales = scales.to(self.scales.device)
        return self

    def extra_repr(self):
        return "%d, %d, bias=%r" % (self.in_features, self.out_features, self.bias is not None)

    def forward(self, x, activation=None):
        return linear_int8(x, QuantizedRows(self.codes, self.scales, self.in_features), self.bias, activation)


def quantize_network(network):
    """Puts a ``LinearInt8`` in the place of every wide layer of a network of ``convnext1d``: the pointwise layers of its plain blocks and its
    classifier.  (The stem, the operators, the norms and gated blocks stay as they are.)  The network is then for inference alone; returned.
    Where one of these layers is a subclass of its own, or has hooks, which would be lost, the call is refused and changes nothing.

    A network of fp32 becomes faster, one of 16-bit type slower, since its own blocks keep what lies between the two layers on the chip: the
    ConvNeXt-T-1D takes 16800 images a second in fp32 at a batch of 128 where it took 8300, and 775 where 483 by themselves; in bfloat16 28200 where 38200, and
    1010 where 1460.  What a 16-bit network gains is the memory of its weights."""
    from .convnext1d import Block, ConvNeXt1D

    found = []
    for module in network.modules():
        names = ("pwconv1", "pwconv2") if isinstance(module, Block) else ("head",) if isinstance(module, ConvNeXt1D) else ()
        for name in names:
            layer = module._modules.get(name)
            if isinstance(layer, nn.Linear):
                if not fused.plain(layer, nn.Linear, fused.Linear):
                    raise ValueError("%s of a %s is more than a linear layer, or has hooks" % (name, type(module).__name__))
                found.append((module, name, layer))
    for module, name, layer in [(m, n, LinearInt8.of(l)) for m, n, l in found]:
        setattr(module, name, layer)
    return network
