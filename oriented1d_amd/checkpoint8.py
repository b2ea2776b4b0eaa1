"""8-bit checkpoints: what a backward pass needs of an activation, held in one byte a value.

Groups of 32 neighbours along the last dimension share a power of two ``s = 2 ** (floor(log2(largest magnitude)) - 6)``, at least
``2 ** -126``, and hold ``q = round(x / s)``, ties to even, in [-127, 127]; what is held is ``q * s``, at most half a step ``s / 2`` away
(a whole one next to the largest magnitude), which is exact in every type.  A group with an infinity or NaN comes back as NaN.

``linear8`` and ``act8`` are ``F.linear`` and an activation whose results are exact and whose backward passes read a checkpoint in place
of the input: a weight gradient, and an activation's slope, are computed at the values held.  Blocks of ``convnext1d`` run on them with
``checkpoint8=True``, as ``feedforward.gated_mlp`` does.

CUDA tensors of type float32, bfloat16 and float16; parameters may have another of these types and get gradients of their own.
Under autocast inputs and parameters are converted as for ``F.linear``.  Gradients of gradients are refused.
"""
from typing import NamedTuple

import torch

from . import _lib, fused
from .dwoconv1d import ordinary

ACTIVATIONS = {"gelu": 0, "silu": 1}


class Packed8(NamedTuple):
    """A tensor in 8 bits: ``codes`` int8 of its shape, ``exponents`` uint8 (biased by 127; 0: zeros, 255: not finite) with one for every
    32 values of a row, and its type."""
    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype


def activation_code(name):
    if name not in ACTIVATIONS:
        raise ValueError("activation must be one of %s" % ", ".join(repr(a) for a in ACTIVATIONS))
    return ACTIVATIONS[name]


def require_ordinary(what, *tensors):
    if not ordinary(*tensors):
        raise RuntimeError("%s takes ordinary tensors outside of compilation, tracing and torch.func transforms" % what)


def pack8(x):
    """``x`` [..., C] in 8 bits, without its history."""
    require_ordinary("pack8", x)
    return Packed8(*_lib.host(x.get_device()).pack8(x), x.dtype)


def unpack8(packed):
    """The values that a checkpoint holds, in the type of what was packed."""
    return _lib.host(packed.codes.get_device()).unpack8(packed.codes, packed.exponents, packed.dtype)


def linear8(x, weight, bias=None):
    """``F.linear(x, weight, bias)`` for ``weight`` [D, C] that keeps ``x`` in 8 bits: the gradients of x and of the bias are exact, the
    weight's is ``dy.T @ unpack8(pack8(x))``."""
    require_ordinary("linear8", x, weight, bias)
    dtype = fused._autocast(x)
    return _lib.host(x.get_device()).linear8(x if dtype is None else x.to(dtype), weight, bias)


def act8(x, activation="gelu"):
    """``F.gelu(x)`` (exact) or ``F.silu(x)`` that keeps ``x`` in 8 bits: its gradient takes the slope at ``unpack8(pack8(x))``."""
    code = activation_code(activation)
    require_ordinary("act8", x)
    return _lib.host(x.get_device()).act8(x, code)
