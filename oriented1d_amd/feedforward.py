"""The gated feed-forward block: ``(act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo``, in place of a block's two pointwise layers and
GELU where a network gates its hidden units.

Both first projections are one product, whose sums become hidden units without going through memory; the backward pass makes their
gradients in the product that they come from.  Between the passes the two halves of the hidden tensor are kept in fp32, or with
``checkpoint8`` nothing but the input in 8 bits (``checkpoint8.pack8``): then the backward pass computes them again, and every gradient is
taken at the values held (``x``'s own as well).
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib, fused
from .checkpoint8 import activation_code, require_ordinary
from .dwoconv1d import ordinary

_FUNCTIONS = {"gelu": F.gelu, "silu": F.silu}


def gated_mlp(x, w_in, b_in, w_out, b_out, activation="gelu", checkpoint8=False):
    """``x`` [..., C], ``w_in`` [2 H, C] (the gates' H rows first), ``b_in`` [2 H] or None, ``w_out`` [D, H], ``b_out`` [D] or None ->
    [..., D].  ``activation``: "gelu" (exact) or "silu".

    CUDA tensors of type float32, bfloat16 and float16; parameters may have another of these types and get gradients of their own.  Under
    autocast x and parameters are converted as for ``F.linear``.  Calls under compilation, tracing or torch.func transforms compose
    the same values from PyTorch ops, which ``checkpoint8`` cannot; gradients of gradients are refused.

    In 16 bits what one product makes for another (hidden units and their gradients) is rounded to the type of x; where rows * H * (2 C + D)
    is at most 2^28 it is held in two such values, and in a forward pass of up to four rows the hidden units are fp32.  So the same row may come
    out with other last bits in a small batch than in a large one, nearer to the formula."""
    code = activation_code(activation)
    if not ordinary(x, w_in, b_in, w_out, b_out):
        if checkpoint8:
            require_ordinary("gated_mlp(checkpoint8=True)", x, w_in, b_in, w_out, b_out)
        gate, up = fused.linear_as(x, w_in, b_in).chunk(2, dim=-1)
        return fused.linear_as(_FUNCTIONS[activation](gate) * up, w_out, b_out)
    dtype = fused._autocast(x)
    return _lib.host(x.get_device()).gated(x if dtype is None else x.to(dtype), w_in, b_in, w_out, b_out, code, bool(checkpoint8))


class GatedMLP(nn.Module):
    """``gated_mlp`` with its parameters: ``dim`` channels in and out, ``hidden`` gated units."""

    def __init__(self, dim, hidden, activation="gelu", bias=True, checkpoint8=False):
        super().__init__()
        activation_code(activation)
        if dim < 1 or hidden < 1:
            raise ValueError("dim and hidden must be at least 1")
        self.activation, self.checkpoint8 = activation, bool(checkpoint8)
        self.w_in = nn.Parameter(torch.empty(2 * hidden, dim))
        self.w_out = nn.Parameter(torch.empty(dim, hidden))
        self.b_in = nn.Parameter(torch.zeros(2 * hidden)) if bias else None
        self.b_out = nn.Parameter(torch.zeros(dim)) if bias else None
        # as every other layer of the networks here
        nn.init.trunc_normal_(self.w_in, std=0.02)
        nn.init.trunc_normal_(self.w_out, std=0.02)

    def extra_repr(self):
        return "%d, %d, activation=%r, bias=%r, checkpoint8=%r" % (self.w_in.shape[1], self.w_out.shape[1], self.activation,
                                                                   self.b_in is not None, self.checkpoint8)

    def forward(self, x):
        return gated_mlp(x, self.w_in, self.b_in, self.w_out, self.b_out, self.activation, self.checkpoint8)


fused.CONSUMERS.append(GatedMLP)
