"""The operators around wide layers at magnitudes where their formulas could leave a type's range, against the formulas in 64 bits.
Tolerances as in test_wide_gpu.py where nothing else is said."""
import pytest
import torch
import torch.nn.functional as F

from oriented1d_amd import checkpoint8, feedforward
from test_wide_gpu import DTYPES, IDS, gated64, held8, leaves64, make_gated, near

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------- SiLU of large numbers
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_silu_of_large_numbers(dtype):
    """Every value of a 16-bit type and steps of 1/32 in fp32, from -1.1e4 to 1.1e4: g / (1 + exp(-g)) and its slope are numbers everywhere.
    Off by a rounding, what fp32 exponentials and quotients lose (1e-6 relative, and the exponent's rounding is in there up to 88), and
    below -87 by the values themselves, which are under 2e-36 as are their slopes."""
    if dtype == torch.float32:
        x = torch.arange(-1.1e4, 1.1e4, 1 / 32, device="cuda", dtype=torch.float64).float()
    else:
        x = torch.arange(-(1 << 15), 1 << 15, device="cuda").to(torch.int16).view(dtype)
        x = x[x.float().abs() <= 1.1e4]
    r = torch.finfo(dtype).eps / 2
    # (in groups of one value each, which the 8-bit form holds to its step of 2^-7)
    for v in (x[: len(x) // 32 * 32].view(-1, 32), x[:, None], x[: len(x) // 31 * 31].view(-1, 31)):
        v = v.clone().requires_grad_()
        y = checkpoint8.act8(v, "silu")
        dx, = torch.autograd.grad(y, v, torch.ones_like(y))
        want = F.silu(v.detach().double())
        at = held8(v.detach()).requires_grad_()
        slope, = torch.autograd.grad(F.silu(at).sum(), at)
        tiny = 2.0 ** -25 if dtype == torch.float16 else 2e-36
        for got, ref, what in ((y, want, "value"), (dx, slope, "slope")):
            assert torch.isfinite(got).all(), "%s: %d not finite" % (what, int((~torch.isfinite(got)).sum()))
            # (a slope is a sum of terms of size 1 at the largest: 1e-6 of them beside the relative error)
            off = (got.double() - ref).abs() - (r + 2e-6) * ref.abs() - (1e-6 if what == "slope" else 0.0) - tiny
            assert float(off.max()) <= 0.0, "%s: %.3g beyond the limit" % (what, float(off.max()))


@pytest.mark.parametrize("held", [False, True], ids=["kept", "held8"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [3, 70, 300])
def test_gated_block_with_large_gates(rows, dtype, held):
    """Gates of -80 to -1e4 among ordinary ones: their hidden units and gradients are zeros, the others as in 64 bits."""
    args, dy = make_gated(rows, 40, 96, 72, dtype)
    with torch.no_grad():
        # biases far from zero for a third of the gates: sums of the projection's spread of 1.5 around them
        far = -torch.logspace(1.9, 4, 32, device="cuda")
        args[2][0:96:3] = far.to(dtype)
    y = feedforward.gated_mlp(*args, activation="silu", checkpoint8=held)
    got = torch.autograd.grad(y, args, dy)
    ref = leaves64(*args)
    near(y, gated64(*ref, "silu"), "y")
    if held:
        ref[0] = held8(args[0].detach()).requires_grad_()
    want = torch.autograd.grad(gated64(*ref, "silu"), ref, dy.double())
    for g, w, name in zip(got, want, ["dx", "dw_in", "db_in", "dw_out", "db_out"]):
        near(g, w, name)
