"""The operators around wide layers without a GPU: status codes of the C entry points before any GPU work, workspace sizes, and what the
Python entry points refuse."""
import ctypes

import pytest
import torch

from oriented1d_amd import _lib, checkpoint8, feedforward, losses
from oriented1d_amd.convnext1d import Block, ConvNeXt1D, gated_hidden

ONE = ctypes.c_void_p(256)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(264)
F32, BF16, F16 = 0, 1, 2


def lib():
    return _lib.load()


def test_workspace_sizes():
    L = lib()
    for dtype in (F32, BF16, F16):
        for rows, C, H, D in [(1, 1, 1, 1), (49, 96, 256, 96), (16384, 1024, 4096, 1024), (1 << 30, 8, 8, 8)]:
            for backward in (0, 1):
                for held in (0, 1):
                    assert L.dwo_gated_workspace_bytes(rows, C, H, D, backward, held, dtype) > 0
                assert L.dwo_layer8_workspace_bytes(rows, C, D, backward, dtype) > 0
        for rows, C, V in [(1, 1, 1), (64, 768, 1000), (8192, 1024, 65536), (1 << 30, 8, 8), (1, 8, 1 << 24)]:
            assert all(L.dwo_head_workspace_bytes(rows, C, V, b, dtype) > 0 for b in (0, 1))
    # a backward pass holds the logits' gradients in pieces of the classes, about 2^27 values each
    piece = L.dwo_head_workspace_bytes(8192, 1024, 1 << 18, 1, BF16)
    assert piece < 3 * (1 << 28) + 8192 * 1024 * 4 + (1 << 28)
    for bad in [(0, 8, 8, 8), (1, 0, 8, 8), (1, 8, 0, 8), (1, 8, 8, 0), ((1 << 30) + 1, 8, 8, 8), (1, 65537, 8, 8), (1, 8, 65537, 8)]:
        assert L.dwo_gated_workspace_bytes(*bad, 0, 0, BF16) == 0
    assert L.dwo_gated_workspace_bytes(1, 8, 8, 8, 0, 0, 3) == 0
    assert L.dwo_head_workspace_bytes(1, 8, (1 << 24) + 1, 0, BF16) == 0 and L.dwo_head_workspace_bytes(1, 8, 0, 0, BF16) == 0
    assert L.dwo_layer8_workspace_bytes(1, 8, 65537, 0, BF16) == 0


def test_status_codes():
    L = lib()

    def gated(x=ONE, w=ONE, y=ONE, keep=None, ws=ONE, need=1 << 40, rows=4, C=8, H=8, D=8, act=0, dtype=BF16):
        return L.dwo_gated_forward(x, w, None, ONE, None, y, keep, ws, need, rows, C, H, D, act, dtype, None)

    assert gated(x=None) == -1 and gated(y=None) == -1 and gated(ws=None) == -1
    assert gated(rows=0) == -2 and gated(C=0) == -2 and gated(act=2) == -2 and gated(act=-1) == -2 and gated(x=ODD) == -2
    assert gated(dtype=3) == -5 and gated(need=1) == -7

    def gated_back(x=ONE, codes=None, exps=None, keep=ONE, dx=ONE, dwi=ONE, dbi=ONE, need=1 << 40, grad=F32):
        return L.dwo_gated_backward(ONE, x, codes, exps, keep, ONE, None, ONE, dx, dwi, dbi, None, None, ONE, need, 4, 8, 8, 8, 0, BF16,
                                    grad, None)

    assert gated_back(x=None) == -1 and gated_back(keep=None) == -1
    assert gated_back(codes=ONE, exps=ONE) == -1  # a checkpoint goes without keep
    assert gated_back(codes=ONE, keep=None) == -1
    assert gated_back(dwi=None) == -2  # a bias gradient without its weight's
    assert gated_back(grad=4) == -5 and gated_back(need=1) == -7

    def head(x=ONE, targets=ONE, smoothing=0.0, need=1 << 40, V=10, dtype=BF16):
        return L.dwo_head_forward(x, ONE, None, targets, -100, smoothing, ONE, ONE, ONE, ONE, need, 4, 8, V, dtype, None)

    assert head(x=None) == -1 and head(targets=None) == -1
    assert head(V=0) == -2 and head(smoothing=1.5) == -2 and head(smoothing=float("nan")) == -2 and head(targets=ctypes.c_void_p(260)) == -2
    assert head(dtype=7) == -5 and head(need=1) == -7
    assert L.dwo_head_backward(ONE, ONE, ONE, None, ONE, -100, 0.0, ONE, None, ONE, None, ONE, ONE, 1 << 40, 4, 8, 10, BF16, F32, None) == -2
    assert L.dwo_head_backward(None, ONE, ONE, None, ONE, -100, 0.0, ONE, None, ONE, ONE, ONE, ONE, 1 << 40, 4, 8, 10, BF16, F32, None) == -1

    assert L.dwo_pack8(None, None, ONE, ONE, 4, 8, 0, BF16, None) == -1
    assert L.dwo_pack8(ONE, None, ONE, ONE, 0, 8, 0, BF16, None) == -2 and L.dwo_pack8(ONE, None, ONE, ONE, 4, 8, 2, BF16, None) == -2
    assert L.dwo_pack8(ONE, None, ONE, ONE, 4, 8, 0, 9, None) == -5
    assert L.dwo_unpack8(ONE, None, None, ONE, 4, 8, 0, BF16, None) == -1 and L.dwo_unpack8(ODD, ONE, None, ONE, 4, 8, 0, BF16, None) == -2
    assert L.dwo_layer8(ONE, ONE, None, ONE, ONE, None, ONE, 1 << 40, 4, 8, 8, BF16, None) == -1  # codes without exponents
    assert L.dwo_layer8(ONE, ONE, None, ONE, None, None, ONE, 1, 4, 8, 8, BF16, None) == -7
    assert L.dwo_layer8_backward(ONE, ONE, ONE, ONE, ONE, None, ONE, ONE, 1 << 40, 4, 8, 8, BF16, F32, None) == -2


def test_python_refusals():
    x, w, b, w_out = torch.randn(4, 8), torch.randn(16, 8), torch.randn(16), torch.randn(8, 8)
    target = torch.zeros(4, dtype=torch.long)
    for call in (lambda: feedforward.gated_mlp(x, w, b, torch.randn(8, 8), None), lambda: checkpoint8.linear8(x, w, b),
                 lambda: checkpoint8.act8(x), lambda: checkpoint8.pack8(x), lambda: losses.linear_cross_entropy(x, w, b, target)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="activation"):
        feedforward.gated_mlp(x, w, b, torch.randn(8, 8), None, activation="relu")
    with pytest.raises(ValueError, match="activation"):
        checkpoint8.act8(x, "tanh")
    with pytest.raises(ValueError, match="activation"):
        feedforward.GatedMLP(8, 16, activation="relu")
    with pytest.raises(ValueError, match="at least 1"):
        feedforward.GatedMLP(8, 0)
    with pytest.raises(ValueError, match="reduction"):
        losses.linear_cross_entropy(x, w, b, target, reduction="sum")
    for value in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="label_smoothing"):
            losses.linear_cross_entropy(x, w, b, target, label_smoothing=value)
    for call in (lambda: torch.func.vmap(lambda v: checkpoint8.linear8(v, w, b))(x[None]),
                 lambda: torch.func.vmap(lambda v: feedforward.gated_mlp(v, w, b, w_out, None, checkpoint8=True))(x[None])):
        with pytest.raises(RuntimeError, match="ordinary tensors"):
            call()


def test_transforms_compose_the_same_values():
    x, w, b, v = torch.randn(3, 4, 8), torch.randn(16, 8), torch.randn(16), torch.randn(5, 8)
    gate, up = torch.nn.functional.linear(x, w, b).chunk(2, -1)
    want = torch.nn.functional.linear(torch.nn.functional.silu(gate) * up, v)
    got = torch.func.vmap(lambda a: feedforward.gated_mlp(a, w, b, v, None, activation="silu"))(x)
    assert torch.allclose(got, want, atol=1e-5)
    target = torch.tensor([[0, 3, -100, 15]] * 3)
    want = torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w, b).flatten(0, 1), target.flatten(), reduction="none")
    got = torch.func.vmap(lambda a, t: losses.linear_cross_entropy(a, w, b, t, reduction="none"))(x, target)
    assert torch.allclose(got.flatten(), want, atol=1e-5)


def test_networks_with_gated_blocks():
    assert [gated_hidden(d) for d in (96, 128, 192, 768, 1)] == [256, 344, 512, 2048, 8]
    block = Block(96, (31,), False, mlp="gated")
    assert block.mlp.w_in.shape == (512, 96) and block.mlp.w_out.shape == (96, 256)
    names = dict(block.named_parameters())
    assert "mlp.w_in" in names and not any(n.startswith("pwconv") for n in names)
    plain = dict(Block(96, (31,), False).named_parameters())
    assert not any(n.startswith("mlp") for n in plain) and "pwconv1.weight" in plain
    # as many weights as the two pointwise layers
    assert abs(sum(names[n].numel() for n in names if n.startswith("mlp.w")) / (8 * 96 * 96) - 1) < 0.01
    with pytest.raises(ValueError, match="gated"):
        Block(96, (15, 31), True, mlp="gated")
    with pytest.raises(ValueError, match="mlp"):
        Block(96, (31,), False, mlp="glu")
    net = ConvNeXt1D(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40), mlp="gated", checkpoint8=True)
    assert all(stage[0].mlp.checkpoint8 for stage in net.stages)
    with pytest.raises(ValueError, match="classes"):
        ConvNeXt1D(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40), out_stages=True).loss(torch.zeros(1, 3, 32, 32), torch.zeros(1))


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_transforms_over_rows(reduction):
    """Per-sample gradients: x [C] and a target of no dimensions inside."""
    F = torch.nn.functional
    x, w, b = torch.randn(4, 8), torch.randn(16, 8), torch.randn(16)
    target = torch.tensor([0, 3, -100, 15])
    each = F.cross_entropy(F.linear(x, w, b), target, reduction="none", label_smoothing=0.1)
    want = torch.where(target == -100, float("nan"), each) if reduction == "mean" else each  # (a mean over no rows)

    def call(row, t, weight):
        return losses.linear_cross_entropy(row, weight, b, t, reduction=reduction, label_smoothing=0.1)

    got = torch.func.vmap(call, (0, 0, None))(x, target, w)
    assert torch.allclose(got, want, atol=1e-5, equal_nan=True)
    grads = torch.func.vmap(torch.func.grad(call, argnums=2), (0, 0, None))(x, target, w)
    leaf = w.clone().requires_grad_()
    for k in range(4):
        loss = F.cross_entropy(F.linear(x[k], leaf, b)[None], target[k:k + 1], reduction="sum", label_smoothing=0.1)
        assert torch.allclose(grads[k], torch.autograd.grad(loss, leaf)[0], atol=1e-5)


def test_transforms_of_targets_that_are_no_class():
    """NaN in the row and its gradient alone, as outside of a transform; and targets to ignore that are a class."""
    F = torch.nn.functional
    x, w, b = torch.randn(3, 5, 8), torch.randn(6, 8), torch.randn(6)
    target = torch.tensor([[0, 6, -1, 5, -100]] * 3)
    got = torch.func.vmap(lambda a, t: losses.linear_cross_entropy(a, w, b, t, reduction="none"))(x, target)
    assert got[:, 1:3].isnan().all() and torch.isfinite(got[:, [0, 3]]).all() and (got[:, 4] == 0).all()
    dx = torch.func.vmap(torch.func.grad(lambda a, t: losses.linear_cross_entropy(a, w, b, t, reduction="none").sum()))(x, target)
    assert dx[:, 1:3].isnan().all() and torch.isfinite(dx[:, [0, 3]]).all() and (dx[:, 4] == 0).all()
    assert torch.func.vmap(lambda a, t: losses.linear_cross_entropy(a, w, b, t))(x, target).isnan().all()
    target = torch.tensor([[0, 5, 2, 5, 1]] * 3)
    want = torch.stack([F.cross_entropy(F.linear(a, w, b), t, ignore_index=5) for a, t in zip(x, target)])
    got = torch.func.vmap(lambda a, t: losses.linear_cross_entropy(a, w, b, t, ignore_index=5))(x, target)
    assert torch.allclose(got, want, atol=1e-5)
    # a row that is ignored may hold anything
    x[:, 1] = float("nan")
    got = torch.func.vmap(lambda a, t: losses.linear_cross_entropy(a, w, b, t, ignore_index=5))(x, target)
    assert torch.isfinite(got).all()
    dx = torch.func.vmap(torch.func.grad(lambda a, t: losses.linear_cross_entropy(a, w, b, t, ignore_index=5)))(x, target)
    assert torch.isfinite(dx).all() and (dx[:, 1] == 0).all()


def test_transforms_with_parameters_of_another_type():
    """16-bit activations and fp32 parameters: converted as outside of a transform, gradients of the parameters' own type."""
    x, w, b, v, c = torch.randn(3, 4, 8).bfloat16(), torch.randn(16, 8), torch.randn(16), torch.randn(5, 8), torch.randn(5)
    target = torch.tensor([[0, 3, -100, 15]] * 3)

    def loss(a, t, w, b):
        return losses.linear_cross_entropy(a, w, b, t)

    def block(a, w, b, v, c):
        return feedforward.gated_mlp(a, w, b, v, c)

    got = torch.func.vmap(loss, (0, 0, None, None))(x, target, w, b)
    assert torch.equal(got, torch.func.vmap(loss, (0, 0, None, None))(x, target, w.bfloat16(), b.bfloat16()))
    dw, db = torch.func.grad(loss, argnums=(2, 3))(x[0], target[0], w, b)
    assert dw.dtype == torch.float32 and db.dtype == torch.float32 and torch.isfinite(dw).all()
    got = torch.func.vmap(block, (0, None, None, None, None))(x, w, b, v, c)
    same = torch.func.vmap(block, (0, None, None, None, None))(x, *[t.bfloat16() for t in (w, b, v, c)])
    assert got.dtype == torch.bfloat16 and torch.equal(got, same)
    grads = torch.func.grad(lambda *p: block(x, *p).float().sum(), argnums=(0, 1, 2, 3))(w, b, v, c)
    assert all(g.dtype == torch.float32 and torch.isfinite(g).all() for g in grads)
    assert torch.equal(torch.func.vmap(block, (0, None, None, None, None))(x, w, None, v, None),
                       torch.func.vmap(block, (0, None, None, None, None))(x, w.bfloat16(), None, v.bfloat16(), None))


def test_workspace_of_many_rows_and_few_classes():
    """The logits' gradients have room for the classes that there are, padded to eight: beside them the inputs' gradient and the partial
    sums of the weights', which are small."""
    for rows, C, V in [(1 << 20, 32, 150), (1 << 24, 32, 10), (1 << 30, 8, 8), (200000, 64, 1000)]:
        for dtype, size in ((F32, 6), (BF16, 2), (F16, 2)):
            staged = rows * C * size if dtype == F32 else 0
            assert lib().dwo_head_workspace_bytes(rows, C, V, 1, dtype) <= rows * -(-V // 8) * 8 * size + staged + (1 << 26)


def test_long_sums_are_split_beside_many_tiles():
    """Weight gradients over many rows have room for their partial sums (eight splits or more) also where the inputs' gradient alone has more tiles than
    fill the chip: in one piece they would be one workgroup's."""
    L = lib()
    for rows, C, V in [(1000000, 32, 16), (1 << 22, 64, 150), (1 << 24, 32, 10)]:
        for dtype in (BF16, F16):
            held = rows * -(-V // 8) * 8 * 2
            assert L.dwo_head_workspace_bytes(rows, C, V, 1, dtype) >= held + 8 * V * C * 4
            odd = 0 if V % 8 == 0 else held  # (a copy of dy with whole pieces of eight)
            assert L.dwo_layer8_workspace_bytes(rows, C, V, 1, dtype) >= rows * C * 2 + odd + 8 * V * C * 4


def test_values_without_codes():
    L = lib()
    assert L.dwo_pack8(ONE, None, None, None, 4, 8, 0, BF16, None) == -1  # neither
    assert L.dwo_pack8(ONE, ONE, ONE, None, 4, 8, 0, BF16, None) == -1  # codes without exponents
    assert L.dwo_pack8(ONE, ONE, None, None, 0, 8, 0, BF16, None) == -2  # (accepted, but for its rows)


def test_blocks_pickled_before_they_had_an_mlp_of_their_own():
    import copy
    import pickle

    block = Block(16, (7,), False)
    state = block.__getstate__() if hasattr(block, "__getstate__") else block.__dict__
    state = {k: v for k, v in copy.copy(state if state is not None else block.__dict__).items() if k not in ("mlp", "checkpoint8")}
    old = Block.__new__(Block)
    old.__setstate__(state)
    assert old.mlp is None and old.checkpoint8 is False
    for mlp in ("plain", "gated"):
        kept = pickle.loads(pickle.dumps(Block(16, (7,), False, mlp=mlp, checkpoint8=True)))
        assert kept.checkpoint8 and (kept.mlp is None) == (mlp == "plain")


def test_transforms_give_fp32_losses_whatever_the_default_type():
    x, w, target = torch.randn(3, 4, 8), torch.randn(16, 8), torch.zeros(3, 4, dtype=torch.long)
    torch.set_default_dtype(torch.float64)
    try:
        for reduction in ("mean", "none"):
            got = torch.func.vmap(lambda a, t: losses.linear_cross_entropy(a, w, None, t, reduction=reduction))(x, target)
            assert got.dtype == torch.float32
    finally:
        torch.set_default_dtype(torch.float32)
