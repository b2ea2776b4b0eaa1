"""The operators between a teacher and its student without a GPU: status codes of the C entry points before any GPU work, workspace sizes, what the
Python entry points refuse, and what they compose under transforms."""
import copy
import ctypes
import pickle

import pytest
import torch
import torch.nn.functional as F

from oriented1d_amd import _lib, int8, losses
from oriented1d_amd.convnext1d import ConvNeXt1D

ONE = ctypes.c_void_p(256)  # never dereferenced: validation fails first
ODD = ctypes.c_void_p(264)
F32, BF16, F16 = 0, 1, 2


def lib():
    return _lib.load()


def test_workspace_sizes():
    L = lib()
    for dtype in (F32, BF16, F16):
        for rows, C, D in [(1, 1, 1), (37, 333, 61), (16384, 4096, 4096), (1 << 30, 8, 8)]:
            # (a product of few or some rows takes their codes straight from x and keeps none)
            held = 0 if rows * C < 1 << 20 else rows * -(-C // 16) * 16 + rows * 4
            assert L.dwo_int8_workspace_bytes(rows, C, D, dtype) > held
        for rows, V, k in [(1, 1, 1), (1, 65536, 64), (1 << 30, 100, 8), (3, 1 << 24, 1024)]:
            assert L.dwo_top_workspace_bytes(rows, V, k, dtype) > 0
        for rows, C, V, k in [(1, 1, 1, 1), (8192, 1024, 65536, 64), (1 << 24, 8, 8, 8), (1, 8, 1 << 24, 1024)]:
            assert all(L.dwo_distill_workspace_bytes(rows, C, V, k, b, dtype) > 0 for b in (0, 1))
    for bad in [(0, 8, 8), (1, 0, 8), (1, 8, 0), ((1 << 30) + 1, 8, 8), (1, 65537, 8), (1, 8, 65537)]:
        assert L.dwo_int8_workspace_bytes(*bad, BF16) == 0
    assert L.dwo_int8_workspace_bytes(1, 8, 8, 3) == 0
    for bad in [(0, 8, 1), (1, 8, 0), (1, 8, 9), (1, 2000, 1025), (1, (1 << 24) + 1, 1), (1 << 30, 1 << 20, 1)]:
        assert L.dwo_top_workspace_bytes(*bad, BF16) == 0
    for bad in [(0, 8, 8, 1), (1, 8, 8, 0), (1, 8, 8, 1025), (1, 8, (1 << 24) + 1, 1), (1, 65537, 8, 1)]:
        assert L.dwo_distill_workspace_bytes(*bad, 0, BF16) == 0
    # the logits are not kept: 268 MB of their gradients a piece, of 1 GB in all, and an eighth of a byte a row and class forward
    assert L.dwo_distill_workspace_bytes(8192, 1024, 65536, 64, 0, BF16) < 8192 * 65536 // 4
    assert L.dwo_distill_workspace_bytes(8192, 1024, 65536, 64, 1, BF16) < 3 * (1 << 28) + 8192 * 1024 * 4


def test_all_logits_are_kept_up_to_256_megabytes():
    """Of few classes for each entry; their rows are of whole sixteen bytes.  Beside them 8 bytes a row and tile of classes."""
    L = lib()
    for V in (5, 9, 13, 4, 16, 31):
        for k in (1, 8):
            pitch = -(-V // 4) * 4
            for rows in ((1 << 26) // V, (1 << 26) // pitch):  # (more than that, or as much)
                # (where they are not kept, a word for each 64 classes, of which a row has whole sixteen bytes as well)
                words = 0 if V <= 24 * k and rows * pitch <= 1 << 26 else rows * 16
                held = (1 << 28 if words == 0 else words) + rows * 8 * (2 if V > 16 else 1)
                assert L.dwo_distill_workspace_bytes(rows, 8, V, k, 0, BF16) <= held + (1 << 23), (V, k, rows)


def test_status_codes():
    L = lib()

    def linear(x=ONE, codes=ONE, steps=ONE, y=ONE, ws=ONE, need=1 << 40, rows=4, C=8, D=8, act=-1, dtype=BF16):
        return L.dwo_int8_linear(x, codes, steps, None, y, ws, need, rows, C, D, act, dtype, None)

    assert linear(x=None) == -1 and linear(codes=None) == -1 and linear(steps=None) == -1 and linear(y=None) == -1 and linear(ws=None) == -1
    assert linear(rows=0) == -2 and linear(C=0) == -2 and linear(D=0) == -2 and linear(act=2) == -2 and linear(act=-2) == -2
    assert linear(x=ODD) == -2 and linear(codes=ODD) == -2 and linear(ws=ODD) == -2 and linear(C=65537) == -2
    assert linear(dtype=3) == -5 and linear(need=1) == -7
    assert L.dwo_int8_rows(None, ONE, ONE, 4, 8, BF16, None) == -1 and L.dwo_int8_rows(ONE, None, ONE, 4, 8, BF16, None) == -1
    assert L.dwo_int8_rows(ONE, ONE, ONE, 0, 8, BF16, None) == -2 and L.dwo_int8_rows(ODD, ONE, ONE, 4, 8, BF16, None) == -2
    assert L.dwo_int8_rows(ONE, ONE, ONE, 4, 8, 5, None) == -5

    def top(x=ONE, v=ONE, p=ONE, ws=ONE, need=1 << 40, rows=4, V=100, k=5, dtype=BF16):
        return L.dwo_top(x, v, p, ws, need, rows, V, k, dtype, None)

    assert top(x=None) == -1 and top(v=None) == -1 and top(p=None) == -1 and top(ws=None) == -1
    assert top(rows=0) == -2 and top(k=0) == -2 and top(k=101) == -2 and top(V=3000, k=1025) == -2 and top(x=ODD) == -2
    assert top(p=ctypes.c_void_p(260)) == -2 and top(v=ctypes.c_void_p(257)) == -2
    assert top(dtype=3) == -5 and top(need=1) == -7

    def forward(x=ONE, t=ONE, c=ONE, T=1.0, keep=ONE, loss=ONE, ws=ONE, need=1 << 40, rows=4, V=10, k=3, dtype=BF16, other=F32):
        return L.dwo_distill_forward(x, ONE, None, t, c, T, keep, loss, ONE, ws, need, rows, 8, V, k, dtype, other, None)

    assert forward(x=None) == -1 and forward(t=None) == -1 and forward(c=None) == -1 and forward(keep=None) == -1 and forward(loss=None) == -1
    assert forward(rows=0) == -2 and forward(V=0) == -2 and forward(k=0) == -2 and forward(k=1025) == -2 and forward(x=ODD) == -2
    for T in (0.0, -1.0, 1e-5, 1e5, float("nan"), float("inf")):
        assert forward(T=T) == -2
    assert forward(c=ctypes.c_void_p(260)) == -2 and forward(t=ctypes.c_void_p(258)) == -2
    assert forward(dtype=3) == -5 and forward(other=7) == -5 and forward(need=1) == -7

    def backward(up=ONE, dx=ONE, dw=ONE, db=ONE, need=1 << 40, grad=F32, T=1.0):
        return L.dwo_distill_backward(up, ONE, ONE, None, ONE, T, None, dx, dw, db, ONE, need, 4, 8, 10, 3, BF16, grad, None)

    assert backward(up=None) == -1 and backward(dw=None) == -2 and backward(T=0.0) == -2 and backward(grad=4) == -5 and backward(need=1) == -7


def test_python_refusals():
    x, w, b = torch.randn(4, 8), torch.randn(16, 8), torch.randn(16)
    t, c = torch.randn(4, 3), torch.zeros(4, 3, dtype=torch.long)
    held = int8.QuantizedRows(torch.zeros(16, 16, dtype=torch.int8), torch.ones(16))
    for call in (lambda: int8.quantize_rows(x), lambda: int8.linear_int8(x, held, b), lambda: losses.top_logits(x, 3),
                 lambda: losses.linear_distillation(x, w, b, t, c)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(ValueError, match="activation"):
        int8.linear_int8(x, held, activation="relu")
    for k in (0, 9, -1):
        with pytest.raises(ValueError, match="k must"):
            losses.top_logits(x, k)
    with pytest.raises(TypeError):
        losses.top_logits(x, 2.5)
    with pytest.raises(ValueError, match="reduction"):
        losses.linear_distillation(x, w, b, t, c, reduction="sum")
    for T in (0.0, -1.0, float("nan"), float("inf"), 1e-5, 1e5):
        with pytest.raises(ValueError, match="temperature"):
            losses.linear_distillation(x, w, b, t, c, temperature=T)
    for call in (lambda: torch.func.vmap(lambda v: int8.linear_int8(v, held))(x[None]), lambda: torch.func.vmap(int8.quantize_rows)(x[None])):
        with pytest.raises(RuntimeError, match="ordinary tensors"):
            call()
    net = ConvNeXt1D(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40), out_stages=True)
    with pytest.raises(ValueError, match="classes"):
        net(torch.zeros(1, 3, 32, 32), teacher=(t, c))
    net = ConvNeXt1D(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40))
    with pytest.raises(ValueError, match="not both"):
        net(torch.zeros(1, 3, 32, 32), torch.zeros(1, dtype=torch.long), teacher=(t, c))
    with pytest.raises(RuntimeError, match="no gradient"):  # (where the loss is composed as well)
        losses.distillation_of(torch.randn(4, 16), t.clone().requires_grad_(), c)


def test_layers_in_8_bits_check_their_channels():
    held = int8.QuantizedRows(torch.zeros(24, 48, dtype=torch.int8), torch.ones(24), 40)
    layer = int8.LinearInt8(int8.QuantizedRows(*held), 40)
    for x in (torch.zeros(4, 41), torch.zeros(4, 33), torch.zeros(2, 48), torch.zeros(2, 3, 39), torch.zeros(40, 1), torch.zeros(())):
        for call in (layer, lambda v: int8.linear_int8(v, held)):
            with pytest.raises(RuntimeError, match="40 channels"):
                call(x)
    for weight, channels in ((held, 41), (held, 16), (int8.QuantizedRows(*held), 49), (int8.QuantizedRows(held.codes[0], held.scales), 40)):
        with pytest.raises(ValueError, match="columns"):
            int8.LinearInt8(weight, channels)
    # a tuple of codes and scales, whose copies know their channels
    codes, scales = held
    assert codes is held.codes and scales is held.scales and len(held) == 2 and held._fields == ("codes", "scales")
    for other in (copy.copy(held), copy.deepcopy(held), pickle.loads(pickle.dumps(held))):
        assert isinstance(other, int8.QuantizedRows) and other.channels == 40 and torch.equal(other.codes, codes)
    assert int8.QuantizedRows(codes, scales).channels is None and copy.deepcopy(layer).in_features == 40


def test_networks_of_stage_outputs_have_no_top_logits():
    net = ConvNeXt1D(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40), out_stages=True)
    for call in (lambda x: net.top_logits(x, 3), lambda x: net.distill(x, (torch.zeros(1, 3), torch.zeros(1, 3, dtype=torch.long)))):
        with pytest.raises(ValueError, match="classes"):
            call(torch.zeros(1, 3, 32, 32))


def plain(logits, t, c, T):
    """Row by row, over the entries that are there."""
    out = []
    for row, tt, cc in zip(logits.double(), t.double(), c):
        there = (cc != -1) & (tt != float("-inf"))
        if not there.any():
            out.append(torch.zeros((), dtype=torch.float64))
            continue
        p, logs = F.softmax(tt[there] / T, 0), F.log_softmax(row / T, 0)[cc[there]]
        out.append(T * T * (torch.xlogy(p, p) - p * logs).sum())
    return torch.stack(out)


def test_transforms_compose_the_same_values():
    torch.manual_seed(1)
    x, w, b = torch.randn(3, 5, 8), torch.randn(16, 8), torch.randn(16)
    t, c = torch.randn(3, 5, 4), torch.randint(0, 16, (3, 5, 4))
    c[:, 1], c[:, 2, 1:], c[:, 3, 2] = -1, -1, 7
    t[:, 1], t[:, 3, 0] = float("nan"), float("-inf")
    want = torch.stack([plain(F.linear(a, w, b), u, v, 2.0) for a, u, v in zip(x, t, c)])
    got = torch.func.vmap(lambda a, u, v: losses.linear_distillation(a, w, b, u, v, temperature=2.0, reduction="none"))(x, t, c)
    assert got.dtype == torch.float32 and torch.allclose(got, want.float(), atol=1e-4)
    mean = torch.func.vmap(lambda a, u, v: losses.linear_distillation(a, w, b, u, v, temperature=2.0))(x, t, c)
    assert torch.allclose(mean, want.float().sum(1) / 4, atol=1e-4)
    # gradients, and rows without entries that hold anything
    x[:, 1] = float("nan")
    dx = torch.func.vmap(torch.func.grad(lambda a, u, v: losses.linear_distillation(a, w, b, u, v, temperature=2.0)))(x, t, c)
    leaf = torch.where(x.isnan(), 0.0, x).double().requires_grad_()
    ref, = torch.autograd.grad(sum(plain(F.linear(a, w.double(), b.double()), u, v, 2.0).sum() / 4 for a, u, v in zip(leaf, t, c)), leaf)
    assert torch.allclose(dx, ref.float(), atol=1e-4) and (dx[:, 1] == 0).all()
    # an entry that is none: NaN in its row alone
    c[:, 0, 2], t[:, 4, 1] = 16, float("inf")
    got = torch.func.vmap(lambda a, u, v: losses.linear_distillation(a, w, b, u, v, reduction="none"))(x, t, c)
    assert got[:, [0, 4]].isnan().all() and torch.isfinite(got[:, 1:4]).all()
    assert torch.func.vmap(lambda a, u: losses.linear_distillation(a, w, b, u, torch.full((5, 4), -1)))(x, t).isnan().all()


def test_the_composed_loss_refuses_other_reductions():
    own, t, c = torch.randn(4, 9), torch.randn(4, 3), torch.randint(0, 9, (4, 3))
    for reduction in ("sum", "batchmean", None):
        with pytest.raises(ValueError, match="reduction"):
            losses.distillation_of(own, t, c, reduction=reduction)


def test_absent_entries_may_be_of_any_class():
    torch.manual_seed(2)
    own, t, c = torch.randn(4, 9), torch.randn(4, 3), torch.randint(0, 9, (4, 3))
    t[:, 1] = float("-inf")
    want = losses.distillation_of(own, t, c, reduction="none")
    c[:, 1] = torch.tensor([9, -2, -1, 1 << 40])
    assert torch.equal(losses.distillation_of(own, t, c, reduction="none"), want)


def test_top_logits_under_transforms():
    x = torch.tensor([[1.0, 3.0, 3.0, float("nan"), -0.0, 0.0], [2.0, 2.0, 2.0, 2.0, 2.0, float("-inf")]])
    got = torch.func.vmap(lambda v: losses.top_logits(v, 5))(x)
    assert got[1].tolist() == [[3, 1, 2, 0, 4], [0, 1, 2, 3, 4]] and got[0][0, 1:4].tolist() == [3.0, 3.0, 1.0]


def test_networks_in_8_bits_keep_the_layers_that_are_not_theirs():
    from oriented1d_amd.convnext1d import Block

    block = Block(16, (7,), False, mlp="gated")
    assert int8.quantize_network(block) is block and not any(isinstance(m, int8.LinearInt8) for m in block.modules())


def test_layers_that_are_more_than_linear_are_not_put_away():
    class Adapted(torch.nn.Linear):
        def forward(self, x):
            return 2 * super().forward(x)

    for change in (lambda n: setattr(n, "head", Adapted(40, 10)), lambda n: n.head.register_forward_hook(lambda m, a, y: 2 * y)):
        net = ConvNeXt1D(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40), num_classes=10)
        change(net)
        with pytest.raises(ValueError, match="head of a ConvNeXt1D"):
            int8.quantize_network(net)
        assert not any(isinstance(m, int8.LinearInt8) for m in net.modules())
