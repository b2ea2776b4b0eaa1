"""The operators around wide layers at magnitudes where their formulas could leave a type's range, against the formulas in 64 bits.
Tolerances as in test_wide_gpu.py where nothing else is said."""
import pytest
import torch
import torch.nn.functional as F

from oriented1d_amd import checkpoint8, feedforward, losses
from oriented1d_amd.convnext1d import ConvNeXt1D
from test_wide_gpu import DTYPES, IDS, gated64, held8, leaves64, make_gated, make_head, near

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


# ---------------------------------------------------------------------------------------------------- label smoothing up to 1
def make_sure(rows, C, V, dtype, sure, seed=0):
    """A classifier that is sure of a class in every row (probability 0.9 and more), the target in some rows and not in others; and one that is
    not (``sure`` 0)."""
    gen = torch.Generator("cuda").manual_seed(seed + rows + V)
    x = torch.randn((rows, C), generator=gen, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn((V, C), generator=gen, device="cuda") * C ** -0.5).to(dtype)
    guess = torch.randint(0, V, (rows,), generator=gen, device="cuda")
    with torch.no_grad():
        # (V classes and as many channels: a row's own channel says what it is sure of)
        if sure:
            w.zero_()
            w[torch.arange(V), torch.arange(V)] = sure
            x[:, :V] = 0
            x[torch.arange(rows), guess] = 1
    w.requires_grad_()
    b = (torch.randn((V,), generator=gen, device="cuda") * 0.3).to(dtype).requires_grad_()
    target = torch.where(torch.rand((rows,), generator=gen, device="cuda") < 0.5, guess, torch.randint(0, V, (rows,), generator=gen, device="cuda"))
    return x, w, b, target


@pytest.mark.parametrize("smoothing", [0.5, 0.75, 0.8, 0.875, 0.9, 0.99, 0.9999, 1.0])
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,C,V", [(40, 72, 10), (5000, 272, 257)], ids=str)
@pytest.mark.parametrize("sure", [0.0, 9.0])
def test_much_smoothing(rows, C, V, dtype, reduction, smoothing, sure):
    x, w, b, target = make_sure(rows, C, V, dtype, sure)
    loss = losses.linear_cross_entropy(x, w, b, target, reduction=reduction, label_smoothing=smoothing)
    up = torch.full_like(loss, 512.0 if reduction == "mean" else 1.0)  # (a mean in fp16 is trained with a scaled loss)
    got = torch.autograd.grad(loss, [x, w, b], up)
    ref = leaves64(x, w, b)
    logits = F.linear(*ref)
    want = F.cross_entropy(logits, target, reduction=reduction, label_smoothing=smoothing)
    assert ((loss.double() - want).abs() <= 4e-6 * (want.abs() + 12)).all()
    # A logit's gradient is p - smoothing / V - (1 - smoothing) [target]: what fp32 leaves of these, 1e-6 of each, and its rounding as an operand, r of
    # it.  They may have the same sign in all rows (a class that nobody has is off by the same rounding in each), so the limit is the sum of the
    # magnitudes; then the result's rounding, and what fp32 sums lose.
    r = torch.finfo(dtype).eps / 2
    up64 = up.double().reshape(-1, 1) / (rows if reduction == "mean" else 1)
    size = torch.softmax(logits, 1).detach() + smoothing / V
    size[torch.arange(rows), target] += 1 - smoothing
    held = torch.autograd.grad(want, logits, up.double(), retain_graph=True)[0].abs()
    size = 1e-6 * size * up64 + (r + 4e-6) * held
    limits = size @ ref[1].detach().abs(), size.t() @ ref[0].detach().abs(), size.sum(0)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    for g, t, m, name in zip(got, torch.autograd.grad(want, ref, up.double()), limits, ["dx", "dw", "db"]):
        assert torch.isfinite(g).all(), "%s: %d not finite" % (name, int((~torch.isfinite(g)).sum()))
        off = (g.double() - t).abs() - r * t.abs() - m - tiny
        assert float(off.max()) <= 0.0, "%s: %.3g beyond the limit" % (name, float(off.max()))


# ---------------------------------------------------------------------------------------------------- what arrives at rows that do not count
@pytest.mark.parametrize("value", [1e30, float("inf"), float("nan")])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_what_arrives_at_ignored_rows_changes_nothing(dtype, value):
    """A weight of a masked row may be anything, 1 / 0 among it: the other rows' gradients are as with a zero there, bit for bit."""
    x, w, b, target = make_head(300, 64, 130, dtype, ignored=0.3)
    up = torch.rand(300, device="cuda") + 0.5
    results = []
    for at_ignored in (0.0, value):
        loss = losses.linear_cross_entropy(x, w, b, target, reduction="none")
        results.append(torch.autograd.grad(loss, [x, w, b], torch.where(target == -100, at_ignored, up)))
    for clean, got in zip(*results):
        assert torch.isfinite(got).all() and torch.equal(got, clean)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_a_row_with_an_infinite_weight_stays_apart(dtype):
    x, w, b, target = make_head(200, 64, 130, dtype)
    up = torch.rand(200, device="cuda") + 0.5
    up[7] = 0
    clean, = torch.autograd.grad(losses.linear_cross_entropy(x, w, b, target, reduction="none"), x, up)
    for value in (float("inf"), float("nan")):
        up[7] = value
        dx, = torch.autograd.grad(losses.linear_cross_entropy(x, w, b, target, reduction="none"), x, up)
        assert not torch.isfinite(dx[7]).any()
        dx[7] = clean[7]
        assert torch.equal(dx, clean)
    # nor does one whose target is no class
    target[9], up[7], up[9] = 130, 1.0, 0.0
    first, = torch.autograd.grad(losses.linear_cross_entropy(x, w, b, target, reduction="none"), x, up)
    up[9] = 1e30
    dx, = torch.autograd.grad(losses.linear_cross_entropy(x, w, b, target, reduction="none"), x, up)
    assert dx[9].isnan().all() and torch.equal(torch.cat([dx[:9], dx[10:]]), torch.cat([first[:9], first[10:]]))


# ---------------------------------------------------------------------------------------------------- fp32 as planes of 16 bits
def test_fp32_errors_have_either_sign():
    """Operands of one sign just below a value of eight bits.  What the products of planes leave out is 2^-24 of each product at the most and of
    either sign, and fp32 sums round to the nearest: each of 4096 results is off by a few 2^-24 at random, their mean by a sixtieth of that
    (planes cut toward zero: by 3.5 2^-24)."""
    gen = torch.Generator("cuda").manual_seed(0)

    def values(*shape):
        steps = torch.randint(1, 128, shape, generator=gen, device="cuda").double() * 2.0 ** -7
        return (1 + steps - torch.randint(1, 100, shape, generator=gen, device="cuda").double() * 2.0 ** -23).float()

    x, w, dy = values(64, 2048).requires_grad_(), values(64, 2048), values(64, 64)
    y = checkpoint8.linear8(x, w)
    dx, = torch.autograd.grad(y, x, dy)
    for got, want in ((y, x.double() @ w.double().t()), (dx, dy.double() @ w.double())):
        error = float(((got.double() - want) / want).mean()) * 2.0 ** 24
        assert abs(error) <= 0.5, error


# ---------------------------------------------------------------------------------------------------- infinities
def same_kind(got, ref, what):
    """Infinite, with its sign, and not a number where the reference is."""
    got, ref = got.double(), ref.double()
    assert torch.equal(got.isnan(), ref.isnan()), "%s: %d, not %d that are no numbers" % (what, int(got.isnan().sum()), int(ref.isnan().sum()))
    assert torch.equal(torch.where(got.isinf(), got, 0), torch.where(ref.isinf(), ref, 0)), "%s: infinities" % what


def products64(a, b):
    """a b^T in 64 bits, term by term."""
    return (a.double()[:, None] * b.double()[None]).sum(-1)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [8, 9, 40, 300])
def test_infinities_of_a_layer(rows, dtype):
    """As the formula has them at any number of rows: infinite of the products' sign, no number where they meet zero or each other."""
    gen = torch.Generator("cuda").manual_seed(rows)
    x = torch.randn((rows, 72), generator=gen, device="cuda").to(dtype)
    w = torch.randn((40, 72), generator=gen, device="cuda").to(dtype)
    dy = torch.randn((rows, 40), generator=gen, device="cuda").to(dtype)
    inf = float("inf")
    w[0], w[1] = 1, -0.5  # (values of a few bits)
    w[2, 3], w[3, 5] = 0, -inf
    x[1, 3], x[2, 71], x[4, 5], x[5, 0], x[5, 1] = inf, -inf, inf, inf, -inf
    dy[1, 7], dy[3, 39], dy[6, 3] = -inf, inf, inf
    b = torch.randn((40,), generator=gen, device="cuda").to(dtype)
    x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = checkpoint8.linear8(x, w, b)
    same_kind(y, products64(x.detach(), w.detach()) + b.detach().double(), "y")
    with torch.no_grad():
        same_kind(checkpoint8.linear8(x, w, b), y, "y")
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    same_kind(dx, products64(dy, w.detach().t()), "dx")
    same_kind(dw, products64(dy.t(), held8(x.detach()).t()), "dw")
    same_kind(db, dy.double().sum(0), "db")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [3, 9, 40, 300])
@pytest.mark.parametrize("place", ["w_out", "dy", "x"])
def test_infinities_of_the_gated_block(place, rows, dtype):
    args, dy = make_gated(rows, 40, 96, 72, dtype)
    with torch.no_grad():
        if place == "w_out":
            args[3][5, 17], args[3][6, 18] = float("inf"), float("-inf")
        elif place == "dy":
            dy[1, 5], dy[2, 71] = float("inf"), float("-inf")
        else:
            args[0][1, 3] = float("inf")
    y = feedforward.gated_mlp(*args)
    ref = leaves64(*args)
    out = gated64(*ref, "gelu")
    same_kind(y, out, "y")
    got = torch.autograd.grad(y, args, dy)
    want = torch.autograd.grad(out, ref, dy.double())
    for g, t, name in zip(got, want, ["dx", "dw_in", "db_in", "dw_out", "db_out"]):
        same_kind(g, t, name)


# ---------------------------------------------------------------------------------------------------- as many rows as there may be
def test_as_many_rows_as_there_may_be():
    """2^30 rows of few channels: more tiles of the smaller sizes than a launch has room for, and more rows than a pass over them has
    threads.  The first and last rows, the others being zeros and ignored."""
    rows, C = 1 << 30, 8
    x = torch.zeros(rows, C, device="cuda", dtype=torch.bfloat16)
    ends = torch.randn(74, C, device="cuda").bfloat16()
    x[:37], x[-37:] = ends[:37], ends[37:]
    w, b = torch.randn(8, C, device="cuda").bfloat16(), torch.randn(8, device="cuda").bfloat16()
    with torch.no_grad():
        y = checkpoint8.linear8(x, w, b)
    near(torch.cat([y[:37], y[-37:]]), ends.double() @ w.double().t() + b.double(), "y")
    for m in (37, rows // 3, rows // 2 + 5, rows - 38):
        assert torch.equal(y[m], b)
    del y
    target = torch.full((rows,), -100, device="cuda")
    some = torch.randint(0, 8, (74,), device="cuda")
    target[:37], target[-37:] = some[:37], some[37:]
    x.requires_grad_()
    w.requires_grad_()
    loss = losses.linear_cross_entropy(x, w, b, target)
    dx, dw = torch.autograd.grad(loss, [x, w])
    ref = leaves64(ends, w)
    want = F.cross_entropy(F.linear(*ref, b.double()), some)
    assert abs(float(loss) - float(want)) <= 4e-6 * (abs(float(want)) + 12)
    for g, t, name in zip((torch.cat([dx[:37], dx[-37:]]), dw), torch.autograd.grad(want, ref), ["dx", "dw"]):
        near(g, t, name)
    assert not dx[37:1000].any() and not dx[rows // 2:rows // 2 + 1000].any() and not dx[-1000:-37].any()
    del x, target, loss, dx, g
    torch.cuda.empty_cache()  # (80 GB)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_rows_and_few_classes(dtype):
    """A product of many tiles next to one of long sums, which are split."""
    rows, C, V = 400003, 24, 20
    x, w, b, target = make_head(rows, C, V, dtype, ignored=0.1)
    up = torch.randn(rows, device="cuda")
    loss = losses.linear_cross_entropy(x, w, b, target, reduction="none")
    ref = leaves64(x, w, b)
    want = F.cross_entropy(F.linear(*ref), target, reduction="none", ignore_index=-100)
    near(loss, want, "loss")
    for g, t, name in zip(torch.autograd.grad(loss, [x, w, b], up), torch.autograd.grad(want, ref, up.double()), ["dx", "dw", "db"]):
        near(g, t, name)
    y = checkpoint8.linear8(x, w, b)
    dy = torch.randn_like(y)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    near(dx, dy.double() @ w.double(), "dx")
    near(dw, dy.double().t() @ held8(x.detach()), "dw")
    near(db, dy.double().sum(0), "db")


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_activation_without_gradients_keeps_nothing(dtype, act):
    """The same bits as with them; no codes are made where nothing will read them."""
    for shape in ((4096, 1024), (1000, 333), (7,), (0, 64)):
        x = (3 * torch.randn(shape, device="cuda")).to(dtype)
        want = checkpoint8.act8(x.clone().requires_grad_(), act).detach()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        y = checkpoint8.act8(x, act)
        taken = torch.cuda.max_memory_allocated() - before
        # (codes are a byte a value; what the allocator hands out beyond what is asked for is at most 1 MB)
        assert taken <= y.numel() * y.element_size() + max(y.numel() // 2, 1 << 20)
        assert torch.equal(y, want)
        with torch.no_grad():
            assert torch.equal(checkpoint8.act8(x.clone().requires_grad_(), act), want)


# ---------------------------------------------------------------------------------------------------- the networks' loss
def test_loss_goes_through_the_networks_call():
    """Hooks on the network see it, and a wrapper of its call can take it."""
    torch.manual_seed(0)
    net = ConvNeXt1D(num_classes=11, depths=(1, 1, 1, 1), dims=(32, 32, 64, 64)).cuda()
    image, target = torch.randn(2, 3, 64, 64, device="cuda"), torch.tensor([3, -1], device="cuda")
    want = F.cross_entropy(net(image), target, ignore_index=-1, label_smoothing=0.2)

    class Wrapper(torch.nn.Module):
        def __init__(self, module):
            super().__init__()
            self.module = module

        def forward(self, *args, **kwargs):
            return self.module(*args, **kwargs)

    seen = []
    handle = net.register_forward_hook(lambda module, args, out: seen.append(out))
    for loss in (net.loss(image, target, ignore_index=-1, label_smoothing=0.2),
                 Wrapper(net)(image, target, ignore_index=-1, label_smoothing=0.2)):
        assert loss.shape == () and abs(float(loss) - float(want)) <= 1e-5 * float(want)
    handle.remove()
    assert len(seen) == 2 and seen[0].shape == ()
    assert net(image).shape == (2, 11)


# ---------------------------------------------------------------------------------------------------- one row without leading dimensions
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_without_leading_dimensions(dtype):
    """x [C]: as a batch of one, in every operator, with any of the biases, and the composed forms on the GPU beside them."""
    args, _ = make_gated(1, 40, 24, 24, dtype)
    x, w_in, b_in, w_out, b_out = args
    target = torch.tensor(5, device="cuda")
    calls = [lambda a, t: checkpoint8.act8(a), lambda a, t: checkpoint8.linear8(a, w_in, b_in),
             lambda a, t: feedforward.gated_mlp(a, w_in, None, w_out, b_out), lambda a, t: feedforward.gated_mlp(a, w_in, b_in, w_out, None),
             lambda a, t: losses.linear_cross_entropy(a, w_in, b_in, t, reduction="none"),
             lambda a, t: losses.linear_cross_entropy(a, w_in, None, t, label_smoothing=0.1)]
    for k, call in enumerate(calls):
        leaf = x.detach()[0].requires_grad_()
        y, batch = call(leaf, target), call(x, target[None])
        assert torch.equal(y.reshape(-1), batch.reshape(-1)) and y.dim() == (0 if k > 3 else 1)
        some = [t for t in (w_in, b_in, w_out, b_out)]
        got = torch.autograd.grad(y, [leaf, *some], torch.ones_like(y), allow_unused=True)
        want = torch.autograd.grad(batch, [x, *some], torch.ones_like(batch), allow_unused=True)
        for g, t in zip(got, want):
            assert (g is None) == (t is None) and (g is None or torch.equal(g.reshape(-1), t.reshape(-1)))
    packed = checkpoint8.pack8(x.detach()[0])
    assert torch.equal(checkpoint8.unpack8(packed).double(), held8(x.detach())[0])
    r = torch.finfo(dtype).eps / 2
    for k in (2, 3, 4, 5):
        got = torch.func.vmap(calls[k])(x.detach().expand(3, -1).contiguous(), target.expand(3))
        size = float(calls[k](x, target[None]).abs().max())
        # (composed of layers: roundings of g, u, their product and the result, each of a half's size at most, through sums of 24 and 40 terms)
        assert (got - calls[k](x, target[None])).abs().max() <= 8 * r * (size + 1)
