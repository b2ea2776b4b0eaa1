"""The operators between a teacher and its student (linear layers in 8-bit integers, top logits, distillation) against their formulas in 64 bits.

Tolerances.  Codes and places are whole numbers and have to be equal.  A layer in 8-bit integers sums exactly; its scale is three fp32 factors and the
sum's conversion (five roundings of 2^-24), and the activations are within 1e-6 of what they are given: a value before the last rounding is
off by 1e-6 of the magnitudes of sum and bias at the most, and the result by half a step (eps / 2 of the type) more.  The loss is a sum of p (log p - log
q) over the entries, T^2 times: logits of at most L and their log-sum-exp are off by 1e-6 L each, divided by T; the logarithms by 2^-23 of themselves.
Gradients are held to ``near`` of test_wide_gpu."""
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
import torch.utils.checkpoint
from test_wide_gpu import DTYPES, IDS, leaves64, near

from oriented1d_amd import int8, losses
from oriented1d_amd.convnext1d import ConvNeXt1D

pytestmark = pytest.mark.gpu
ACT = {None: lambda v: v, "gelu": F.gelu, "silu": F.silu}


# ---------------------------------------------------------------------------------------------------- 8-bit integers
def codes64(x):
    """Codes of the rows of x and their largest magnitudes, in 64 bits: whole steps, and what is left of them against half a step, all exact."""
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    t = x.abs() * 127
    whole = torch.floor(t / a)
    rest = 2 * (t - whole * a)
    whole = torch.where((rest > a) | ((rest == a) & (whole % 2 == 1)), whole + 1, whole)
    return torch.where(a > 0, torch.sign(x) * whole, 0.0), a


def values(*shape, dtype=torch.float32, seed=0, std=1.0):
    gen = torch.Generator("cuda").manual_seed(seed + sum(shape))
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (5, 7), (3, 16), (70, 100), (9, 128), (33, 136), (17, 512), (64, 333), (2, 3, 2048), (5, 2050), (3, 8192),
                                   (3, 9001), (2, 65536), (1000, 24)], ids=str)
def test_quantize_rows(shape, dtype):
    torch.manual_seed(shape[0])
    x = values(*shape, dtype=dtype)
    x = x * torch.exp(3 * torch.randn(shape[:-1] + (1,), device="cuda")).to(dtype)
    got = int8.quantize_rows(x)
    C = shape[-1]
    # (of many rows in fp16 one may be beyond its largest number: zeros, and a scale that is NaN)
    odd = ~torch.isfinite(x).all(-1)
    assert got.scales[odd].isnan().all() and not got.codes[odd].any()
    got = int8.QuantizedRows(got.codes, torch.where(odd, 0.0, got.scales))
    want, a = codes64(torch.where(odd.unsqueeze(-1), 0.0, x))
    assert got.codes.dtype == torch.int8 and got.codes.shape == shape[:-1] + (-(-C // 16) * 16,) and got.scales.shape == shape[:-1]
    assert torch.equal(got.codes[..., :C].double(), want) and not got.codes[..., C:].any()
    assert torch.equal(got.scales, (a[..., 0] / 127).float()) or ((got.scales.double() - a[..., 0] / 127).abs() <= 2.0 ** -24 * a[..., 0] / 127).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("C", [254, 256, 1021])
def test_codes_at_the_middle_of_two(C, dtype):
    """127 x / a is the middle of two whole numbers at odd multiples of a / 254; a = 254 2^e, and the neighbours of such values."""
    k = torch.arange(-253, 254, 2, device="cuda").float()
    rows = []
    for e in (-14, -3, 0, 7):
        row = torch.zeros(C, device="cuda")
        n = min(C - 1, k.numel())
        row[:n] = k[:n]
        row[C - 1] = 254.0
        rows.append(row * 2.0 ** e)
    x = torch.stack(rows).to(dtype)
    x = torch.cat([x, x.flip(-1), -x])
    # neighbours: the last place of each value up and down
    bits = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    for step in (1, -1):
        moved = torch.where((x != 0) & (x.abs() < x.abs().amax(-1, keepdim=True)), bits + step, bits).view(dtype)
        x = torch.cat([x, moved])
        bits = x.view(bits.dtype)
    want, _ = codes64(x)
    assert torch.equal(int8.quantize_rows(x).codes[:, :C].double(), want)
    # and of any values
    y = values(200, C, dtype=dtype, seed=1)
    y[:, 0] = y.abs().amax(1)
    y[:, 1] = y[:, 0] / 2
    assert torch.equal(int8.quantize_rows(y).codes[:, :C].double(), codes64(y)[0])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_codes_of_extreme_rows(dtype):
    info = torch.finfo(dtype)
    tiny = info.smallest_normal * info.eps  # the smallest number
    x = torch.zeros(9, 40, device="cuda", dtype=dtype)
    x[1, 3] = tiny
    x[2] = torch.arange(40, device="cuda").to(dtype) * tiny
    x[3] = values(40, dtype=torch.float32).clamp(-1, 1).mul(info.max).to(dtype)
    x[4], x[4, 7] = 1.0, float("inf")
    x[5], x[5, 39] = 1.0, float("nan")
    x[6, 0], x[6, 1] = -info.max, info.smallest_normal
    x[7] = -0.0
    x[8] = 1.0
    got = int8.quantize_rows(x)
    good = [0, 1, 2, 3, 6, 7, 8]
    assert torch.equal(got.codes[good, :40].double(), codes64(x[good])[0])
    assert (got.codes[4:6] == 0).all() and got.scales[4:6].isnan().all() and got.scales[0] == 0 and got.scales[7] == 0
    w = int8.quantize_rows(torch.eye(40, device="cuda", dtype=dtype))
    for rows in (x, x.repeat(20, 1)):
        y = int8.linear_int8(rows, w)
        want, a = codes64(x)
        ref = (want * a / 127)[good]
        floor = tiny / 2 if dtype != torch.float32 else tiny
        assert ((y[:9][good].double() - ref).abs() <= (info.eps / 2 + 1e-6) * ref.abs() + floor).all()
        assert y[4:6].isnan().all() and torch.equal(y[-9:].isnan(), y[:9].isnan())


def int8_64(x, w, b, act):
    q, a = codes64(x)
    p, s = codes64(w)
    s = (s[:, 0] / 127).float().double()  # (as the scales are held)
    v = (q @ p.t()) * (a / 127) * s
    size = v.abs()
    if b is not None:
        v, size = v + b.double(), size + b.double().abs()
    return ACT[act](v), size


def int8_near(y, ref, size, what=""):
    r = torch.finfo(y.dtype).eps / 2
    floor = 2.0 ** -25 if y.dtype == torch.float16 else 1e-36
    off = (y.double() - ref).abs() - r * ref.abs() - 1e-6 * (1 + r) * size - floor
    assert torch.isfinite(y).all() and float(off.max()) <= 0, "%s: %.3g too far" % (what, float(off.max()))


INT8 = [(1, 1, 1), (1, 16, 7), (1, 1024, 4096), (2, 333, 61), (3, 4096, 40), (4, 48, 5000), (5, 100, 33), (8, 2048, 96), (9, 520, 130), (16, 64, 64),
        (17, 1040, 72), (37, 333, 61), (64, 768, 1000), (130, 31, 257), (300, 2064, 200), (1100, 384, 1536), (2049, 136, 640), (33, 8200, 24),
        (40, 2000, 70), (100, 1500, 33), (3000, 17, 30), (4000, 384, 300), (17000, 40, 16)]


@pytest.mark.parametrize("act", [None, "gelu", "silu"], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", INT8, ids=str)
def test_linear_int8(shape, dtype, act):
    rows, C, D = shape
    x, w = values(rows, C, dtype=dtype) * torch.linspace(0.1, 8, rows, device="cuda").to(dtype)[:, None], values(D, C, dtype=dtype, std=C ** -0.5)
    b = values(D, dtype=dtype, std=0.3) if rows % 2 == 1 else None
    y = int8.linear_int8(x, int8.quantize_rows(w), b, activation=act)
    assert y.dtype == dtype and y.shape == (rows, D) and y.is_contiguous()
    int8_near(y, *int8_64(x, w, b, act))


@pytest.mark.parametrize("rows,C,D", [(6001, 1030, 2100), (20000, 72, 96), (700, 65536, 40), (2, 65536, 3)], ids=str)
def test_linear_int8_large(rows, C, D):
    x, w, b = values(rows, C, dtype=torch.bfloat16), values(D, C, std=C ** -0.5), values(D, dtype=torch.bfloat16)
    # (the largest sums: every code 127)
    x[0], w[0] = 1.0, 1.0
    y = int8.linear_int8(x, int8.quantize_rows(w), b, activation="gelu")
    int8_near(y, *int8_64(x, w, b, "gelu"))


def test_linear_int8_shapes_strides_and_types():
    w = values(40, 50)
    held, b = int8.quantize_rows(w), values(40)
    x = values(2, 3, 4, 50)
    want = int8.linear_int8(x.reshape(24, 50), held, b)
    assert torch.equal(int8.linear_int8(x, held, b), want.view(2, 3, 4, 40))
    assert torch.equal(int8.linear_int8(x[0, 0, 0], held, b), want[0])
    wide = torch.zeros(24, 101, device="cuda")
    wide[:, 1::2] = x.reshape(24, 50)
    assert torch.equal(int8.linear_int8(wide[:, 1::2], held, b), want)
    part = torch.zeros(24 * 50 + 1, device="cuda")
    part[1:] = x.flatten()
    assert torch.equal(int8.linear_int8(part[1:].view(24, 50), held, b), want)
    wider = int8.QuantizedRows(torch.cat([held.codes, held.codes]).t().contiguous().t()[:40], held.scales)
    assert torch.equal(int8.linear_int8(x.reshape(24, 50), wider, b), want)
    assert int8.linear_int8(torch.zeros(0, 50, device="cuda"), held).shape == (0, 40)
    assert int8.linear_int8(torch.zeros(3, 0, 50, device="cuda"), held, activation="gelu").shape == (3, 0, 40)
    assert int8.quantize_rows(torch.zeros(0, 50, device="cuda")).codes.shape == (0, 64)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = int8.linear_int8(x.reshape(24, 50), held, b)
    assert torch.equal(y, int8.linear_int8(x.reshape(24, 50).bfloat16(), held, b.bfloat16()))
    # a bias of another type is converted, as parameters are
    assert torch.equal(int8.linear_int8(x.half(), held, b), int8.linear_int8(x.half(), held, b.half()))


def test_linear_int8_rows_stay_apart():
    """A row is the same alone, among others, and beside rows that are not finite."""
    for dtype in DTYPES:
        w, b = int8.quantize_rows(values(130, 200, dtype=dtype)), values(130, dtype=dtype)
        x = values(300, 200, dtype=dtype)
        y = int8.linear_int8(x, w, b, "gelu")
        for n in (1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 64, 65):
            assert torch.equal(int8.linear_int8(x[:n], w, b, "gelu"), y[:n]), n
        x[3, 4], x[7, 199] = float("nan"), float("-inf")
        for n in (8, 300):
            z = int8.linear_int8(x[:n], w, b, "gelu")
            others = [m for m in range(n) if m not in (3, 7)]
            assert z[3].isnan().all() and z[7].isnan().all() and torch.equal(z[others], y[others])


@pytest.mark.parametrize("act", [None, "gelu", "silu"], ids=str)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_int8_is_the_same_whichever_way_a_row_goes(dtype, act):
    """Few rows, some, many short ones, and tiles: whole numbers are summed, and what follows is rounded alike."""
    w, b = int8.quantize_rows(values(800, 200, dtype=dtype)), values(800, dtype=dtype)
    x = values(2100, 200, dtype=dtype) * torch.exp(3 * values(2100, 1)).to(dtype).clamp(max=1000)
    y = int8.linear_int8(x, w, b, act)
    for n in (1, 16, 17, 200, 1900):
        assert torch.equal(int8.linear_int8(x[:n], w, b, act), y[:n]), n


def test_linear_int8_scales_of_all_sizes():
    """Steps whose product with a row's is no number of fp32, though the result is; and weights that are not finite."""
    x, w = values(6, 64), values(5, 64)
    held = int8.quantize_rows(w)
    want = int8_64(x, w, None, None)[0]
    for e in (-100, 100):
        y = int8.linear_int8(x * 2.0 ** e, int8.QuantizedRows(held.codes, held.scales * 2.0 ** -e))
        assert ((y.double() - want).abs() <= 1e-6 * want.abs()).all()
    w[2, 3], w[4, 5] = float("inf"), float("nan")
    y = int8.linear_int8(x, int8.quantize_rows(w))
    assert y[:, [2, 4]].isnan().all() and ((y[:, [0, 1, 3]].double() - want[:, [0, 1, 3]]).abs() <= 1e-6 * want[:, [0, 1, 3]].abs()).all()


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
def test_linear_int8_is_the_same_where_a_step_is_almost_none(dtype):
    """Magnitudes and scales around 2^-60: what a whole number stands for is near 2^-127, where fp32 has a bit less, and the results above that."""
    w = values(800, 200, dtype=dtype)
    held = int8.quantize_rows(w)
    x = values(2100, 200, dtype=dtype)
    for e, f in ((-61, -60), (-60, -60), (-60, -61), (-59, -60), (-59, -59), (-62, -58)):
        # every row's largest is 1.0 .. 2.0 times 2^e, every scale 1.0 .. 2.0 times 2^f
        a = x * (torch.rand(2100, 1, device="cuda").add(1.0) * 2.0 ** e).to(dtype) / x.abs().amax(1, keepdim=True)
        scales = torch.rand(800, device="cuda").add(1.0) * 2.0 ** f
        weight = int8.QuantizedRows(held.codes, scales)
        y = int8.linear_int8(a, weight)
        q, most = codes64(a)
        want = (q @ held.codes[:, :200].double().t()) * (most / 127) * scales.double()
        assert ((y.double() - want).abs() <= (torch.finfo(dtype).eps / 2 + 3e-7) * want.abs() + 2.0 ** -127).all()
        for n in (1, 16, 17, 200, 1900):
            assert torch.equal(int8.linear_int8(a[:n], weight), y[:n]), (e, f, n)


def test_linear_int8_refusals():
    x, w = values(4, 40), int8.quantize_rows(values(24, 40))
    with pytest.raises(RuntimeError, match="no gradients"):
        int8.linear_int8(x.clone().requires_grad_(), w)
    with torch.no_grad():
        int8.linear_int8(x.clone().requires_grad_(), w)
    for bad in (int8.QuantizedRows(w.codes[:, :40].contiguous(), w.scales), int8.QuantizedRows(w.codes.float(), w.scales),
                int8.QuantizedRows(w.codes, w.scales.double()), int8.QuantizedRows(w.codes, w.scales[:3]), int8.QuantizedRows(w.codes.cpu(), w.scales),
                int8.QuantizedRows(w.codes[:0], w.scales[:0]), int8.QuantizedRows(w.codes[0], w.scales)):
        with pytest.raises(RuntimeError):
            int8.linear_int8(x, bad)
    with pytest.raises(RuntimeError):
        int8.linear_int8(x, w, torch.zeros(25, device="cuda"))
    with pytest.raises(RuntimeError):
        int8.linear_int8(x.double(), w)
    with pytest.raises(ValueError, match="activation"):
        int8.linear_int8(x, w, activation="relu")


def test_linear_int8_refuses_other_channels():
    """Codes are filled up to whole sixteen: an x with some more or fewer channels would meet zeros there, and have another largest magnitude."""
    layer = nn.Linear(40, 24).cuda()
    held, mine = int8.quantize_rows(layer.weight), int8.LinearInt8.of(layer)
    assert held.channels == 40
    x = values(4, 40)
    with torch.no_grad():
        want = int8.linear_int8(x, held, layer.bias)
        assert torch.equal(mine(x), want)
        for C in (33, 39, 41, 48, 49):
            for call in (mine, lambda v: int8.linear_int8(v, held)):
                with pytest.raises(RuntimeError, match="40 channels"):
                    call(values(4, C))
        # codes and scales by themselves say nothing of it
        assert torch.equal(int8.linear_int8(x, int8.QuantizedRows(*held), layer.bias), want)


# ---------------------------------------------------------------------------------------------------- top logits
def top64(x, k):
    v, c = torch.sort(x.cpu(), dim=-1, descending=True, stable=True)
    return v[..., :k], c[..., :k]


def same_values(a, b):
    """Bit for bit, but for which of the values that are no number."""
    a, b = a.cpu(), b.cpu()
    bits = torch.int32 if a.dtype == torch.float32 else torch.int16
    return bool(((a.view(bits) == b.view(bits)) | (a.isnan() & b.isnan())).all())


def check_top(x, k):
    got, want = losses.top_logits(x, k), top64(x, k)
    assert got.values.dtype == x.dtype and got.classes.dtype == torch.int64 and got.values.shape == x.shape[:-1] + (k,)
    assert torch.equal(got.classes.cpu(), want[1]), (tuple(x.shape), k)
    assert same_values(got.values, want[0])


TOP = [(1, 1, 1), (3, 5, 5), (7, 64, 64), (5, 65, 1), (64, 150, 8), (9, 256, 64), (10, 257, 33), (6, 1000, 64), (6, 1000, 65), (4, 1024, 16), (3, 1025, 20),
       (3, 1025, 1024), (5, 4097, 100), (2, 16376, 256), (2, 16377, 7), (3, 16384, 64), (2, 21841, 100), (2, 65528, 64), (2, 65536, 64), (1, 65537, 64),
       (3, 131072, 1), (2, 150001, 256), (1, 600000, 1024), (2, 70000, 1000),
       (4, 9000, 1024), (4, 5000, 900), (4, 3000, 256), (600, 8193, 3), (9, 512, 17), (5, 255, 16),
       (520, 700, 300), (520, 4096, 512), (520, 4097, 512), (520, 8191, 256), (3, 8192, 129), (520, 600, 512), (520, 513, 257), (3, 300, 300), (4100, 600, 300),
       (4100, 1030, 512), (4100, 4096, 257)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,V,k", TOP, ids=str)
def test_top_logits(rows, V, k, dtype):
    check_top(values(rows, V, dtype=dtype, std=3.0), k)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("V,k", [(40, 7), (200, 64), (1000, 64), (1000, 200), (5003, 64), (30001, 64), (65536, 100), (80001, 30)], ids=str)
def test_top_logits_of_special_rows(V, k, dtype):
    """Rows of one value, of few values, in order, with zeros of both signs, infinities and NaN, and their largest together."""
    base = values(16, V, dtype=dtype)
    at = torch.arange(V, device="cuda")
    base[0] = 1.5
    base[1] = (at % 3).to(dtype)
    base[2] = (at.float() / V).to(dtype)
    base[3] = (-at.float() / V).to(dtype)
    base[4] = torch.where(at % 2 == 0, 0.0, -0.0).to(dtype)
    base[5] = float("-inf")
    base[6] = float("-inf")
    base[6, V // 2] = 1.0
    base[7] = float("inf")
    base[8, ::5] = float("nan")
    base[9, V - 1], base[9, 3] = float("nan"), float("inf")
    base[10] = float("nan")
    base[11] = torch.where(at >= V - k, 100.0, 0.0).to(dtype)
    base[12, V // 3:V // 3 + k] += 50.0
    base[13] = torch.where(at % 97 == 0, base[13], base[13].clamp(max=0))
    base[14] = torch.where(at == V - 1, float("-nan"), -1.0).to(dtype)
    base[14].view(torch.int32 if dtype == torch.float32 else torch.int16)[1] = -1  # (a NaN with the sign)
    base[15] = torch.finfo(dtype).min
    check_top(base, k)
    # fewer values that are no number than k, more, and of both signs, at the ends of a row and inside; and ties behind them
    more = values(8, V, dtype=dtype, seed=3)
    bits = more.view(torch.int32 if dtype == torch.float32 else torch.int16)
    more[0, :k // 2 + 1] = float("nan")
    more[1, -(k // 2) - 1:] = float("nan")
    bits[2, 1::3] = -1
    bits[3, 5], bits[3, V - 2] = -1, -1
    more[3, 7] = float("nan")
    more[4] = 0.0
    more[4, 3::7] = float("nan")
    more[5] = 2.0
    bits[5, 8] = -1
    more[6] = float("inf")
    more[6, V // 2:] = float("nan")
    more[7] = float("-inf")
    more[7, 1] = float("nan")
    check_top(more, k)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("V,k", [(1000, 70), (1100, 4), (5003, 64), (8193, 300), (65536, 4), (65536, 600), (80001, 30)], ids=str)
def test_top_logits_of_numbers_that_are_none_in_several_ways(V, k, dtype):
    """NaN of different bits are one value: the lowest classes, whichever bits they have."""
    x = values(6, V, dtype=dtype)
    bits = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    low = {torch.float32: 0x7fc00000, torch.bfloat16: 0x7fc0, torch.float16: 0x7e00}[dtype]
    smallest = {torch.float32: 0x7f800001, torch.bfloat16: 0x7f81, torch.float16: 0x7c01}[dtype]
    far = torch.arange(V - 8 * min(2 * k + 20, V // 16), V, 8, device="cuda")
    bits[0, :4], bits[0, far] = low, low + 1
    bits[1, :k], bits[1, far] = smallest, low + 3
    # in every unit, the first by one bit and the others by another
    bits[2, ::2], bits[2, :k // 8 * 8 + 8] = low + 1, low
    bits[3, :], bits[3, V // 2:] = low, low + 1
    bits[4, far], bits[4, 1], bits[4, 2] = low + 2, smallest, low + 5
    bits[5, V - k - 3:V - 3], bits[5, V - 3:] = low + 1, low
    x[5, 7] = float("inf")
    assert x.isnan().any(1).all()
    check_top(x, k)


@pytest.mark.parametrize("V,k", [(2093057, 400), (2093065, 79), (2314929, 573)], ids=str)
def test_top_logits_of_a_short_last_part(V, k):
    """Rows taken in parts, the last of which has fewer values than k (17, 25 and 561) and is joined by itself at first."""
    x = values(1, V, dtype=torch.float32)
    x[0, -1] = 100.0
    for fill in (255, 1):  # (in memory that held anything)
        junk = torch.full((1 << 26,), fill, dtype=torch.uint8, device="cuda")
        del junk
        check_top(x, k)
    check_top(x.bfloat16(), k)


def test_top_logits_shapes_and_strides():
    x = values(3, 4, 200)
    check_top(x, 9)
    check_top(x[1, 2], 9)
    check_top(x.transpose(0, 1), 5)
    check_top(x[..., ::2], 5)
    check_top(x.flatten()[1:1 + 10 * 201].view(10, 201), 5)
    got = losses.top_logits(torch.zeros(0, 20, device="cuda"), 3)
    assert got.values.shape == (0, 3) and got.classes.shape == (0, 3)
    y = x.clone().requires_grad_()
    assert not losses.top_logits(y, 3).values.requires_grad
    for k in (0, -1, 201, 1025):
        with pytest.raises(ValueError, match="k must"):
            losses.top_logits(x, k)
    with pytest.raises(ValueError, match="k must"):
        losses.top_logits(values(2, 2000), 1025)
    with pytest.raises(RuntimeError):
        losses.top_logits(x.double(), 3)
    many = values(100000, 33, dtype=torch.bfloat16)
    check_top(many, 4)


# ---------------------------------------------------------------------------------------------------- distillation
def make_distill(rows, C, V, k, dtype, bias=True, absent=False, seed=0, teacher=None):
    gen = torch.Generator("cuda").manual_seed(seed + rows + V)
    x = torch.randn((rows, C), generator=gen, device="cuda").to(dtype).requires_grad_()
    w = (torch.randn((V, C), generator=gen, device="cuda") * 2 * C ** -0.5).to(dtype).requires_grad_()
    b = (torch.randn((V,), generator=gen, device="cuda") * 0.3).to(dtype).requires_grad_() if bias else None
    logits = (torch.randn((rows, k), generator=gen, device="cuda") * 3).to(teacher or dtype)
    # (classes at random: some twice, where the entries are many)
    classes = torch.randint(0, V, (rows, k), generator=gen, device="cuda")
    if absent:
        off = torch.rand((rows, k), generator=gen, device="cuda") < 0.4
        off[1::3] = True
        off[0] = False
        classes = torch.where(off, -1, classes)
        logits = torch.where(off & (torch.arange(k, device="cuda") % 2 == 0), float("nan"), logits)
        # an entry of no weight stands for none as well
        logits[2::3, k // 2] = float("-inf")
    return x, w, b, logits, classes


def distill64(x, w, b, logits, classes, T, reduction="mean"):
    """The formula, for rows without anything that is not a number."""
    own = F.log_softmax(F.linear(x, w, b) / T, -1)
    there = (classes != -1) & (logits != float("-inf"))
    t = torch.where(there, logits.double() / T, -1e300)
    some = there.any(-1)
    p = torch.where(there, torch.softmax(t, -1), 0.0)
    each = T * T * (torch.xlogy(p, p) - p * own.gather(-1, torch.where(there, classes, 0))).sum(-1)
    each = torch.where(some, each, 0.0)
    return each if reduction == "none" else each.sum() / some.sum()


def loss_limit(x, w, b, logits, T):
    with torch.no_grad():
        L = float(F.linear(x.double(), w.double(), None if b is None else b.double()).abs().max()) + 12
    finite = logits[torch.isfinite(logits)].double()
    spread = float(finite.max() - finite.min()) if finite.numel() else 0.0
    return T * T * (2e-6 * L / T + 2.0 ** -23 * (2 * L / T + 2 * spread / T + 8))


DISTILL = [(1, 16, 1, 1), (1, 16, 10, 3), (5, 7, 13, 4), (64, 768, 1000, 16), (300, 100, 257, 64), (33, 64, 21841, 100), (2000, 8, 3, 2), (700, 96, 4099, 65),
           (40, 24, 50, 1024), (17, 32, 300, 257), (130, 72, 64, 8), (3, 40, 65, 7)]


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("T,absent", [(1.0, False), (2.5, True)], ids=["plain", "warm"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", DISTILL, ids=str)
def test_linear_distillation(shape, dtype, T, absent, reduction):
    x, w, b, logits, classes = make_distill(*shape, dtype, bias=shape[0] != 5, absent=absent)
    leaves = [t for t in (x, w, b) if t is not None]
    loss = losses.linear_distillation(x, w, b, logits, classes, temperature=T, reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == (classes.shape[:1] if reduction == "none" else ())
    up = torch.rand_like(loss) + 0.5 if reduction == "none" else torch.full_like(loss, 256.0)
    got = torch.autograd.grad(loss, leaves, up)
    ref = leaves64(x, w, b)
    want = distill64(*ref, logits, classes, T, reduction)
    assert ((loss.double() - want).abs() <= loss_limit(x, w, b, logits, T) + 1e-6 * want.abs()).all()
    # the logits' gradients are differences of two probabilities, T times
    with torch.no_grad():
        there = (classes != -1) & (logits != float("-inf"))
        p = torch.where(there, torch.softmax(torch.where(there, logits.double() / T, -1e300), -1), 0.0)
        size = torch.softmax(F.linear(*ref) / T, 1).scatter_add_(1, torch.where(there, classes, 0), p)
        some = there.any(1)
        size *= torch.where(some, T * up.double() / (1 if reduction == "none" else some.sum()), 0.0)[:, None]
        terms = size @ ref[1].abs(), size.t() @ ref[0].abs(), size.sum(0)
    own = F.linear(*ref)
    each = distill64(own, torch.eye(shape[2], device="cuda").double(), None, logits, classes, T, reduction)
    size = torch.autograd.grad(each, own, up.double())[0].abs()
    rounded = size @ ref[1].abs(), size.t() @ ref[0].abs(), size.sum(0)
    for g, r, t, o, name in zip(got, torch.autograd.grad(want, [t for t in ref if t is not None], up.double()), terms, rounded, ["dx", "dw", "db"]):
        near(g, r, name, terms=t, rounded=o.detach())
    with torch.no_grad():
        again = losses.linear_distillation(x, w, b, logits, classes, temperature=T, reduction=reduction)
    assert torch.equal(again, loss)


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(500, 40, 86, 81), (150, 33, 2401, 100), (150, 33, 2400, 100), (700, 24, 193, 128), (9, 20, 7, 129), (3, 640, 20001, 5),
                                   (17, 600, 21000, 12), (100, 24, 9000, 70), (128, 100, 16388, 3)], ids=str)
def test_distillation_of_many_entries_and_of_few_rows(shape, dtype, reduction):
    """Entries that are many of few classes, and few rows of many classes, to either side of where they go another way."""
    test_linear_distillation(shape, dtype, 1.5, True, reduction)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,C,V,k", [(20000, 32, 8003, 20), (1601, 520, 2041, 64), (25003, 100, 603, 9)], ids=str)
def test_distillation_in_large_tiles_and_pieces(rows, C, V, k, dtype):
    """More rows times classes than a piece of the backward pass holds, and tiles of all sizes."""
    x, w, b, logits, classes = make_distill(rows, C, V, k, dtype)
    up = torch.tensor(512.0, device="cuda")
    loss = losses.linear_distillation(x, w, b, logits, classes, temperature=1.5)
    got = torch.autograd.grad(loss, [x, w, b], up)
    ref = leaves64(x, w, b)
    want = distill64(*ref, logits, classes, 1.5)
    assert abs(float(loss) - float(want)) <= loss_limit(x, w, b, logits, 1.5)
    for g, r, name in zip(got, torch.autograd.grad(want, ref, up.double()), ["dx", "dw", "db"]):
        near(g, r, name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_distillation_of_little_work_rounds_once(dtype):
    """The logits' gradients are held in two halves there, at the entries' places as elsewhere."""
    x, w, b, logits, classes = make_distill(37, 72, 130, 9, dtype)
    got = torch.autograd.grad(losses.linear_distillation(x, w, b, logits, classes, temperature=2.0), [x, w, b])
    ref = leaves64(x, w, b)
    r = torch.finfo(dtype).eps / 2
    for g, t, name in zip(got, torch.autograd.grad(distill64(*ref, logits, classes, 2.0), ref), ["dx", "dw", "db"]):
        rms = float(t.norm()) / math.sqrt(t.numel())
        off = (g.double() - t).abs() - r * t.abs() - 2.0 ** -14 * rms - (2.0 ** -25 if dtype == torch.float16 else 0.0)
        assert float(off.max()) <= 0, name


def test_distillation_special_rows():
    x, w, b, logits, classes = make_distill(40, 24, 50, 5, torch.float32)
    x2 = x.detach().clone()
    clean = losses.linear_distillation(x, w, b, logits, classes, reduction="none")
    clean_dx, = torch.autograd.grad(clean.sum(), x)
    logits[3, 2], logits[4, 0] = float("nan"), float("inf")
    classes[5, 1], classes[6, 4], classes[7] = 50, -2, -1
    classes[8, 1:], logits[9] = -1, float("-inf")
    logits[10, 1:] = float("-inf")
    x2[7] = float("nan")  # (a row without entries may hold anything)
    x2[9] = float("inf")
    x2.requires_grad_()
    loss = losses.linear_distillation(x2, w, b, logits, classes, reduction="none")
    dx, dw = torch.autograd.grad(loss.sum(), [x2, w])
    assert loss[3:7].isnan().all() and dx[3:7].isnan().all() and (loss[[7, 9]] == 0).all() and (dx[[7, 9]] == 0).all()
    others = [m for m in range(40) if m not in (3, 4, 5, 6, 7, 8, 9, 10)]
    assert torch.equal(loss[others], clean[others]) and torch.equal(dx[others], clean_dx[others])
    # one entry: -log q of its class
    with torch.no_grad():
        single = F.cross_entropy(F.linear(x2.double(), w.double(), b.double())[[8, 10]], classes[[8, 10], 0], reduction="none")
    assert ((loss[[8, 10]].double() - single).abs() <= 1e-4).all()
    # the mean counts the rows with entries; NaN where one is none
    assert losses.linear_distillation(x2, w, b, logits, classes).isnan()
    keep = [m for m in range(40) if m not in (3, 4, 5, 6)]
    some = losses.linear_distillation(x2[keep], w, b, logits[keep], classes[keep])
    assert abs(float(some) - float(loss[keep].sum()) / 34) <= 1e-5 * float(some)
    # no row with entries
    none = torch.full_like(classes, -1)
    loss = losses.linear_distillation(x, w, b, logits, none)
    assert loss.isnan()
    for g in torch.autograd.grad(loss, [x, w, b]):
        assert (g == 0).all()
    assert (losses.linear_distillation(x, w, b, logits, none, reduction="none") == 0).all()


def test_distillation_of_absent_entries_of_any_class():
    x, w, b, logits, classes = make_distill(20, 24, 50, 5, torch.float32)
    logits[::2, 1:3] = float("-inf")
    clean = losses.linear_distillation(x, w, b, logits, classes, reduction="none")
    wild = classes.clone()
    wild[::2, 1], wild[::4, 2] = 50, -7
    wild[2, 2] = 1 << 40
    loss = losses.linear_distillation(x, w, b, logits, wild, reduction="none")
    assert torch.isfinite(clean).all() and torch.equal(loss, clean)
    assert torch.equal(torch.autograd.grad(loss.sum(), x)[0], torch.autograd.grad(clean.sum(), x)[0])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_distillation_with_classes_twice(dtype):
    """Entries of one class count each for itself: the gradient takes the sum of their p."""
    x, w, b, logits, classes = make_distill(30, 40, 200, 12, dtype)
    classes[:, 5] = classes[:, 2]
    classes[:, 9] = classes[:, 2]
    classes[::2, 11] = classes[::2, 0]
    classes[4] = 7
    loss = losses.linear_distillation(x, w, b, logits, classes, temperature=0.5)
    ref = leaves64(x, w, b)
    want = distill64(*ref, logits, classes, 0.5)
    assert abs(float(loss) - float(want)) <= loss_limit(x, w, b, logits, 0.5)
    up = torch.tensor(64.0, device="cuda")
    for g, r in zip(torch.autograd.grad(loss, [x, w, b], up), torch.autograd.grad(want, ref, up.double())):
        near(g, r, "gradient")


def test_distillation_of_impossible_classes():
    """A class whose logit is -infinity: no loss can be finite where the teacher has it; elsewhere it changes nothing."""
    x, w, b, logits, classes = make_distill(20, 24, 70, 4, torch.float32)
    classes = torch.where(classes == 5, 6, classes)
    classes[3, 1] = 5
    with torch.no_grad():
        b[5] = float("-inf")
    loss = losses.linear_distillation(x, w, b, logits, classes, reduction="none")
    with torch.no_grad():
        want = distill64(x.double(), w.double(), b.double(), logits, classes, 1.0, "none")
    assert loss[3] == float("inf") and torch.isfinite(loss[:3]).all() and torch.isfinite(loss[4:]).all()
    fine = torch.isfinite(want)
    assert ((loss[fine].double() - want[fine]).abs() <= 1e-4).all()
    dx, = torch.autograd.grad(loss[[0, 1, 2, 4]].sum(), x)
    assert torch.isfinite(dx).all()


@pytest.mark.parametrize("T", [1e-4, 0.05, 30.0, 1e4])
def test_distillation_temperatures(T):
    x, w, b, logits, classes = make_distill(50, 32, 90, 6, torch.float32)
    loss = losses.linear_distillation(x, w, b, logits, classes, temperature=T)
    ref = leaves64(x, w, b)
    want = distill64(*ref, logits, classes, T)
    assert abs(float(loss) - float(want)) <= loss_limit(x, w, b, logits, T)
    # softmax of logits / T moves by what its logits do, 1e-6 of them over T, at the most by all
    got, target = torch.autograd.grad(loss, [x, w, b]), torch.autograd.grad(want, ref)
    for g, r in zip(got, target):
        assert float((g.double() - r).norm()) <= min(1.0, 1e-5 + 4e-6 * 20 / T) * float(r.norm()) + 1e-6 * T


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("T", [1e-4, 1e-3, 0.05, 1.0, 8.0])
def test_distillation_of_exact_logits_at_all_temperatures(T, dtype, reduction):
    """Logits that fp32 holds exactly, some 64 and within a few T of each other: no error of theirs is there to be divided by T, and
    the limits are the same at every T.

    x and w are whole numbers up to 3 times powers of two, the bias is 64, and a unit of the logits is from T / 16 to T / 8, 2^-17 or more, which numbers
    of 64 to 128 have for a step or a multiple of it.  Logits of 32 products are some 23 units apart, 3 T, seldom 20 T: what is d T below the
    largest has an exponent that is d 2^-23 off, of its q of e^-d at most 1e-7; sums of 50 and logarithms of up to 4 are 2^-22 off.  So a loss is within (20
    2^-23 + 2^-22 + as much for the teacher's) T^2 < 1e-5 T^2, and gradients, differences of p and q, within 1e-5 of their norm, and half a step more
    where they are rounded to 16 bits (held in two halves before)."""
    rows, C, V, k = 40, 32, 50, 6
    gen = torch.Generator("cuda").manual_seed(7)
    unit = 2.0 ** (math.floor(math.log2(T)) - 3)
    shares = 2.0 ** (math.floor(math.log2(unit)) // 2)

    def whole(*shape):
        return torch.randint(-3, 4, shape, generator=gen, device="cuda").float()

    x, w = (whole(rows, C) * shares).to(dtype).requires_grad_(), (whole(V, C) * (unit / shares)).to(dtype).requires_grad_()
    b = torch.full((V,), 64.0, device="cuda", dtype=dtype).requires_grad_()
    ref = leaves64(x, w, b)
    own = F.linear(*ref)
    assert torch.equal(own.detach().float().double(), own.detach()) and torch.equal(F.linear(ref[0], ref[1]).detach() / unit % 1, torch.zeros_like(own))
    classes = torch.rand(rows, V, generator=gen, device="cuda").argsort(1)[:, :k]
    logits = whole(rows, k) * T
    loss = losses.linear_distillation(x, w, b, logits, classes, temperature=T, reduction=reduction)
    want = distill64(*ref, logits, classes, T, reduction)
    assert ((loss.double() - want).abs() <= 1e-5 * T * T + 2.0 ** -23 * want.abs()).all()
    # (gradients of size 1 in fp16 as well)
    up = torch.full_like(loss, 1.0 / T)
    got = torch.autograd.grad(loss, [x, w, b], up)
    r = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    for g, t, name in zip(got, torch.autograd.grad(want, ref, up.double()), ["dx", "dw", "db"]):
        floor = 2.0 ** -25 * math.sqrt(t.numel()) if dtype == torch.float16 else 0.0
        off = float((g.double() - t).norm())
        assert off <= (r + 1e-5) * float(t.norm()) + floor, "%s: %.3g of its norm" % (name, off / float(t.norm()))


def test_distillation_types_and_autocast():
    x, w, b, logits, classes = make_distill(66, 64, 144, 7, torch.float32)
    for other in DTYPES:
        t = logits.to(other)
        got = losses.linear_distillation(x, w, b, t, classes)
        assert torch.equal(got, losses.linear_distillation(x, w, b, t.float(), classes))
    # parameters of another type: gradients of their own
    x16 = x.detach().bfloat16().requires_grad_()
    loss = losses.linear_distillation(x16, w, b, logits, classes)
    grads = torch.autograd.grad(loss, [x16, w, b])
    assert [g.dtype for g in grads] == [torch.bfloat16, torch.float32, torch.float32]
    ref = leaves64(x16, w.detach().bfloat16(), b.detach().bfloat16())
    for g, r in zip(grads, torch.autograd.grad(distill64(*ref, logits, classes, 1.0), ref)):
        near(g, r, "gradient", rounding=2.0 ** -8)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        auto = losses.linear_distillation(x, w, b, logits, classes)
    assert auto.dtype == torch.float32 and torch.equal(auto, loss)
    assert [g.dtype for g in torch.autograd.grad(auto, [x, w, b])] == [torch.float32] * 3
    # leading dimensions, strides, none
    want = losses.linear_distillation(x, w, b, logits, classes, reduction="none")
    shaped = losses.linear_distillation(x.view(6, 11, 64), w, b, logits.view(6, 11, 7), classes.view(6, 11, 7), reduction="none")
    assert torch.equal(shaped.flatten(), want)
    one = losses.linear_distillation(x[4], w, b, logits[4], classes[4], reduction="none")
    assert one.shape == () and abs(float(one) - float(want[4])) <= 1e-5
    strided = losses.linear_distillation(x.t().contiguous().t(), w.t().contiguous().t(), b, logits.t().contiguous().t(), classes.t().contiguous().t(),
                                         reduction="none")
    assert torch.equal(strided, want)
    empty = losses.linear_distillation(x[:0], w, b, logits[:0], classes[:0])
    assert empty.isnan() and (torch.autograd.grad(empty, w)[0] == 0).all()


def test_distillation_differences():
    """The gradient against differences of the loss: (f(x + h d) - f(x - h d)) / 2 h is off by the third derivative, about h^2, and by what fp32 leaves
    of the two losses of about 5, 2e-6 each, over h: 1e-3 for h = 1e-2."""
    x, w, b, logits, classes = make_distill(20, 24, 40, 6, torch.float32, absent=True, seed=5)
    args = [x, w, b]
    got = torch.autograd.grad(losses.linear_distillation(*args, logits, classes, temperature=2.0), args)
    h = 1e-2
    for i, g in enumerate(got):
        d = torch.randn_like(args[i])
        d /= d.norm()
        with torch.no_grad():
            moved = [losses.linear_distillation(*[t + s * h * d if j == i else t for j, t in enumerate(args)], logits, classes, temperature=2.0)
                     for s in (1, -1)]
        slope = (float(moved[0]) - float(moved[1])) / (2 * h)
        assert abs(slope - float((g * d).sum())) <= 2e-3, i


def test_distillation_gradients_of_some_inputs():
    x, w, b, logits, classes = make_distill(70, 48, 90, 6, torch.float32)
    ref = leaves64(x, w, b)
    want = torch.autograd.grad(distill64(*ref, logits, classes, 1.0), ref)
    for wanted in ([0], [1], [2], [0, 1], [1, 2], [0, 2]):
        some = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        loss = losses.linear_distillation(*some, logits, classes)
        for g, i in zip(torch.autograd.grad(loss, [some[i] for i in wanted]), wanted):
            near(g, want[i], str(wanted))


def test_distillation_refusals():
    x, w, b, logits, classes = make_distill(6, 16, 48, 5, torch.float32)
    L = losses.linear_distillation
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(L(x, w, b, logits, classes), x, create_graph=True)
    with pytest.raises(RuntimeError, match="detach"):
        L(x, w, b, logits.clone().requires_grad_(), classes)
    for bad in (dict(teacher_logits=logits[:5]), dict(teacher_classes=classes.int()), dict(teacher_classes=classes[:, :4]),
                dict(teacher_logits=logits.double()), dict(teacher_logits=logits[:, :0], teacher_classes=classes[:, :0]),
                dict(teacher_logits=logits.cpu()), dict(weight=w.detach()[:, :8]), dict(bias=b.detach()[:5]),
                dict(teacher_logits=logits.repeat(1, 205), teacher_classes=classes.repeat(1, 205))):
        with pytest.raises(RuntimeError):
            L(**{**dict(x=x, weight=w, bias=b, teacher_logits=logits, teacher_classes=classes), **bad})


# ---------------------------------------------------------------------------------------------------- beyond 32 bits
def test_offsets_beyond_32_bits():
    """More than 2^32 bytes, and 2^31 values, in front of the last rows."""
    # top logits: rows by themselves, and short rows
    for V, k in ((65536, 64), (150, 8)):
        rows = (1 << 31) // V + 40
        x = torch.zeros(rows, V, device="cuda", dtype=torch.bfloat16)
        x[-30:] = values(30, V, dtype=torch.bfloat16)
        got = losses.top_logits(x, k)
        want = top64(x[-30:], k)
        assert torch.equal(got.classes[-30:].cpu(), want[1]) and same_values(got.values[-30:], want[0])
        assert torch.equal(got.classes[0].cpu(), torch.arange(k))
        del x, got
    # rows of codes, many short rows and others
    for C in (96, 1100):
        rows = (1 << 31) // C + 70
        x = torch.zeros(rows, C, device="cuda", dtype=torch.bfloat16)
        x[-50:] = values(50, C, dtype=torch.bfloat16)
        w = values(8, C)
        y = int8.linear_int8(x, int8.quantize_rows(w))
        assert not y[:-50].any()
        int8_near(y[-50:], *int8_64(x[-50:], w, None, None))
        del x, y
    rows = (1 << 31) // 40 + 100
    w = values(40, 96)
    x = torch.zeros(rows, 96, device="cuda", dtype=torch.bfloat16)
    x[-50:] = values(50, 96, dtype=torch.bfloat16)
    y = int8.linear_int8(x, int8.quantize_rows(w))
    int8_near(y[-50:], *int8_64(x[-50:], w, None, None))
    del x, y
    # distillation: entries, and logits' gradients in pieces
    rows, C, V, k = (1 << 31) // 128 + 60, 8, 16, 128
    x, w, b = values(rows, C, dtype=torch.bfloat16).requires_grad_(), values(V, C, dtype=torch.bfloat16), values(V, dtype=torch.bfloat16)
    logits, classes = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16), torch.full((rows, k), -1, device="cuda")
    logits[-40:], classes[-40:] = values(40, k, dtype=torch.bfloat16), torch.randint(0, V, (40, k), device="cuda")
    loss = losses.linear_distillation(x, w, b, logits, classes, reduction="none")
    dx, = torch.autograd.grad(loss.sum(), x)
    ref = x[-40:].detach().double().requires_grad_()
    want = distill64(ref, w.double(), b.double(), logits[-40:], classes[-40:], 1.0, "none")
    assert not loss[:-40].any() and ((loss[-40:].double() - want).abs() <= 1e-4).all()
    near(dx[-40:], torch.autograd.grad(want.sum(), ref)[0], "dx")
    assert not dx[:-40].any()


# ---------------------------------------------------------------------------------------------------- together
def chain(x, held, b, w, bias, student):
    """A teacher's layer in 8 bits and its top logits, a student's loss, and its gradients."""
    with torch.no_grad():
        top = losses.top_logits(int8.linear_int8(x, held, b), 9)
    loss = losses.linear_distillation(student, w, bias, *top, temperature=2.0)
    return [*top, loss, *torch.autograd.grad(loss, [student, w, bias])]


def make_chain(rows, dtype, seed=0):
    x, held, b = values(rows, 96, dtype=dtype, seed=seed), int8.quantize_rows(values(130, 96, dtype=dtype, std=0.2)), values(130, dtype=dtype)
    w, bias = values(130, 48, dtype=dtype, std=0.2).requires_grad_(), values(130, dtype=dtype).requires_grad_()
    return x, held, b, w, bias, values(rows, 48, dtype=dtype, seed=seed + 1).requires_grad_()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_together_streams_and_graphs(dtype):
    args = make_chain(200, dtype)
    want = [t.detach().clone() for t in chain(*args)]
    for got, t in zip(chain(*args), want):
        assert torch.equal(got, t)
    # against the formulas, in their order
    y, size = int8_64(args[0], values(130, 96, dtype=dtype, std=0.2), args[2], None)
    z = int8.linear_int8(*args[:3])
    int8_near(z, y, size)
    v, c = top64(z, 9)
    assert torch.equal(want[1].cpu(), c) and same_values(want[0], v)
    ref = leaves64(args[5], args[3], args[4])
    loss = distill64(*ref, want[0], want[1], 2.0)
    assert abs(float(want[2]) - float(loss)) <= loss_limit(args[5], args[3], args[4], want[0], 2.0)
    for g, r in zip(want[3:], torch.autograd.grad(loss, ref)):
        near(g, r, "gradient")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = chain(*args)
    torch.cuda.current_stream().wait_stream(side)
    for got, t in zip(again, want):
        assert torch.equal(got, t)
    del again, got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain(*args)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        for got, t in zip(captured, want):
            assert torch.equal(got, t)
        chain(*args)
        torch.randn(1 << 20, device="cuda").sum().item()
    args[0].copy_(args[0].roll(1, 0))
    fresh = [t.detach().clone() for t in chain(*args)]
    graph.replay()
    for got, t in zip(captured, fresh):
        assert torch.equal(got, t)


def test_together_two_graphs_and_two_streams():
    sets = [make_chain(150, torch.bfloat16, 1), make_chain(3, torch.bfloat16, 2)]
    want = [[t.detach().clone() for t in chain(*a)] for a in sets]
    graphs, held = [], []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(chain(*a))
        graphs.append(g)
    for order in ((0, 1), (1, 0), (0, 0, 1)):
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in set(order):
            for got, t in zip(held[k], want[k]):
                assert torch.equal(got, t)
    streams = [torch.cuda.Stream() for _ in sets]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(20):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = chain(*sets[k])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for g, t in zip(a, b):
            assert torch.equal(g, t)


def test_distillation_captured_beside_an_eager_graph_is_refused():
    x, w, b, logits, classes = make_distill(20, 32, 40, 5, torch.float32)
    eager = losses.linear_distillation(x, w, b, logits, classes)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(graph):
            loss = losses.linear_distillation(x, w, b, logits, classes)
            torch.autograd.grad(loss, x)
    del eager, loss
    torch.cuda.synchronize()
    assert torch.isfinite(torch.autograd.grad(losses.linear_distillation(x, w, b, logits, classes), x)[0]).all()


def test_distillation_recomputed_and_in_inference_mode():
    x, w, b, logits, classes = make_distill(60, 40, 90, 5, torch.float32)

    def f(*a):
        return losses.linear_distillation(*a, logits, classes)

    want = torch.autograd.grad(f(x, w, b), [x, w, b])
    got = torch.autograd.grad(torch.utils.checkpoint.checkpoint(f, x, w, b, use_reentrant=False), [x, w, b])
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    with torch.autograd.graph.save_on_cpu():
        y = f(x, w, b)
    for a, c in zip(torch.autograd.grad(y, [x, w, b]), want):
        assert torch.equal(a, c)
    with torch.inference_mode():
        assert torch.equal(f(x.detach(), w.detach(), b.detach()), y.detach())


def networks():
    torch.manual_seed(3)
    make = dict(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40), num_classes=50)
    return ConvNeXt1D(**make, layer_scale_init_value=0.5).cuda(), ConvNeXt1D(**make).cuda()


def test_a_network_learns_from_another():
    teacher, student = networks()
    images = torch.randn(4, 3, 64, 64, device="cuda")
    top = teacher.top_logits(images, 5)
    assert top.values.shape == (4, 5) and not top.values.requires_grad
    with torch.no_grad():
        assert torch.equal(top.classes, losses.top_logits(teacher(images), 5).classes)
    seen = []
    hook = student.register_forward_hook(lambda m, a, out: seen.append(out))
    loss = student.distill(images, top, temperature=2.0)
    hook.remove()
    assert len(seen) == 1
    learnt = [p for name, p in student.named_parameters() if not name.endswith("theta")]
    grads = torch.autograd.grad(loss, learnt)
    want = losses.distillation_of(student(images), *top, 2.0)
    assert abs(float(loss) - float(want)) <= 1e-4
    for g, r in zip(grads, torch.autograd.grad(want, learnt)):
        assert torch.isfinite(g).all() and float((g - r).norm()) <= 1e-3 * float(r.norm()) + 1e-6
    with pytest.raises(ValueError, match="not both"):
        student(images, torch.zeros(4, dtype=torch.long, device="cuda"), teacher=top)
    # a head with hooks composes the same
    hook = student.head.register_forward_hook(lambda m, a, out: None)
    assert abs(float(student.distill(images, top, temperature=2.0)) - float(want)) <= 1e-5
    hook.remove()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("variant", ["1d", "1dpp"])
def test_a_network_in_8_bits(variant, dtype):
    """Its layers are the formula's, and its logits near: each layer's codes are off by half a step of 1 / 127 of the row's largest at the most."""
    torch.manual_seed(4)
    net = ConvNeXt1D(depths=(1, 1, 1, 1), dims=(16, 24, 32, 40), num_classes=50, variant=variant, layer_scale_init_value=0.5).cuda().to(dtype).eval()
    images = torch.randn(3, 3, 64, 64, device="cuda", dtype=dtype)
    with torch.no_grad():
        want = net(images)
        block = net.stages[2][0]
        layer = block.pwconv1
        assert int8.quantize_network(net) is net
        assert isinstance(block.pwconv1, int8.LinearInt8) and isinstance(net.head, int8.LinearInt8)
        x = values(7, 32, dtype=dtype)
        int8_near(block.pwconv1(x, activation="gelu"), *int8_64(x, layer.weight, layer.bias, "gelu"))
        got = net(images)
        assert got.dtype == dtype and float((got - want).float().norm()) <= 0.1 * float(want.float().norm())
        state = net.state_dict()
        net.half()
        assert net.head.scales.dtype == torch.float32 and net.head.bias.dtype == torch.float16
        assert torch.equal(net.head.scales, state["head.scales"])
        net.to(dtype).train()
        assert torch.isfinite(net(images)).all()
    with pytest.raises(RuntimeError, match="no gradients"):
        net(images)
