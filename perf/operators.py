"""The operators around a network's wide layers, as measurable cases: what each computes, in a plain form and through the framework.

Four operators of training and evaluation:

* ``gated``: a gated feed-forward block, ``(act(x Wg^T + bg) * (x Wu^T + bu)) Wo^T + bo``: forward only, or a training pass
  (result and the gradients of input, weights and biases).  With ``bits8`` the training pass keeps nothing but its input in 8 bits.
* ``head``: softmax cross entropy of a linear layer over many classes, without keeping the logits: the losses, or a training pass.
* ``linear8``: a linear layer whose backward pass reads its input from an 8-bit checkpoint.
* ``act8``: an activation whose backward pass reads its input from an 8-bit checkpoint.

An 8-bit checkpoint holds, for every 32 neighbours along the last dimension, whole numbers q in [-127, 127] and a power of two s, and
stands for q * s: s = 2^(floor(log2(largest magnitude)) - 6), at least 2^-126, and q = round(x / s), ties to even.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_IGNORED = -100


def _gated(rows, C, H, D, dtype, act="gelu", bias=True, train=True, bits8=False):
    return {"kind": "gated", "rows": rows, "C": C, "H": H, "D": D, "dtype": dtype, "act": act, "bias": bias, "train": train,
            "bits8": bits8}


def _head(rows, C, V, dtype, smoothing=0.0, ignored=0.0, reduction="mean", bias=True, train=True):
    return {"kind": "head", "rows": rows, "C": C, "V": V, "dtype": dtype, "smoothing": smoothing, "ignored": ignored,
            "reduction": reduction, "bias": bias, "train": train}


def _linear8(rows, C, D, dtype, bias=True):
    return {"kind": "linear8", "rows": rows, "C": C, "D": D, "dtype": dtype, "bias": bias}


def _act8(rows, C, dtype, act="gelu"):
    return {"kind": "act8", "rows": rows, "C": C, "dtype": dtype, "act": act}


def listed():
    cases = {
        # one row at inference: reading the weights and two launches
        "gated_one_row": _gated(1, 1024, 4096, 1024, "bf16", train=False),
        # the smallest training pass, one 7 x 7 image of 96 channels in fp32: latency
        "gated_small_f32": _gated(49, 96, 256, 96, "f32", act="silu"),
        # a batch of 64 images at 7 x 7 that keeps 8 bits of its input alone
        "gated_8bits_f16": _gated(3136, 768, 2048, 768, "f16", bits8=True),
        # a large training pass in bf16
        "gated_large": _gated(16384, 1024, 4096, 1024, "bf16"),
        # the classifier of a training step: 64 images, 1000 classes, label smoothing
        "head_small": _head(64, 768, 1000, "bf16", smoothing=0.1),
        # dense prediction: pixels of eight maps of 64 x 64, 150 classes, pixels without a label
        "head_pixels_f16": _head(32768, 256, 150, "f16", ignored=0.2),
        # a class for every label of a large image collection, in fp32; the number of classes is odd
        "head_wide_f32": _head(1024, 512, 21841, "f32"),
        # a large vocabulary at a large batch
        "head_large": _head(8192, 1024, 65536, "bf16"),
        # the first pointwise layer of a stage of 384 channels, 128 images of 14 x 14
        "linear8_large": _linear8(25088, 384, 1536, "bf16"),
        # a small layer of sizes that nothing divides
        "linear8_small_f32": _linear8(301, 100, 61, "f32"),
        # the activation behind that layer
        "act8_large": _act8(25088, 1536, "bf16"),
        # a few rows with a partial group
        "act8_small_f32": _act8(49, 333, "f32", act="silu"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of eight, as networks have them; one in four is any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def _drawn(rng):
    kind = rng.choice(["gated", "gated", "head", "head", "linear8", "act8"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    act, bias = rng.choice(["gelu", "silu"]), rng.random() < 0.8
    if kind == "gated":
        train = rng.random() < 0.7
        C = _width(rng, 32, 1024)
        return _gated(_log(rng, 1, 16384), C, _width(rng, 64, 4096), C if rng.random() < 0.7 else _width(rng, 32, 1024), dtype, act,
                      bias, train, train and rng.random() < 0.4)
    if kind == "head":
        return _head(_log(rng, 1, 32768), _width(rng, 32, 1024), _log(rng, 10, 65536), dtype, rng.choice([0.0, 0.0, 0.1]),
                     rng.choice([0.0, 0.0, 0.3]), rng.choice(["mean", "mean", "none"]), bias, rng.random() < 0.7)
    if kind == "linear8":
        return _linear8(_log(rng, 1, 32768), _width(rng, 32, 2048), _width(rng, 32, 2048), dtype, bias)
    return _act8(_log(rng, 1, 32768), _width(rng, 16, 4096), dtype, act)


def draw(rng):
    most = max(work(c)["flops"] for c in listed())
    while True:
        case = _drawn(rng)
        # (a product in fp32 costs several times the same product of 16-bit values)
        if work(case)["flops"] * (4 if case["dtype"] == "f32" else 1) <= most:
            return case


def work(case):
    M, C, size = case["rows"], case["C"], _DTYPES[case["dtype"]].itemsize
    if case["kind"] == "gated":
        H, D = case["H"], case["D"]
        weights = 2 * H * C + D * H + ((2 * H + D) if case["bias"] else 0)
        once = 4 * M * C * H + 2 * M * H * D
        if not case["train"]:
            return {"bytes": size * (M * (C + D) + weights), "flops": once}
        # x, dy, weights in; y, dx and the weights' gradients out; without the hidden tensors the first products are made twice
        return {"bytes": size * (2 * M * (C + D) + 2 * weights), "flops": 3 * once + (4 * M * C * H if case["bits8"] else 0)}
    if case["kind"] == "head":
        V = case["V"]
        weights = V * C + (V if case["bias"] else 0)
        ends = 8 * M + 4 * (M if case["reduction"] == "none" else 1)
        if not case["train"]:
            return {"bytes": size * (M * C + weights) + ends, "flops": 2 * M * C * V}
        return {"bytes": 2 * size * (M * C + weights) + ends, "flops": 6 * M * C * V}
    held = M * (C + -(-C // 32))
    if case["kind"] == "linear8":
        D = case["D"]
        weights = D * C + (D if case["bias"] else 0)
        return {"bytes": size * (2 * M * (C + D) + 2 * weights) + 2 * held, "flops": 6 * M * C * D}
    return {"bytes": size * 4 * M * C + 2 * held, "flops": 40 * M * C}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, M, C = _DTYPES[case["dtype"]], case["rows"], case["C"]

    def values(*shape, std=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    state = dict(case)
    if case["kind"] == "act8":
        # a pre-activation: groups of different magnitudes
        x = values(M, C) * torch.exp(0.5 * torch.randn((M, 1), generator=gen, device="cuda")).to(dtype)
        leaves = [x]
        state["dy"] = values(M, C)
    elif case["kind"] == "linear8":
        D = case["D"]
        leaves = [values(M, C), values(D, C, std=C ** -0.5)] + ([values(D, std=0.1)] if case["bias"] else [])
        state["dy"] = values(M, D)
    elif case["kind"] == "gated":
        H, D = case["H"], case["D"]
        leaves = [values(M, C), values(2 * H, C, std=1.5 * C ** -0.5), values(D, H, std=H ** -0.5)]
        leaves += [values(2 * H, std=0.1), values(D, std=0.1)] if case["bias"] else []
        state["dy"] = values(M, D)
    else:
        V = case["V"]
        leaves = [values(M, C), values(V, C, std=2.0 * C ** -0.5)] + ([values(V, std=0.1)] if case["bias"] else [])
        target = torch.randint(0, V, (M,), generator=gen, device="cuda")
        if case["ignored"] > 0 and M > 1:
            off = torch.rand((M,), generator=gen, device="cuda") < case["ignored"]
            off[0] = False
            target = torch.where(off, _IGNORED, target)
        state["target"] = target
        # what arrives at the loss in a backward pass; a mean in fp16 is trained with a scaled loss
        shape = (M,) if case["reduction"] == "none" else ()
        scale = 4096.0 if case["dtype"] == "f16" and not shape else 1.0
        state["dy"] = (torch.rand(shape, generator=gen, device="cuda") + 0.5) * scale
    train = case.get("train", True)
    state["leaves"] = [t.requires_grad_(train) for t in leaves]
    return state


# ---------------------------------------------------------------------------------------------- through the framework


def _own(s):
    from oriented1d_amd import checkpoint8, feedforward, losses

    leaves, kind = s["leaves"], s["kind"]
    if kind == "gated":
        x, w_in, w_out, b_in, b_out = leaves if s["bias"] else (*leaves, None, None)
        out = feedforward.gated_mlp(x, w_in, b_in, w_out, b_out, activation=s["act"], checkpoint8=s["bits8"])
    elif kind == "head":
        x, w, b = leaves if s["bias"] else (*leaves, None)
        out = losses.linear_cross_entropy(x, w, b, s["target"], reduction=s["reduction"], ignore_index=_IGNORED,
                                          label_smoothing=s["smoothing"])
    elif kind == "linear8":
        x, w, b = leaves if s["bias"] else (*leaves, None)
        out = checkpoint8.linear8(x, w, b)
    else:
        out = checkpoint8.act8(leaves[0], activation=s["act"])
    if not s.get("train", True):
        return [out]
    return [out, *torch.autograd.grad(out, leaves, s["dy"])]


# ---------------------------------------------------------------------------------------------- the plain form


def _held8(x):
    """The values that an 8-bit checkpoint of x stands for, in 32 bits."""
    M, C = x.shape
    groups = -(-C // 32)
    v = torch.zeros((M, groups * 32), dtype=torch.float32, device=x.device)
    v[:, :C] = x.float()
    v = v.reshape(M, groups, 32)
    most = v.abs().amax(-1, keepdim=True)
    # the exponent's own bits are floor(log2), exactly
    e = ((most.view(torch.int32) >> 23) - 127 - 6).clamp(min=-126)
    s = ((e + 127) << 23).view(torch.float32)
    q = torch.round(v / s).clamp(-127, 127)
    return (q * s).reshape(M, groups * 32)[:, :C]


def _act(g, name):
    """The activation of g and its derivative."""
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-g))
        return g * p, p * (1.0 + g * (1.0 - p))
    p = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
    return g * p, p + g * torch.exp(-0.5 * g * g) * (0.5 / math.pi) ** 0.5


def _plain_gated(s):
    x, w_in, w_out, *biases = s["leaves"]
    dtype, H = x.dtype, s["H"]
    wi, wo = w_in.float(), w_out.float()
    bi, bo = (b.float() for b in biases) if biases else (0.0, 0.0)

    def hidden(rows):
        a = rows @ wi.t() + bi
        return a[:, :H], a[:, H:]

    rows = x.float()
    g, u = hidden(rows)
    a, da = _act(g, s["act"])
    y = ((a * u) @ wo.t() + bo).to(dtype)
    if not s["train"]:
        return [y]
    if s["bits8"]:
        rows = _held8(x)
        g, u = hidden(rows)
        a, da = _act(g, s["act"])
    dy = s["dy"].float()
    dh = dy @ wo
    da = torch.cat([dh * u * da, dh * a], 1)
    grads = [da @ wi, da.t() @ rows, dy.t() @ (a * u)] + ([da.sum(0), dy.sum(0)] if biases else [])
    return [y] + [t.to(dtype) for t in grads]


def _plain_head(s):
    x, w, *bias = s["leaves"]
    dtype, eps, V, target = x.dtype, s["smoothing"], s["V"], s["target"]
    rows, wf = x.float(), w.float()
    logits = rows @ wf.t()
    if bias:
        logits = logits + bias[0].float()
    valid = target != _IGNORED
    at = torch.where(valid, target, 0)[:, None]
    most = logits.amax(1, keepdim=True)
    e = torch.exp(logits - most)
    total = e.sum(1, keepdim=True)
    lse = most + torch.log(total)
    loss = (1.0 - eps) * (lse - logits.gather(1, at)) + eps * (lse - logits.mean(1, keepdim=True))
    loss = torch.where(valid, loss[:, 0], 0.0)
    count = valid.sum()
    out = loss if s["reduction"] == "none" else loss.sum() / count
    if not s["train"]:
        return [out]
    up = torch.where(valid, s["dy"] if s["reduction"] == "none" else s["dy"] / count, 0.0)
    del logits
    g = e / total - eps / V
    g.scatter_add_(1, at, torch.full_like(total, eps - 1.0))
    g = g * up[:, None]
    grads = [g @ wf, g.t() @ rows] + ([g.sum(0)] if bias else [])
    return [out] + [t.to(dtype) for t in grads]


def _plain_linear8(s):
    x, w, *bias = s["leaves"]
    dtype, wf, dy = x.dtype, w.float(), s["dy"].float()
    y = x.float() @ wf.t()
    if bias:
        y = y + bias[0].float()
    grads = [dy @ wf, dy.t() @ _held8(x)] + ([dy.sum(0)] if bias else [])
    return [y.to(dtype)] + [t.to(dtype) for t in grads]


def _plain_act8(s):
    x = s["leaves"][0]
    return [_act(x.float(), s["act"])[0].to(x.dtype), (s["dy"].float() * _act(_held8(x), s["act"])[1]).to(x.dtype)]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"gated": _plain_gated, "head": _plain_head, "linear8": _plain_linear8, "act8": _plain_act8}[state["kind"]](state)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits


def _exact8(x):
    """The values that an 8-bit checkpoint of x (64 bits) stands for, with exponents by frexp."""
    C = x.shape[1]
    groups = torch.nn.functional.pad(x, (0, -C % 32)).unflatten(1, (-1, 32))
    exponent = torch.frexp(torch.linalg.vector_norm(groups, ord=math.inf, dim=2, keepdim=True))[1] - 7
    # (the power of two by its bits: torch.ldexp goes through pow, which is not exact)
    step = ((exponent.clamp(min=-126).long() + 1023) << 52).view(torch.float64)
    return (torch.round(groups / step).clamp(-127, 127) * step).flatten(1)[:, :C]


def exact(case, seed):
    F = torch.nn.functional
    s = prepare(case, seed)
    leaves = [t.detach().double().requires_grad_(case.get("train", True)) for t in s["leaves"]]
    activation = {"gelu": F.gelu, "silu": F.silu}[case.get("act", "gelu")]
    dy = s["dy"].double()

    def value(x, *parameters):
        if case["kind"] == "act8":
            return activation(x)
        if case["kind"] == "linear8":
            return F.linear(x, *parameters)
        if case["kind"] == "head":
            return F.cross_entropy(F.linear(x, *parameters), s["target"], ignore_index=_IGNORED, reduction=case["reduction"],
                                   label_smoothing=case["smoothing"])
        w_in, w_out, b_in, b_out = parameters if case["bias"] else (*parameters, None, None)
        gate, up = F.linear(x, w_in, b_in).chunk(2, dim=1)
        return F.linear(activation(gate) * up, w_out, b_out)

    out = value(*leaves)
    if not case.get("train", True):
        return [out]
    result = out.detach()
    if case["kind"] == "linear8":
        # (the gradient of the input needs no input)
        dx, = torch.autograd.grad(out, leaves[:1], dy)
        held = _exact8(leaves[0].detach()).requires_grad_()
        return [result, dx, *torch.autograd.grad(value(held, *leaves[1:]), leaves[1:], dy)]
    if case["kind"] == "act8" or case.get("bits8"):
        held = _exact8(leaves[0].detach()).requires_grad_()
        return [result, *torch.autograd.grad(value(held, *leaves[1:]), [held, *leaves[1:]], dy)]
    return [result, *torch.autograd.grad(out, leaves, dy)]
