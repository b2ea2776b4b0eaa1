"""The operators between a teacher and its student, as measurable cases: what each computes, in a plain form and through the framework.

Three operators:

* ``int8``: a linear layer at inference as a product of 8-bit integers.  A row of x with largest magnitude a stands as whole numbers
  q = round(127 x / a), ties to even, times a / 127; the weight's rows are held so already, codes and scales.  The result is
  ``act(sums * (a / 127) * scales + bias)``.
* ``top``: the k largest logits of each row and their classes, largest first, of equal ones the lowest class first.
* ``distill``: a linear classifier's loss against a teacher's top logits: with p the softmax over the row's entries of t / T and q that of the
  classifier's own logits over all classes, l / T, it is T^2 * sum_j p_j (log p_j - log q_j).  Entries of class -1 are absent; rows without
  entries are 0 and do not count in the mean.  The loss alone, or a training pass.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _int8(rows, C, D, dtype, act="none", bias=True):
    return {"kind": "int8", "rows": rows, "C": C, "D": D, "dtype": dtype, "act": act, "bias": bias}


def _top(rows, V, k, dtype):
    return {"kind": "top", "rows": rows, "V": V, "k": k, "dtype": dtype}


def _distill(rows, C, V, k, dtype, T=1.0, absent=0.0, reduction="mean", bias=True, train=True):
    return {"kind": "distill", "rows": rows, "C": C, "V": V, "k": k, "dtype": dtype, "T": T, "absent": absent, "reduction": reduction,
            "bias": bias, "train": train}


def listed():
    cases = {
        # one row at inference: reading the codes and as few launches as can be
        "int8_one_row": _int8(1, 1024, 4096, "bf16", act="gelu"),
        # a small layer of sizes that nothing divides, in fp32
        "int8_small_f32": _int8(37, 333, 61, "f32"),
        # the first pointwise layer and activation of a stage of 384 channels, 128 images of 14 x 14
        "int8_stage": _int8(25088, 384, 1536, "bf16", act="gelu"),
        # a wide layer at a large batch
        "int8_large": _int8(16384, 4096, 4096, "f16"),
        # one row of a large vocabulary: latency
        "top_one_row_f32": _top(1, 65536, 64, "f32"),
        # dense prediction: pixels of eight maps of 64 x 64, 150 classes
        "top_pixels_f16": _top(32768, 150, 8, "f16"),
        # a teacher's batch over a large vocabulary
        "top_large": _top(8192, 65536, 64, "bf16"),
        # the classifier of a training step: 64 images, 1000 classes
        "distill_small": _distill(64, 768, 1000, 16, "bf16", T=2.0),
        # dense prediction, pixels without a label and with fewer entries than others
        "distill_pixels_f16": _distill(32768, 256, 150, 8, "f16", absent=0.2),
        # a class for every label of a large image collection, in fp32; the number of classes is odd
        "distill_wide_f32": _distill(1024, 512, 21841, 100, "f32", T=4.0),
        # a large vocabulary at a large batch
        "distill_large": _distill(8192, 1024, 65536, 64, "bf16"),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Mostly multiples of eight, as networks have them; one in four is any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def _drawn(rng):
    kind = rng.choice(["int8", "int8", "top", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "int8":
        return _int8(_log(rng, 1, 32768), _width(rng, 32, 4096), _width(rng, 32, 8192), dtype, rng.choice(["none", "gelu", "silu"]),
                     rng.random() < 0.8)
    if kind == "top":
        V = _log(rng, 10, 131072)
        return _top(_log(rng, 1, 32768), V, _log(rng, 1, min(V, 256)), dtype)
    V = _log(rng, 10, 65536)
    return _distill(_log(rng, 1, 32768), _width(rng, 32, 1024), V, _log(rng, 1, min(V, 128)), dtype, rng.choice([1.0, 1.0, 2.0, 4.0]),
                    rng.choice([0.0, 0.0, 0.3]), rng.choice(["mean", "mean", "none"]), rng.random() < 0.8, rng.random() < 0.7)


def draw(rng):
    most = {kind: max(work(c)["flops"] for c in listed() if c["kind"] == kind) for kind in ("int8", "top", "distill")}
    while True:
        case = _drawn(rng)
        # (a product in fp32 costs several times the same product of 16-bit values)
        if work(case)["flops"] * (4 if case["dtype"] == "f32" and case["kind"] == "distill" else 1) <= most[case["kind"]]:
            return case


def work(case):
    M, size = case["rows"], _DTYPES[case["dtype"]].itemsize
    if case["kind"] == "int8":
        C, D = case["C"], case["D"]
        weights = D * C + 4 * D + (size * D if case["bias"] else 0)
        return {"bytes": size * M * (C + D) + weights, "flops": 2 * M * C * D}
    if case["kind"] == "top":
        # (a comparison for each value)
        return {"bytes": size * M * case["V"] + M * case["k"] * (size + 8), "flops": M * case["V"]}
    C, V = case["C"], case["V"]
    weights = V * C + (V if case["bias"] else 0)
    ends = M * case["k"] * (size + 8) + 4 * (M if case["reduction"] == "none" else 1)
    if not case["train"]:
        return {"bytes": size * (M * C + weights) + ends, "flops": 2 * M * C * V}
    return {"bytes": 2 * size * (M * C + weights) + ends, "flops": 6 * M * C * V}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, M = _DTYPES[case["dtype"]], case["rows"]

    def values(*shape, std=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    state = dict(case)
    if case["kind"] == "top":
        # a classifier's logits: a few classes of each row stand out
        logits = torch.randn((M, case["V"]), generator=gen, device="cuda")
        logits += torch.relu(logits - 1.5) * 2.0
        state["logits"] = (logits * 2.0).to(dtype)
        return state
    C = case["C"]
    if case["kind"] == "int8":
        D = case["D"]
        # rows of different magnitudes, as layers leave them
        state["x"] = values(M, C) * torch.exp(0.5 * torch.randn((M, 1), generator=gen, device="cuda")).to(dtype)
        w = torch.randn((D, C), generator=gen, device="cuda") * C ** -0.5
        most = w.abs().amax(1)
        codes = torch.round(w.double() * 127.0 / most.double()[:, None]).to(torch.int8)
        # as the framework holds a weight: rows filled up with zeros to whole 16 bytes, and what a code's step stands for
        state["codes"] = torch.nn.functional.pad(codes, (0, -C % 16)).contiguous()
        state["scales"] = (most.double() / 127.0).float()
        state["b"] = values(D, std=0.1) if case["bias"] else None
        return state
    V, k = case["V"], case["k"]
    leaves = [values(M, C), values(V, C, std=2.0 * C ** -0.5)] + ([values(V, std=0.1)] if case["bias"] else [])
    # the teacher's largest first, each class once in a row
    state["teacher"] = torch.sort((torch.rand((M, k), generator=gen, device="cuda") * 8.0 + 4.0).to(dtype), dim=1, descending=True)[0]
    gaps = torch.randint(1, V // k + 1, (M, k), generator=gen, device="cuda")
    classes = (torch.randint(0, V, (M, 1), generator=gen, device="cuda") + gaps.cumsum(1)) % V
    classes = classes.gather(1, torch.rand((M, k), generator=gen, device="cuda").argsort(1))
    if case["absent"] > 0 and M > 1:
        there = torch.randint(1, k + 1, (M, 1), generator=gen, device="cuda")
        off = torch.rand((M, 1), generator=gen, device="cuda") < case["absent"]
        off[0] = False
        there = torch.where(off, 0, there)
        classes = torch.where(torch.arange(k, device="cuda") < there, classes, -1)
    state["classes"] = classes
    # what arrives at the loss in a backward pass; a mean in fp16 is trained with a scaled loss
    shape = (M,) if case["reduction"] == "none" else ()
    scale = 4096.0 if case["dtype"] == "f16" and not shape else 1.0
    state["dy"] = (torch.rand(shape, generator=gen, device="cuda") + 0.5) * scale
    state["leaves"] = [t.requires_grad_(case["train"]) for t in leaves]
    return state


# ---------------------------------------------------------------------------------------------- through the framework


def _own(s):
    from oriented1d_amd import int8, losses

    if s["kind"] == "int8":
        return [int8.linear_int8(s["x"], int8.QuantizedRows(s["codes"], s["scales"]), s["b"], activation=None if s["act"] == "none" else s["act"])]
    if s["kind"] == "top":
        return list(losses.top_logits(s["logits"], s["k"]))
    x, w, b = s["leaves"] if s["bias"] else (*s["leaves"], None)
    out = losses.linear_distillation(x, w, b, s["teacher"], s["classes"], temperature=s["T"], reduction=s["reduction"])
    if not s["train"]:
        return [out]
    return [out, *torch.autograd.grad(out, s["leaves"], s["dy"])]


# ---------------------------------------------------------------------------------------------- the plain form


def _plain_int8(s):
    x, C = s["x"], s["C"]
    most = x.abs().amax(1, keepdim=True).float()
    # (64 bits: a quotient next to the middle of two whole numbers)
    q = torch.round(x.double() * 127.0 / most.double()).float()
    q = torch.where(most > 0, q, 0.0)
    y = (q @ s["codes"][:, :C].float().t()) * (most / 127.0) * s["scales"]
    if s["b"] is not None:
        y = y + s["b"].float()
    if s["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif s["act"] == "gelu":
        y = y * 0.5 * (1.0 + torch.erf(y * 0.5 ** 0.5))
    return [y.to(x.dtype)]


def _plain_top(s):
    x = s["logits"]
    # whole numbers in the logits' order (their bits, of negative ones turned round; a zero is a zero), of equal ones the lower class above
    bits = (x.float() + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = order * (1 << 32) + ((1 << 31) - torch.arange(s["V"], device=x.device))
    classes = (1 << 31) - (torch.topk(key, s["k"], dim=1)[0] & 0xFFFFFFFF)
    return [x.gather(1, classes), classes]


def _plain_distill(s):
    x, w, *bias = s["leaves"]
    dtype, T, classes = x.dtype, s["T"], s["classes"]
    there = classes >= 0
    at = torch.where(there, classes, 0)
    counts = there.any(1, keepdim=True)
    # the teacher's distribution over the entries that are there
    t = torch.where(there, s["teacher"].float() / T, -math.inf)
    most = torch.where(counts, t.amax(1, keepdim=True), 0.0)
    e = torch.exp(t - most)
    total = torch.where(counts, e.sum(1, keepdim=True), 1.0)
    p = e / total
    log_p = torch.where(there, t - most - torch.log(total), 0.0)
    rows, wf = x.float(), w.float()
    logits = rows @ wf.t()
    if bias:
        logits = logits + bias[0].float()
    logits = logits / T
    most = logits.amax(1, keepdim=True)
    e = torch.exp(logits - most)
    total = e.sum(1, keepdim=True)
    log_q = logits.gather(1, at) - most - torch.log(total)
    loss = T * T * (p * (log_p - log_q)).sum(1)
    counts = counts[:, 0]
    loss = torch.where(counts, loss, 0.0)
    number = counts.sum()
    out = loss if s["reduction"] == "none" else loss.sum() / number
    if not s["train"]:
        return [out]
    up = torch.where(counts, s["dy"] if s["reduction"] == "none" else s["dy"] / number, 0.0)
    del logits
    g = (e / total).scatter_add_(1, at, -p)
    g = g * (up * T)[:, None]
    grads = [g @ wf, g.t() @ rows] + ([g.sum(0)] if bias else [])
    return [out] + [t.to(dtype) for t in grads]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"int8": _plain_int8, "top": _plain_top, "distill": _plain_distill}[state["kind"]](state)


# ---------------------------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    F = torch.nn.functional
    s = prepare(case, seed)
    if case["kind"] == "top":
        values, classes = torch.sort(s["logits"], dim=1, descending=True, stable=True)
        return [values[:, :case["k"]].clone(), classes[:, :case["k"]].clone()]
    if case["kind"] == "int8":
        x = s["x"].double()
        a = torch.linalg.vector_norm(x, ord=math.inf, dim=1, keepdim=True)
        # whole steps, and what is left of them against half a step: whole numbers times a, all exact
        t = x.abs() * 127.0
        whole = torch.floor(t / a)
        rest = 2.0 * (t - whole * a)
        whole = torch.where((rest > a) | ((rest == a) & (whole % 2 == 1)), whole + 1.0, whole)
        held = torch.where(a > 0, torch.sign(x) * whole * a / 127.0, 0.0)
        weight = s["codes"][:, :case["C"]].double() * s["scales"].double()[:, None]
        y = F.linear(held, weight, None if s["b"] is None else s["b"].double())
        return [{"none": lambda v: v, "gelu": F.gelu, "silu": F.silu}[case["act"]](y)]
    leaves = [t.detach().double().requires_grad_(case["train"]) for t in s["leaves"]]
    T, there = case["T"], s["classes"] >= 0
    logs = F.log_softmax(F.linear(*leaves) / T, 1)
    teacher = torch.where(there, s["teacher"].double() / T, -1e300)
    p = torch.where(there, F.softmax(teacher, 1), 0.0)
    loss = T * T * (torch.xlogy(p, p).sum(1) - (p * logs.gather(1, s["classes"].clamp(min=0))).sum(1))
    counts = there.any(1)
    loss = torch.where(counts, loss, 0.0)
    out = loss if case["reduction"] == "none" else loss.sum() / counts.sum()
    if not case["train"]:
        return [out]
    return [out.detach(), *torch.autograd.grad(out, leaves, s["dy"].double())]
