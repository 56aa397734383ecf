"""Products over weights of 8 bits, as cases that can be timed and compared.

Three operators.  ``linear``: rows times a matrix of e4m3 numbers with one fp32 scale for each block of 128 x 128, the rows themselves
rounded to e4m3 with one scale for each run of 128 of a row.  ``mlp``: the gated feed-forward of such matrices, whose inner rows are
rounded the same way.  ``experts``: a whole mixture-of-experts layer (router, choice, the chosen experts' feed-forwards, their sum) for
the few tokens of a decoding step, over experts of bf16 numbers or of e4m3 numbers with block scales; its activations stay as they are.

A case is a dict of plain values.  Widths are those of the framework's Qwen3 configurations and of its benchmark's experts, or generic.
"""

import math
import os
import sys

import torch

own = False

DEV = "cuda"
BLOCK = 128
TOP = 448.0           # the largest e4m3 number
SMALLEST = 2.0**-100  # a run of smaller numbers is scaled as if this were its largest
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one decoding request: the fused q|k|v projection of the 4B configuration, where latency counts
        dict(name="linear_1x2560x6144", kind="linear", rows=1, width=2560, outputs=6144, bias=False, type="bf16"),
        # a decoding batch on its way out of the attention
        dict(name="linear_24x4096x2560", kind="linear", rows=24, width=4096, outputs=2560, bias=False, type="bf16"),
        # odd sizes, whose last blocks are cut, with a bias, in the type that models are checked in
        dict(name="linear_77x1000x333_fp32", kind="linear", rows=77, width=1000, outputs=333, bias=True, type="fp32"),
        # the last portion of a prompt: a ragged number of rows
        dict(name="linear_333x2560x9728", kind="linear", rows=333, width=2560, outputs=9728, bias=False, type="bf16"),
        # a whole prompt through a down projection
        dict(name="linear_4096x9728x2560", kind="linear", rows=4096, width=9728, outputs=2560, bias=False, type="bf16"),
        # the feed-forward of the 4B configuration: a decoding request, a batch of odd size, a prompt portion
        dict(name="mlp_1x2560x9728", kind="mlp", rows=1, width=2560, inner=9728, type="bf16"),
        dict(name="mlp_37x1000x1400", kind="mlp", rows=37, width=1000, inner=1400, type="bf16"),
        dict(name="mlp_2048x2560x9728", kind="mlp", rows=2048, width=2560, inner=9728, type="bf16"),
        # the benchmark's experts: one request in both weight types, a small batch, the largest step that counts as few tokens
        dict(name="experts_1_bf16", kind="experts", tokens=1, width=2048, inner=1408, experts=64, top=6, weights="bf16"),
        dict(name="experts_1_e4m3", kind="experts", tokens=1, width=2048, inner=1408, experts=64, top=6, weights="e4m3"),
        dict(name="experts_5_odd_e4m3", kind="experts", tokens=5, width=1096, inner=712, experts=20, top=3, weights="e4m3"),
        dict(name="experts_32_e4m3", kind="experts", tokens=32, width=2048, inner=1408, experts=64, top=6, weights="e4m3"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("linear", "mlp", "experts"))
    if kind == "linear":
        c = dict(kind=kind, rows=_log(rng, 1, 4096), width=_log(rng, 64, 10000), outputs=_log(rng, 64, 10000), bias=rng.random() < 0.3, type=rng.choice(("bf16", "bf16", "fp32")))
        while c["rows"] * c["width"] * c["outputs"] > 4096 * 9728 * 2560:
            c["rows"] = c["rows"] // 2
        return c
    if kind == "mlp":
        c = dict(kind=kind, rows=_log(rng, 1, 2048), width=_log(rng, 64, 4096), inner=_log(rng, 64, 9728), type="bf16")
        while 3 * c["rows"] * c["width"] * c["inner"] > 4096 * 9728 * 2560:
            c["rows"] = c["rows"] // 2
        return c
    experts = _log(rng, 4, 128)
    c = dict(kind=kind, tokens=_log(rng, 1, 32), width=8 * _log(rng, 16, 384), inner=8 * _log(rng, 16, 256), experts=experts, top=rng.randint(1, min(8, experts)),
             weights=rng.choice(("bf16", "e4m3")))
    while experts * c["width"] * c["inner"] > 64 * 2048 * 1408 or c["tokens"] * c["top"] * c["width"] * c["inner"] > 192 * 2048 * 1408:
        c["width"], c["inner"] = c["width"] // 16 * 8, c["inner"] // 16 * 8
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _blocks(n):
    return -(-n // BLOCK)


def _wide(scales, rows, cols):
    """A block's scale for every entry of its matrix."""
    return scales.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def _matrix(gen, *shape):
    """A stack of random matrices as e4m3 numbers and block scales, the largest of a block at 448."""
    n, k = shape[-2:]
    w = torch.randn(*shape, generator=gen, device=DEV) * k**-0.5
    # columns of unlike size, as trained matrices have
    w = w * torch.exp(0.5 * torch.randn(k, generator=gen, device=DEV))
    padded = torch.nn.functional.pad(w, (0, -k % BLOCK, 0, -n % BLOCK))
    most = padded.abs().reshape(*shape[:-2], _blocks(n), BLOCK, _blocks(k), BLOCK).amax(dim=(-3, -1))
    scales = (most / TOP).clamp_min(1e-30)
    return (w / _wide(scales, n, k)).to(torch.float8_e4m3fn), scales


def _rows(gen, rows, width, dtype):
    """What a norm hands on: about unit size, some channels far larger."""
    x = torch.randn(rows, width, generator=gen, device=DEV)
    return (x * torch.exp(0.7 * torch.randn(width, generator=gen, device=DEV))).to(dtype)


def _package():
    at = os.path.join(os.getcwd(), "tiny-llm_b200")
    if at not in sys.path:
        sys.path.insert(0, at)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "linear":
        dtype = TYPES[case["type"]]
        s = {"x": _rows(gen, case["rows"], case["width"], dtype), "w": _matrix(gen, case["outputs"], case["width"])}
        s["bias"] = torch.randn(case["outputs"], generator=gen, device=DEV).to(dtype) if case["bias"] else None
        return s
    if case["kind"] == "mlp":
        d, ff = case["width"], case["inner"]
        return {"x": _rows(gen, case["rows"], d, TYPES[case["type"]]), "gate": _matrix(gen, ff, d), "up": _matrix(gen, ff, d), "down": _matrix(gen, d, ff)}
    d, ff, e = case["width"], case["inner"], case["experts"]
    s = {"x": _rows(gen, case["tokens"], d, torch.bfloat16), "top": case["top"]}
    s["router"] = (2.0 * torch.randn(e, d, generator=gen, device=DEV) * d**-0.5).to(torch.bfloat16)
    for name, shape in (("gate", (e, ff, d)), ("up", (e, ff, d)), ("down", (e, d, ff))):
        if case["weights"] == "bf16":
            s[name] = ((torch.randn(*shape, generator=gen, device=DEV) * shape[-1] ** -0.5).to(torch.bfloat16), None)
        else:
            s[name] = _matrix(gen, *shape)
    return s


def prepare(case, seed):
    s = {**case, **_inputs(case, seed)}
    if own:
        _package()
        from tiny_llm_b200 import Fp8Weights

        weights = lambda pair: pair[0] if pair[1] is None else Fp8Weights(*pair)  # noqa: E731
        if case["kind"] == "linear":
            s["weights"] = weights(s["w"])
        elif case["kind"] == "mlp":
            from tiny_llm_b200.mlp import Fp8GatedMLP

            s["layer"] = Fp8GatedMLP(weights(s["gate"]), weights(s["up"]), weights(s["down"]), "silu")
        else:
            from tiny_llm_b200.mlp import FewTokenExperts, TopKRouter

            s["layer"] = FewTokenExperts(TopKRouter(s["router"], None, s["top"]), weights(s["gate"]), weights(s["up"]), weights(s["down"]), "silu")
    return s


# ---- the plain forms, in 32 bits ------------------------------------------------------------------------------------


def _e4m3_rows(x):
    """The rows as the numbers that their e4m3 form stands for: every run of 128 of a row against its own largest."""
    rows, k = x.shape
    g = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).reshape(rows, -1, BLOCK)
    most = g.abs().amax(dim=-1, keepdim=True).clamp_min(SMALLEST)
    top = torch.full_like(most, TOP)  # a tensor: torch takes a quotient with a plain number as a product with a rounded reciprocal
    scale = torch.where(torch.isfinite(most), most / top, math.nan)
    q = (g * (top / most)).to(torch.float8_e4m3fn).float()
    return (q * scale).reshape(rows, -1)[:, :k]


def _numbers(pair):
    w, scales = pair
    return w.float() if scales is None else w.float() * _wide(scales, *w.shape[-2:])


def _product(rows, pair):
    return _e4m3_rows(rows) @ _numbers(pair).t()


def _silu(g):
    return g / (1.0 + torch.exp(-g))


def _plain_experts(s):
    x = s["x"].float()
    logits = s["x"].double() @ s["router"].double().t()  # in 64 bits: a choice lies next to a border
    chosen, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    chosen, ids = chosen[:, : s["top"]], ids[:, : s["top"]]
    share = torch.exp(chosen - chosen[:, :1])
    share = (share / share.sum(dim=-1, keepdim=True)).float()
    flat = ids.reshape(-1)
    of = lambda pair: _numbers((pair[0][flat] if pair[1] is None else pair[0].view(torch.uint8)[flat].view(torch.float8_e4m3fn), None if pair[1] is None else pair[1][flat]))  # noqa: E731
    rows = x.repeat_interleave(s["top"], 0)[:, :, None]
    inner = _silu(torch.bmm(of(s["gate"]), rows)) * torch.bmm(of(s["up"]), rows)
    out = torch.bmm(of(s["down"]), inner)[:, :, 0].reshape(*ids.shape, -1)
    return (out * share[:, :, None]).sum(dim=1)


def run(state):
    s = state
    if s["kind"] == "linear":
        if own:
            _package()
            from tiny_llm_b200 import fp8_linear

            return fp8_linear(s["x"], s["weights"], s["bias"])
        y = _product(s["x"], s["w"])
        return (y if s["bias"] is None else y + s["bias"].float()).to(s["x"].dtype)
    if own:
        return s["layer"](s["x"])
    if s["kind"] == "mlp":
        inner = _silu(_product(s["x"], s["gate"])) * _product(s["x"], s["up"])
        return _product(inner, s["down"]).to(s["x"].dtype)
    return _plain_experts(s).to(s["x"].dtype)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    matrix = lambda n, k: n * k + 4 * _blocks(n) * _blocks(k)  # noqa: E731
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["width"], case["outputs"]
        size = TYPES[case["type"]].itemsize
        return {"bytes": matrix(n, k) + size * (m * k + m * n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    if case["kind"] == "mlp":
        m, d, ff = case["rows"], case["width"], case["inner"]
        return {"bytes": 2 * matrix(ff, d) + matrix(d, ff) + 2 * TYPES[case["type"]].itemsize * m * d, "flops": 6 * m * d * ff}
    t, d, ff, e, top = (case[k] for k in ("tokens", "width", "inner", "experts", "top"))
    hit = e * (1.0 - (1.0 - top / e) ** t)  # experts that a token chooses, if choices are even
    each = 3 * d * ff * 2 if case["weights"] == "bf16" else 2 * matrix(ff, d) + matrix(d, ff)
    return {"bytes": int(hit * each) + 2 * e * d + 4 * t * d, "flops": 2 * t * e * d + 6 * t * top * d * ff}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------


def _nearest_e4m3(v):
    """The e4m3 number nearest to each v (|v| up to a little over 448), ties to the even one: three bits behind the leading one, steps of 2^-9 at the least."""
    _, e = torch.frexp(v)
    step = torch.exp2(torch.clamp(e.double() - 4, min=-9.0))
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _exact_rows(x):
    """Held numbers are what they are: a scale is the fp32 quotient, a number before its rounding the fp32 product."""
    x = x.float().double()
    out = torch.empty_like(x)
    for k in range(0, x.shape[1], BLOCK):
        run_ = x[:, k : k + BLOCK]
        most = run_.abs().max(dim=1, keepdim=True).values.clamp(min=SMALLEST)
        top = torch.full_like(most, 448.0)
        scale, times = (most / top).float().double(), (top / most).float().double()
        out[:, k : k + BLOCK] = _nearest_e4m3((run_ * times).float().double()) * scale
    return out


def _exact_matrix(values, scales):
    w = values.float().double()
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            w[i * BLOCK : (i + 1) * BLOCK, j * BLOCK : (j + 1) * BLOCK] *= scales[i, j].double()
    return w


def _exact_product(x, pair):
    return torch.einsum("mk,nk->mn", _exact_rows(x), _exact_matrix(*pair))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "linear":
        y = _exact_product(s["x"], s["w"])
        return y if s["bias"] is None else y + s["bias"].double()
    if case["kind"] == "mlp":
        g, u = _exact_product(s["x"], s["gate"]), _exact_product(s["x"], s["up"])
        return _exact_product(g * torch.sigmoid(g) * u, s["down"])
    x = s["x"].double()
    logits = torch.einsum("td,ed->te", x, s["router"].double())
    y = torch.zeros_like(x)
    for t in range(x.shape[0]):
        order = sorted(range(case["experts"]), key=lambda e, z=logits[t].tolist(): (-z[e], e))[: case["top"]]
        share = torch.softmax(logits[t, order], dim=0)
        for k, e in enumerate(order):
            m = [(p[0][e].double() if p[1] is None else _exact_matrix(p[0][e], p[1][e])) for p in (s["gate"], s["up"], s["down"])]
            g = m[0] @ x[t]
            y[t] += share[k] * (m[2] @ (g * torch.sigmoid(g) * (m[1] @ x[t])))
    return y
