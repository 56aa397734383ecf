"""A paged key/value cache of 8 bits, as cases that can be timed and compared.

Two operators.  ``append``: the keys and values of a step's new tokens go into the pages as e4m3 numbers, with one scale (a power of two) for each
16 tokens of a head; queries and keys pass an RMS norm per head and a rotation by their position on the way.  ``attend``: grouped-query
attention of a step's queries over such pages, for a decoded token, a few tokens at once, portions of a prompt.

A case is a dict of plain values; ``lengths`` are the requests' tokens in the cache once the step's ``new`` ones are in it (0: an idle slot).
Head layouts, page sizes and contexts are those of the framework's Qwen3 configurations and of its serving benchmark, or generic.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TOKENS = 16  # that share a scale
LEAST = -100  # the smallest scale is 2^-100
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _text(values):
    return ",".join(str(v) for v in values)


def listed():
    qwen = dict(heads=32, kv_heads=8, dim=128, page=128, type="bf16")  # the attention of the 4B configuration
    rotated = dict(rot=128, interleaved=False, norm=True)
    odd = dict(heads=10, kv_heads=2, dim=80, page=48, type="fp32")  # sizes that fill no tile, in the type that models are checked in
    return [
        # one decoding request: a token into a block that is begun already
        dict(name="append_1", kind="append", new=1, lengths="1011", **qwen, **rotated),
        # a decoding batch of full size, lengths as they come; some tokens begin a block, some a page
        dict(name="append_64", kind="append", new=1, lengths=_text(17 + 53 * i % 1011 for i in range(64)), **qwen, **rotated),
        # short portions of several requests beside an idle slot, odd sizes, interleaved pairs, part of a head rotated
        dict(name="append_3x37_odd_fp32", kind="append", new=37, lengths="37,0,1290,481", **odd, rot=64, interleaved=True, norm=False),
        # the scheduler's portion of a prompt
        dict(name="append_128", kind="append", new=128, lengths="1500", **qwen, **rotated),
        # a whole prompt behind an earlier turn
        dict(name="append_2048", kind="append", new=2048, lengths="3500", **qwen, **rotated),
        # one decoding request, where latency counts
        dict(name="attend_1x1011", kind="attend", new=1, lengths="1011", causal=True, **qwen),
        # one decoding request far into a long document: few rows, one long axis
        dict(name="attend_1x32000", kind="attend", new=1, lengths="32000", causal=True, **qwen),
        # a serving step of two dozen answers
        dict(name="attend_24", kind="attend", new=1, lengths=_text(70 + 113 * i % 1901 for i in range(24)), causal=True, **qwen),
        # the serving benchmark with contexts of 8K
        dict(name="attend_64x8192", kind="attend", new=1, lengths=_text([8192] * 64), causal=True, **qwen),
        # a few tokens at once over odd sizes, an idle slot among them, every key visible
        dict(name="attend_3_odd_fp32", kind="attend", new=3, lengths="900,3,0,2111,48", causal=False, **odd),
        # the scheduler's portion of a long prompt
        dict(name="attend_128x3500", kind="attend", new=128, lengths="3500", causal=True, **qwen),
        # a large portion
        dict(name="attend_2048x3500", kind="attend", new=2048, lengths="3500", causal=True, **qwen),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    heads, kv_heads = rng.choice([(32, 8), (16, 8), (10, 2), (8, 8), (12, 1), (14, 2)])
    c = dict(kind=rng.choice(["append", "attend", "attend"]), heads=heads, kv_heads=kv_heads, dim=rng.choice([128, 128, 64, 80, 96, 256]), page=rng.choice([128, 128, 64, 48, 16]),
             type=rng.choice(["bf16", "bf16", "fp32"]))
    c["new"] = rng.choice([1, 1, log(2, 16), log(17, 2048)])
    # rows x keys, and keys x their bytes, stay below the largest listed ones
    most = min(8192, max(c["new"] + 1, (2048 * 3500 * 32 * 128) // (c["new"] * heads * c["dim"])))
    room = 64 * 8192 * 8 * 128 // (kv_heads * c["dim"])
    rows = log(1, max(1, min(64, 4096 // c["new"]))) if c["new"] < 64 else 1
    lengths = []
    for _ in range(rows):
        n = log(c["new"], max(c["new"], most))
        if c["type"] == "fp32":
            n = max(c["new"], min(n, 2500))
        lengths.append(0 if rows > 2 and rng.random() < 0.1 else n)
    if not any(lengths):
        lengths[0] = c["new"]
    while sum(lengths) > room or sum(lengths) * c["new"] * heads * c["dim"] > 2048 * 3500 * 32 * 128:
        lengths.pop()
    c["lengths"] = _text(lengths or [c["new"]])
    if c["kind"] == "append":
        c.update(rot=rng.choice([0, c["dim"], c["dim"] // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.5)
    else:
        c["causal"] = rng.random() < 0.8
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _power(e):
    """2^e, to the bit."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(most):
    """The smallest e, at least LEAST, with ``most`` <= 448 * 2^e."""
    m, e = torch.frexp(most)
    return torch.clamp(e - 9 + (m > 0.875), min=LEAST)


def _cache(gen, pages, case, like):
    """Pages of earlier tokens, as the operator leaves them: -> numbers [P, H, page, D], scales [P, H, page / 16]."""
    h, n, d = case["kv_heads"], case["page"], case["dim"]
    x = torch.randn(pages, h, n, d, generator=gen, device=DEV)
    x *= torch.exp((1.0 if like == "keys" else 0.3) * torch.randn(h, 1, d, generator=gen, device=DEV))  # keys have channels far larger than others
    x *= torch.exp(0.5 * torch.randn(pages, h, n, 1, generator=gen, device=DEV))  # and tokens are of unlike size
    blocks = x.view(pages, h, n // TOKENS, TOKENS * d)
    e = _exponent(blocks.abs().amax(dim=-1))
    blocks *= _power(-e)[..., None]
    return x.to(torch.float8_e4m3fn), _power(e)


def _inputs(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lengths, page = _lengths(case), case["page"]
    live = [-(-n // page) for n in lengths]
    pages = sum(live) + 2
    order = np.random.RandomState(seed % 2**32).permutation(pages).astype(np.int32)
    table = np.full((len(lengths), max(live)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(live):
        table[b, :n] = order[at : at + n]
        at += n
    s = {"table_host": table, "lengths_host": np.asarray(lengths, dtype=np.int32)}
    s["table"], s["lengths"] = torch.from_numpy(table).to(DEV), torch.from_numpy(s["lengths_host"]).to(DEV)
    s["keys"], s["key_scales"] = _cache(gen, pages, case, "keys")
    s["values"], s["value_scales"] = _cache(gen, pages, case, "values")
    b, new, d, dtype = len(lengths), case["new"], case["dim"], TYPES[case["type"]]
    # a step's projections come token by token, heads side by side
    make = lambda heads: torch.randn(b, new, heads, d, generator=gen, device=DEV)  # noqa: E731
    if case["kind"] == "attend":
        s["query"] = (2.0 * make(case["heads"])).to(dtype).transpose(1, 2)
        return s
    wide = lambda heads: torch.exp(0.5 * torch.randn(heads, d, generator=gen, device=DEV))  # noqa: E731
    for name, heads in (("query", case["heads"]), ("key", case["kv_heads"]), ("value", case["kv_heads"])):
        s[name] = (make(heads) * wide(heads)).to(dtype).transpose(1, 2)
    s["query_weight"], s["key_weight"] = ((1.0 + 0.3 * torch.randn(d, generator=gen, device=DEV)).to(dtype) if case["norm"] else None for _ in range(2))
    return s


def _package():
    at = os.path.join(os.getcwd(), "tiny-llm_b200")
    if at not in sys.path:
        sys.path.insert(0, at)


BASE = 1000000


def prepare(case, seed):
    s = {**case, **_inputs(case, seed)}
    if own:
        _package()
        from tiny_llm_b200 import FastRMSNorm, FastRoPE, Fp8KvPages

        s["pages"] = Fp8KvPages(s["keys"], s["values"], s["key_scales"], s["value_scales"])
        if case["kind"] == "append":
            s["rope"] = FastRoPE(case["rot"], 32768, BASE, traditional=case["interleaved"]) if case["rot"] else None
            s["query_norm"], s["key_norm"] = (None if w is None else FastRMSNorm(case["dim"], w, eps=EPS) for w in (s["query_weight"], s["key_weight"]))
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------


def _turn(x, s, weight, positions):
    """Norm and rotation of ``x`` [B, H, L, D], in ``x``'s own number of bits."""
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * weight.to(x.dtype)
    if not s["rot"]:
        return x
    half = s["rot"] // 2
    frequency = torch.pow(torch.tensor(float(BASE), dtype=torch.float64, device=DEV), -torch.arange(half, dtype=torch.float64, device=DEV) / half)
    angle = positions.double()[:, None, :, None] * frequency  # in 64 bits: a far position times a frequency
    c, n = torch.cos(angle).to(x.dtype), torch.sin(angle).to(x.dtype)
    if s["interleaved"]:
        one, two = x[..., 0 : s["rot"] : 2], x[..., 1 : s["rot"] : 2]
        turned = torch.stack([one * c - two * n, two * c + one * n], dim=-1).flatten(-2)
    else:
        one, two = x[..., :half], x[..., half : s["rot"]]
        turned = torch.cat([one * c - two * n, two * c + one * n], dim=-1)
    return torch.cat([turned, x[..., s["rot"] :]], dim=-1)


def _store(x, numbers, scales, s):
    """The new tokens' ``x`` [B, H, L, D] into the pages: a block's scale grows with them, what it held is rounded again to the new one."""
    b, h, new, d = x.shape
    lengths, page = s["lengths"].long(), s["page"]
    first = lengths - new
    blocks = (new + 2 * TOKENS - 2) // TOKENS
    block = (first // TOKENS).clamp_min(0)[:, None] + torch.arange(blocks, device=DEV)  # [B, n]
    position = block[:, :, None] * TOKENS + torch.arange(TOKENS, device=DEV)  # [B, n, 16]
    fresh = (position >= first[:, None, None]) & (position < lengths[:, None, None])
    row, slot = torch.nonzero(fresh.any(dim=-1), as_tuple=True)
    at, fresh = block[row, slot], fresh[row, slot]  # [N], [N, 16]
    token = (position[row, slot] - first[row, None]).clamp(0, new - 1)
    x = x[row[:, None], :, token].transpose(1, 2)  # [N, H, 16, D]
    x = torch.where(fresh[:, None, :, None], x, torch.zeros_like(x))
    numbers = numbers.view(torch.uint8).view(-1, h, page // TOKENS, TOKENS, d)
    home, part = s["table"][row, at * TOKENS // page].long(), at % (page // TOKENS)
    held = numbers[home, :, part].view(torch.float8_e4m3fn).float()
    before = torch.where((at * TOKENS < first[row])[:, None], scales[home, :, part], torch.zeros_like(scales[home, :, part]))
    scale = torch.maximum(before, _power(_exponent(x.abs().amax(dim=(-1, -2)))))
    under = 1.0 / scale[:, :, None, None]
    kept = (held * (before[:, :, None, None] * under)).to(torch.float8_e4m3fn).view(torch.uint8)
    put = torch.where(fresh[:, None, :, None], (x * under).to(torch.float8_e4m3fn).view(torch.uint8), kept)
    old = (position[row, slot] < first[row, None]) | fresh  # slots behind the last token stay as they are
    numbers[home, :, part] = torch.where(old[:, None, :, None], put, numbers[home, :, part])
    scales[home, :, part] = scale


def _append(s):
    positions = (s["lengths"][:, None] - s["new"] + torch.arange(s["new"], device=DEV)).clamp_min(0)
    query = _turn(s["query"].float(), s, s["query_weight"], positions)
    query = torch.where(s["lengths"][:, None, None, None] > 0, query, torch.zeros_like(query)).to(s["query"].dtype)
    # keys in 64 bits, and then as numbers of 32: they are rounded to few bits, next to a border of which the last ones decide
    _store(_turn(s["key"].double(), s, s["key_weight"], positions).float(), s["keys"], s["key_scales"], s)
    _store(s["value"].float(), s["values"], s["value_scales"], s)
    return query


def _gather(numbers, scales, s):
    """The cache of every request as fp32 numbers [B, H, S, D], rows behind its last token among them."""
    table = s["table"].long().clamp_min(0)
    wide = numbers.view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * scales[table].repeat_interleave(TOKENS, -1)[..., None]  # [B, pages, H, page, D]
    return wide.transpose(1, 2).flatten(2, 3)


def _attend(s):
    b, heads, new, d = s["query"].shape
    h = s["kv_heads"]
    q = s["query"].float().reshape(b, h, heads // h * new, d)
    scores = (q @ _gather(s["keys"], s["key_scales"], s).transpose(-1, -2)).view(b, h, heads // h, new, -1) * d**-0.5
    key = torch.arange(scores.shape[-1], device=DEV)
    limit = s["lengths"].long()[:, None].expand(b, new)
    if s["causal"]:
        limit = (limit - new + 1 + torch.arange(new, device=DEV)).clamp_min(0)
    seen = key < limit[:, :, None]  # [B, L, S]
    scores = torch.where(seen[:, None, None], scores, torch.full_like(scores, -math.inf))
    most = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isfinite(most), most, torch.zeros_like(most)))
    p = p / p.sum(dim=-1, keepdim=True).clamp_min(1e-30)
    values = _gather(s["values"], s["value_scales"], s)
    return (p.view(b, h, -1, key.numel()) @ values).view(b, heads, new, d).to(s["query"].dtype)


def run(state):
    s = state
    if s["kind"] == "attend":
        if own:
            _package()
            from tiny_llm_b200 import paged_attention_fp8

            return paged_attention_fp8(s["query"], s["pages"], s["table"], s["lengths"], mask="causal" if s["causal"] else None, block_table_host=s["table_host"],
                                       context_lens_host=s["lengths_host"])
        return _attend(s)
    if own:
        _package()
        from tiny_llm_b200 import rotate_append_fp8

        query = rotate_append_fp8(s["query"], s["key"], s["value"], s["pages"], s["table"], s["lengths"], rope=s["rope"], query_norm=s["query_norm"], key_norm=s["key_norm"],
                                  block_table_host=s["table_host"], context_lens_host=s["lengths_host"])
    else:
        query = _append(s)
    return {"query": query, "keys": s["keys"], "values": s["values"], "key_scales": s["key_scales"], "value_scales": s["value_scales"]}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(case):
    lengths, new, d, size = _lengths(case), case["new"], case["dim"], TYPES[case["type"]].itemsize
    rows = sum(n > 0 for n in lengths) * new
    if case["kind"] == "append":
        read = size * rows * d * (case["heads"] + 2 * case["kv_heads"])
        blocks = sum((n - 1) // TOKENS - (n - new) // TOKENS + 1 for n in lengths if n)
        write = size * rows * d * case["heads"] + 2 * case["kv_heads"] * (rows * d + 4 * blocks)
        return {"bytes": read + write, "flops": 6 * rows * d * (case["heads"] + case["kv_heads"])}
    keys = sum(n for n in lengths)
    pairs = sum(n * new - (new * (new - 1) // 2 if case["causal"] else 0) for n in lengths if n)
    each = 2 * d + 2 * 4 / TOKENS
    return {"bytes": int(keys * case["kv_heads"] * each) + 2 * size * rows * d * case["heads"], "flops": 4 * d * case["heads"] * pairs}


# ---- the definition, in 64 bits -------------------------------------------------------------------------------------


def _nearest_e4m3(v):
    """The e4m3 number nearest to each v (up to 448), ties to the even one: three bits behind the leading one, steps of 2^-9 at the least."""
    _, e = torch.frexp(v)
    step = torch.exp2(torch.clamp(e.double() - 4, min=-9.0))
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def _exact_rows(x, weight, case, position):
    """``x`` [H, L, D] in 64 bits, token i at ``position + i``."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(torch.mean(y.square(), dim=-1, keepdim=True) + EPS) * weight.double()
    rot = case["rot"]
    if rot:
        z = y.clone()
        at = torch.arange(position, position + x.shape[1], dtype=torch.float64, device=DEV)
        for i in range(rot // 2):
            c, n = torch.cos(at * float(BASE) ** (-2.0 * i / rot)), torch.sin(at * float(BASE) ** (-2.0 * i / rot))
            j, k = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + rot // 2)
            z[..., j] = y[..., j] * c - y[..., k] * n
            z[..., k] = y[..., j] * n + y[..., k] * c
        y = z
    return y


def _exact_append(case, s):
    out = {"query": torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)}
    turned = []
    for b, n in enumerate(_lengths(case)):
        if n:
            out["query"][b] = _exact_rows(s["query"][b], s["query_weight"], case, n - case["new"])
            turned.append((b, n, _exact_rows(s["key"][b], s["key_weight"], case, n - case["new"]).float().double(), s["value"][b].double()))
    for name, which in (("key", 2), ("value", 3)):
        numbers, scales = s[name + "s"].float().double(), s[name + "_scales"].double()
        for entry in turned:
            b, n, x = entry[0], entry[1], entry[which]
            first = n - case["new"]
            for start in range(first - first % TOKENS, n, TOKENS):
                lo, hi = max(start, first), min(start + TOKENS, n)
                home, at = int(s["table_host"][b, start // case["page"]]), start % case["page"]
                part = x[:, lo - first : hi - first]
                most = part.abs().amax(dim=(1, 2))
                e = torch.clamp(torch.ceil(torch.log2(most / 448.0)), min=LEAST)
                e = torch.where(most > 448.0 * torch.exp2(e), e + 1, torch.where((most <= 448.0 * torch.exp2(e - 1)) & (e > LEAST), e - 1, e))
                scale = torch.exp2(e)
                if lo > start:
                    before = scales[home, :, at // TOKENS].clone()
                    scale = torch.maximum(scale, before)
                    held = numbers[home, :, at : at + lo - start]
                    numbers[home, :, at : at + lo - start] = _nearest_e4m3(held * (before / scale)[:, None, None])
                numbers[home, :, at + lo - start : at + hi - start] = _nearest_e4m3(part / scale[:, None, None])
                scales[home, :, at // TOKENS] = scale
        out[name + "s"], out[name + "_scales"] = numbers, scales
    return out


def _exact_attend(case, s):
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=DEV)
    group, new = case["heads"] // case["kv_heads"], case["new"]
    for b, n in enumerate(_lengths(case)):
        if not n:
            continue
        homes = s["table"][b, : -(-n // case["page"])].long()
        dense = []
        for numbers, scales in ((s["keys"], s["key_scales"]), (s["values"], s["value_scales"])):
            x = numbers.view(torch.uint8)[homes].view(torch.float8_e4m3fn).double().unflatten(2, (-1, TOKENS)) * scales[homes].double()[..., None, None]
            dense.append(torch.cat(list(x.flatten(2, 3)), dim=1)[:, :n])
        hidden = torch.arange(n, device=DEV)[None, :] > torch.arange(n - new, n, device=DEV)[:, None] if case["causal"] else None
        for head in range(case["heads"]):
            scores = torch.einsum("ld,sd->ls", s["query"][b, head].double(), dense[0][head // group]) / math.sqrt(case["dim"])
            if hidden is not None:
                scores = scores.masked_fill(hidden, -math.inf)
            out[b, head] = torch.einsum("ls,sd->ld", torch.softmax(scores, dim=-1), dense[1][head // group])
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_append(case, s) if case["kind"] == "append" else _exact_attend(case, s)
