"""The paged cache of 8 bits against float64: what an append leaves in the pages and what attention makes of them, at the edges of blocks, pages and
tiles, over strides, idle slots, numbers that are none; streams, captured graphs, both in a row.

Tolerances.  A number in the pages is the e4m3 number nearest to the exact value over the block's scale: half a step of e4m3 (2^-4 relative, 2^-10 of the
scale among the smallest), and 2^-23 of the value for its way through fp32.  Scores are sums of exact products, added in the tensor cores (an addition
is off by at most 2^-23 of what is added, if it cuts); see ``attention_tolerance``."""

import math

import numpy as np
import pytest
import torch

from tiny_llm_b200 import FastRMSNorm, FastRoPE, Fp8KvPages, paged_attention_fp8, rotate_append_fp8

DEV = "cuda"
gpu = pytest.mark.gpu
BASE = 10000


def nearest_e4m3(v):
    _, e = torch.frexp(v)
    step = torch.exp2(torch.clamp(e.double() - 4, min=-9.0))
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def exponent(most):
    """The smallest e >= -100 with most <= 448 * 2^e."""
    e = -100
    while most > 448.0 * 2.0**e:
        e += 1
    return e


def table_of(lengths, page, seed=0, spare=2, width=None):
    live = [-(-n // page) for n in lengths]
    order = np.random.RandomState(seed).permutation(sum(live) + spare).astype(np.int32)
    table = np.full((len(lengths), width or max(max(live), 1)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(live):
        table[b, :n] = order[at : at + n]
        at += n
    return table, sum(live) + spare


def random_pages(count, heads, page, dim, gen, wide=1.0):
    """Pages of random numbers with random powers of two as scales, every slot of them filled."""
    pages = Fp8KvPages.zeros(count, heads, page, dim, device="cpu")
    pages.keys.copy_((torch.randn(pages.keys.shape, generator=gen) * 60).clamp(-448, 448).to(torch.float8_e4m3fn))
    pages.values.copy_((torch.randn(pages.keys.shape, generator=gen) * 60).clamp(-448, 448).to(torch.float8_e4m3fn))
    for s, base in ((pages.key_scales, -6), (pages.value_scales, -5)):
        s.copy_(torch.exp2(base + torch.round(wide * torch.randn(s.shape, generator=gen))))
    return pages


def to_gpu(pages):
    return Fp8KvPages(*(t.to(DEV) for t in (pages.keys, pages.values, pages.key_scales, pages.value_scales)))


def copy_of(pages):
    return Fp8KvPages(*(t.clone() for t in (pages.keys, pages.values, pages.key_scales, pages.value_scales)))


def on_host(t):
    return t.cpu().float().double()


# ---- append -----------------------------------------------------------------------------------------------------------


def turned(x, weight, eps, rot, traditional, position):
    """``x`` [L, D] of one head in 64 bits: norm, then rotation."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(dim=-1, keepdim=True) + eps) * weight.double()
    z = y.clone()
    for i in range(rot // 2):
        angle = (position + torch.arange(x.shape[0], dtype=torch.float64)) * float(BASE) ** (-2.0 * i / rot)
        j, k = (2 * i, 2 * i + 1) if traditional else (i, i + rot // 2)
        z[:, j] = y[:, j] * torch.cos(angle) - y[:, k] * torch.sin(angle)
        z[:, k] = y[:, j] * torch.sin(angle) + y[:, k] * torch.cos(angle)
    return z


def check_side(name, got, got_scales, old, old_scales, x64, table, lengths, new, page):
    """One side of the pages after an append of ``x64`` [B, H, L, D] (float64): new numbers, numbers rounded again, and everything else as it was."""
    want_q, want_s = old.clone(), old_scales.clone()
    touched = torch.zeros(old.shape[:3], dtype=torch.bool)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        first = n - new
        for start in range(first - first % 16, n, 16):
            lo, hi = max(first, start), min(n, start + 16)
            home, at = int(table[b, start // page]), start % page
            for h in range(old.shape[1]):
                part = x64[b, h, lo - first : hi - first]
                before = float(old_scales[home, h, at // 16])
                s = float(got_scales[home, h, at // 16])
                if not torch.isfinite(part).all() or (lo > start and math.isnan(before)):
                    assert math.isnan(s), (name, b, h, start)
                    touched[home, h, at : at + 16] = True
                    want_s[home, h, at // 16] = math.nan
                    continue
                most = float(part.abs().max())
                choices = {2.0 ** exponent(most * (1 - 2.0**-23)), 2.0 ** exponent(most * (1 + 2.0**-23))}  # the border itself may fall either way
                if lo > start:
                    choices = {max(c, before) for c in choices}
                assert s in choices, (name, b, h, start, s, choices)
                want_s[home, h, at // 16] = s
                if lo > start:
                    want_q[home, h, at : at + lo - start] = nearest_e4m3(old[home, h, at : at + lo - start] * (before / s))
                num = got[home, h, at + lo - start : at + hi - start]
                want = part / s
                half = torch.maximum(torch.exp2(torch.floor(torch.log2(want.abs().clamp_min(2.0**-6))) - 4), torch.tensor(2.0**-10, dtype=torch.float64))
                assert ((num - want).abs() <= half * (1 + 2.0**-10) + 2.0**-23 * want.abs()).all(), (name, b, h, start)
                assert torch.equal(num, nearest_e4m3(num))
                touched[home, h, at + lo - start : at + hi - start] = True
    same = ~touched
    assert torch.equal(got[same], want_q[same]), name
    assert torch.equal(torch.nan_to_num(got_scales, nan=-1.0), torch.nan_to_num(want_s, nan=-1.0)), name


def run_append(lengths, new, heads, kv_heads, dim, page, dtype, *, rot=None, traditional=False, norm=True, seed=0, change=None, layout="tokens", width=None):
    gen = torch.Generator().manual_seed(seed + 1)
    table, count = table_of(lengths, page, seed, width=width)
    pages = random_pages(count, kv_heads, page, dim, gen)
    b = len(lengths)

    def rows(h):
        x = torch.randn(b, new, h, dim, generator=gen) * torch.exp(torch.randn(h, dim, generator=gen)) * torch.exp2(torch.randint(-3, 4, (b, new, 1, 1), generator=gen).float())
        return x.to(dtype)

    q, k, v = rows(heads), rows(kv_heads), rows(kv_heads)
    if change:
        change(q, k, v)
    if layout == "tokens":
        gq, gk, gv = (x.to(DEV).transpose(1, 2) for x in (q, k, v))
    elif layout == "heads":
        gq, gk, gv = (x.transpose(1, 2).contiguous().to(DEV) for x in (q, k, v))
    else:  # columns of one wide product
        wide = torch.cat([x.reshape(b, new, -1) for x in (q, k, v)] + [torch.full((b, new, 3), 9.0, dtype=dtype)], dim=-1).to(DEV)
        cuts = [0, heads * dim, (heads + kv_heads) * dim, (heads + 2 * kv_heads) * dim]
        gq, gk, gv = (wide[..., lo:hi].unflatten(-1, (-1, dim)).transpose(1, 2) for lo, hi in zip(cuts, cuts[1:]))
    rot = dim if rot is None else rot
    eps = 1e-6
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype) if norm else None for _ in range(2))
    norms = {} if not norm else dict(query_norm=FastRMSNorm(dim, wq.to(DEV), eps=eps), key_norm=FastRMSNorm(dim, wk.to(DEV), eps=eps))
    gp = to_gpu(pages)
    out = rotate_append_fp8(gq, gk, gv, gp, torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV),
                            rope=FastRoPE(rot, 4096, BASE, traditional=traditional) if rot else None, **norms)
    assert out.shape == gq.shape and out.dtype == dtype
    k64 = torch.zeros(b, kv_heads, new, dim, dtype=torch.float64)
    for i, n in enumerate(lengths):
        for h in range(heads):
            want = turned(q[i, :, h], wq, eps, rot, traditional, n - new) if n else torch.zeros(new, dim, dtype=torch.float64)
            got = out[i, h].cpu().double()
            if not torch.isfinite(want).all():
                bad = ~torch.isfinite(q[i, :, h].double()).all(dim=-1)
                got, want = got[~bad], want[~bad]
            # the norm: a sum of D squares (D / 32 + 5 additions), a division, a root, their products; the turn: two products, an addition, rounded cos and sin
            size = want.abs() if rot == 0 else want.abs() + turned(q[i, :, h], wq, eps, 0, False, 0)[: want.shape[0]].abs().amax(dim=-1, keepdim=True) if torch.isfinite(q[i, :, h].double()).all() else want.abs() + 1e9
            tol = (dim / 32 + 16) * 2.0**-24 * size + torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + 1e-30
            assert ((got - want).abs() <= tol).all(), (i, h, float(((got - want).abs() - tol).max()))
        if n:
            for h in range(kv_heads):
                k64[i, h] = turned(k[i, :, h], wk, eps, rot, traditional, n - new)
    check_side("keys", on_host(gp.keys), on_host(gp.key_scales), on_host(pages.keys), on_host(pages.key_scales), k64, table, lengths, new, page)
    check_side("values", on_host(gp.values), on_host(gp.value_scales), on_host(pages.values), on_host(pages.value_scales), v.double().transpose(1, 2), table, lengths, new, page)


@gpu
@pytest.mark.parametrize("lengths,new", [([1], 1), ([16], 1), ([17], 1), ([128], 1), ([129], 1), ([1000, 0, 33, 48], 1), ([5], 5), ([16], 16), ([17], 17), ([40, 300], 15), ([64, 0, 95], 33),
                                         ([0, 0], 1), ([700], 256)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_at_the_edges_of_blocks_and_pages(lengths, new, dtype):
    run_append(lengths, new, 4, 2, 64, 64, dtype, seed=sum(lengths) + new)


@gpu
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(1, 1, 16, 16), (4, 2, 32, 32), (10, 2, 80, 48), (12, 1, 96, 16), (32, 8, 128, 128), (6, 6, 256, 80), (3, 3, 144, 16)])
@pytest.mark.parametrize("layout", ["tokens", "heads", "columns"])
def test_append_over_head_layouts_and_strides(heads, kv_heads, dim, page, layout):
    run_append([70, 0, 9], 7, heads, kv_heads, dim, page, torch.bfloat16, seed=dim, layout=layout)


@gpu
@pytest.mark.parametrize("rot,traditional,norm", [(0, False, False), (0, False, True), (32, False, True), (96, True, False), (2, True, True), (94, False, False)])
def test_append_with_parts_of_the_way_left_out(rot, traditional, norm):
    run_append([50, 21], 20, 6, 2, 96, 32, torch.float32, rot=rot, traditional=traditional, norm=norm)
    run_append([1200], 3, 6, 2, 96, 32, torch.bfloat16, rot=rot, traditional=traditional, norm=norm)


@gpu
def test_append_of_zeros_tiny_and_huge_numbers():
    def change(q, k, v):
        k[0, :, 0], v[0, :, 0] = 0.0, 0.0
        k[0, :, 1], v[0, :, 1] = k[0, :, 1] * 1e-36, v[0, :, 1] * 1e-36
        k[1], v[1] = k[1] * 1e30, v[1] * 1e30

    run_append([16, 48], 16, 4, 2, 32, 16, torch.float32, norm=False, change=change)
    run_append([21, 53], 16, 4, 2, 32, 16, torch.bfloat16, norm=False, change=change)


@gpu
def test_a_number_that_is_none_takes_its_block_along_and_nothing_else():
    def change(q, k, v):
        k[0, 3, 0, 5] = math.inf
        v[1, 10, 1, 7] = math.nan
        q[0, 2, 1, 1] = math.nan

    run_append([40, 24], 20, 4, 2, 32, 16, torch.bfloat16, norm=False, change=change)


@gpu
def test_a_block_begun_anew_forgets_the_scale_before():
    pages = Fp8KvPages.zeros(1, 1, 16, 16)
    pages.key_scales.fill_(math.nan)
    pages.value_scales.fill_(2.0**90)
    x = torch.full((1, 1, 1, 16), 3.0, device=DEV)
    rotate_append_fp8(x, x, x, pages, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV))
    assert pages.key_scales.item() == pages.value_scales.item() == 2.0**-7  # 3 <= 448 / 128
    k, v = pages.dequantize()
    assert (k[0, 0, 0] == 3).all() and (v[0, 0, 0] == 3).all()


@gpu
def test_tokens_one_by_one_and_together_leave_nearly_the_same():
    """Scales are powers of two: rounding again costs a number nothing unless it falls below 2^-6 of the scale."""
    gen = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(1, h, 40, 64, generator=gen).to(torch.bfloat16).to(DEV) for h in (4, 2, 2))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    one, all_ = Fp8KvPages.zeros(3, 2, 16, 64), Fp8KvPages.zeros(3, 2, 16, 64)
    rope = FastRoPE(64, 128, BASE)
    width = lambda n: torch.where(torch.arange(3, device=DEV) < -(-n // 16), table, torch.full_like(table, -1))  # noqa: E731
    rotate_append_fp8(q, k, v, all_, table, torch.tensor([40], dtype=torch.int32, device=DEV), rope=rope)
    for i in range(40):
        rotate_append_fp8(q[:, :, i : i + 1], k[:, :, i : i + 1], v[:, :, i : i + 1], one, width(i + 1), torch.tensor([i + 1], dtype=torch.int32, device=DEV), rope=rope)
    assert torch.equal(one.key_scales, all_.key_scales) and torch.equal(one.value_scales, all_.value_scales)
    for a, b, s in zip(one.dequantize(), all_.dequantize(), (one.key_scales, one.value_scales)):
        step = s.repeat_interleave(16, -1)[..., None] * 2.0**-9
        assert ((a - b).abs() <= step).all()


# ---- attention --------------------------------------------------------------------------------------------------------


def dense(pages, table, n, page):
    """(keys, values) of a request in 64 bits [H, n, D]."""
    homes = [int(p) for p in table[: -(-n // page)]]
    out = []
    for numbers, scales in ((pages.keys, pages.key_scales), (pages.values, pages.value_scales)):
        wide = on_host(numbers)[homes] * on_host(scales)[homes].repeat_interleave(16, -1)[..., None]
        out.append(wide.transpose(0, 1).flatten(1, 2)[:, :n])
    return out


def attention_tolerance(q, k, v, p, scale, want, dtype, dim):
    """``q`` [L, D], ``k`` and ``v`` [n, D], weights ``p`` [L, n].  A score: D exact products added up in steps of 16 (each with an addition per product at the most), queries that keep all bits (bf16) or 22;
    the running maximum is exact for what it is used for; exp2 2^-22; the weight rounded to f16 (2^-12, and 2^-25 of the largest that the running maximum allows, 2^8) or to 22 bits.  A weight off by a
    factor 1 + d is off in the output and in the sum."""
    most = q.abs() @ k.abs().t() * abs(scale)
    score = (dim / 16 + 6) * 2.0**-22 * most
    d = score + 2.0**-21 + (2.0**-12 if dtype == torch.bfloat16 else 2.0**-22)
    d = d + 2.0**-20  # sums of weights and of products in fp32
    floor = 2.0**-16 if dtype == torch.bfloat16 else 2.0**-27  # a weight among f16's smallest, relative to the row's largest
    size = (p * d) @ v.abs() + (p * d).sum(-1, keepdim=True) * want.abs() + floor * p.max(-1, keepdim=True).values * (v.abs().sum(0) / 64 + v.abs().max(0).values)
    return size + torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + 1e-30


def check_attention(out, q, pages, table, lengths, causal, scale, dtype):
    page, dim = pages.page_size, pages.head_dim
    group, new = q.shape[1] // pages.kv_heads, q.shape[2]
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = dense(pages, table[b], n, page)
        for h in range(q.shape[1]):
            x = q[b, h].double()
            s = x @ k[h // group].t() * scale
            if causal:
                s = s.masked_fill(torch.arange(n)[None] > torch.arange(n - new, n)[:, None], -math.inf)
            p = torch.softmax(s, dim=-1)
            want = p @ v[h // group]
            tol = attention_tolerance(x, k[h // group], v[h // group], p, scale, want, dtype, dim)
            far = (out[b, h].cpu().double() - want).abs() - tol
            assert (far <= 0).all(), (b, h, float(far.max()), float(tol.mean()))


def run_attention(lengths, new, heads, kv_heads, dim, page, dtype, *, causal=True, scale=None, seed=0, wide=1.0, layout="tokens", strength=1.0, width=None):
    gen = torch.Generator().manual_seed(seed + 5)
    table, count = table_of(lengths, page, seed, width=width)
    pages = random_pages(count, kv_heads, page, dim, gen, wide)
    q = (strength * torch.randn(len(lengths), new, heads, dim, generator=gen)).to(dtype)
    gq = q.to(DEV).transpose(1, 2) if layout == "tokens" else q.transpose(1, 2).contiguous().to(DEV)
    out = paged_attention_fp8(gq, to_gpu(pages), torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=scale, mask="causal" if causal else None,
                              block_table_host=table, context_lens_host=np.asarray(lengths, dtype=np.int32))
    assert out.shape == gq.shape and out.dtype == dtype
    check_attention(out, q.transpose(1, 2), pages, table, lengths, causal, dim**-0.5 if scale is None else scale, dtype)


@gpu
@pytest.mark.parametrize("lengths,new", [([1], 1), ([15], 1), ([16], 1), ([17], 1), ([64], 1), ([65], 1), ([0, 1, 700], 1), ([257], 2), ([3, 0, 40], 3), ([130, 31], 9), ([16], 16), ([90], 33), ([2049], 1)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_at_the_edges_of_blocks_and_pages(lengths, new, causal, dtype):
    run_attention(lengths, new, 8, 2, 64, 64, dtype, causal=causal, seed=sum(lengths) + new)


@gpu
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(1, 1, 16, 16), (4, 2, 32, 32), (10, 2, 80, 48), (12, 1, 96, 16), (32, 8, 128, 128), (6, 6, 256, 80), (3, 3, 144, 16), (16, 1, 128, 64), (17, 1, 64, 16)])
@pytest.mark.parametrize("new", [1, 4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_over_head_layouts(heads, kv_heads, dim, page, new, dtype):
    run_attention([150, 0, 37], new, heads, kv_heads, dim, page, dtype, seed=dim + new, layout="heads" if new == 1 else "tokens")


@gpu
@pytest.mark.parametrize("lengths,new", [([300], 128), ([128], 128), ([1000, 450], 200), ([77, 0], 77)])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 128), (8, 2, 64, 16), (6, 1, 128, 48), (8, 8, 128, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_portions(lengths, new, heads, kv_heads, dim, page, causal):
    run_attention(lengths, new, heads, kv_heads, dim, page, torch.bfloat16, causal=causal, seed=new)


@gpu
@pytest.mark.parametrize("new", [1, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_with_scales_far_apart_and_strong_queries(new, dtype):
    run_attention([333], new, 4, 2, 128, 64, dtype, wide=4.0, strength=0.05, seed=3)
    run_attention([333], new, 4, 2, 128, 64, dtype, wide=0.5, strength=20.0, seed=4)
    run_attention([200], new, 4, 2, 128, 64, dtype, strength=1e-30, seed=5)  # every weight alike
    run_attention([200], new, 4, 2, 128, 64, dtype, scale=-0.3, seed=6)
    run_attention([200], new, 4, 2, 128, 64, dtype, scale=0.0, seed=7)


@gpu
@pytest.mark.parametrize("new", [1, 3, 40])
def test_what_lies_behind_the_last_token_and_in_other_pages_is_not_read_as_a_number(new):
    """Slots behind the last token hold e4m3's NaN, their blocks and all other pages scales of NaN."""
    lengths, page, dim = [53, 0, 64], 32, 128
    lengths[2] = max(lengths[2], new)
    table, count = table_of(lengths, page, 3, width=5)
    gen = torch.Generator().manual_seed(9)
    pages = random_pages(count, 2, page, dim, gen)
    spoiled = copy_of(pages)
    live = torch.zeros(count, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for i in range(n):
            live[int(table[b, i // page]), i % page] = True
    for t in (spoiled.keys, spoiled.values):
        t.view(torch.uint8)[~live[:, None, :, None].expand(t.shape)] = 0x7F
    blocks = live.view(count, page // 16, 16).any(-1)
    for s in (spoiled.key_scales, spoiled.value_scales):
        s[~blocks[:, None].expand(s.shape)] = math.nan
    q = torch.randn(3, 4, new, dim, generator=gen).to(torch.bfloat16)
    args = (torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    out = paged_attention_fp8(q.to(DEV), to_gpu(spoiled), *args, mask="causal")
    check_attention(out, q, pages, table, lengths, True, dim**-0.5, torch.bfloat16)


@gpu
@pytest.mark.parametrize("new", [2, 48, 130])
@pytest.mark.parametrize("side", ["key_scales", "value_scales"])
def test_a_block_that_is_no_number_reaches_the_rows_that_see_it_and_no_others(new, side):
    n, page, dim = 200, 16, 128
    table, count = table_of([n], page, 1)
    gen = torch.Generator().manual_seed(2)
    pages = random_pages(count, 1, page, dim, gen)
    bad = (n - new // 2 - 1) // 16  # the block of a token amid the new ones
    spoiled = copy_of(pages)
    getattr(spoiled, side)[int(table[0, bad])] = math.nan
    q = torch.randn(1, 4, new, dim, generator=gen).to(torch.bfloat16)
    out = paged_attention_fp8(q.to(DEV), to_gpu(spoiled), torch.from_numpy(table).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), mask="causal").cpu()
    first = max(bad * 16 - (n - new), 0)  # new tokens from here on see the block
    assert torch.isnan(out[:, :, first:]).all()
    if first:
        good = paged_attention_fp8(q.to(DEV), to_gpu(pages), torch.from_numpy(table).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), mask="causal").cpu()
        assert torch.equal(out[:, :, :first], good[:, :, :first])


@gpu
@pytest.mark.parametrize("new", [1, 20])
def test_a_query_that_is_no_number_spoils_its_own_row(new):
    table, count = table_of([100], 16, 1)
    gen = torch.Generator().manual_seed(2)
    pages = to_gpu(random_pages(count, 2, 16, 64, gen))
    q = torch.randn(1, 4, new, 64, generator=gen).to(torch.bfloat16).to(DEV)
    args = (pages, torch.from_numpy(table).to(DEV), torch.tensor([100], dtype=torch.int32, device=DEV))
    good = paged_attention_fp8(q, *args, mask="causal")
    q[0, 1, 0, 3] = math.nan
    out = paged_attention_fp8(q, *args, mask="causal")
    assert torch.isnan(out[0, 1, 0]).all()
    keep = torch.ones(out.shape[:3], dtype=torch.bool, device=DEV)
    keep[0, 1, 0] = False
    assert torch.equal(out[keep], good[keep])


@gpu
def test_answers_are_the_same_every_time():
    for lengths, new in (([3000, 17, 900], 1), ([1500], 100)):
        table, count = table_of(lengths, 64, 1)
        gen = torch.Generator().manual_seed(2)
        pages = to_gpu(random_pages(count, 2, 64, 128, gen))
        q = torch.randn(len(lengths), 8, new, 128, generator=gen).to(torch.bfloat16).to(DEV)
        args = (pages, torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
        first = paged_attention_fp8(q, *args, mask="causal")
        for _ in range(5):
            assert torch.equal(first, paged_attention_fp8(q, *args, mask="causal"))


@gpu
def test_a_long_cache_whose_offsets_pass_32_bits():
    """Pages of 2^31 and more numbers a side: only the last ones are used."""
    page, heads, dim, count = 128, 8, 128, 2**31 // (128 * 8 * 128) + 3
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    pages = Fp8KvPages.zeros(count, heads, page, dim)
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(1, h, 150, dim, generator=gen).to(torch.bfloat16).to(DEV) for h in (8, 8, 8))
    table = torch.tensor([[count - 1, count - 2]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([150], dtype=torch.int32, device=DEV)
    small = Fp8KvPages.zeros(2, heads, page, dim)
    there = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    rope = FastRoPE(dim, 4096, BASE)
    a, b = rotate_append_fp8(q, k, v, pages, table, lens, rope=rope), rotate_append_fp8(q, k, v, small, there, lens, rope=rope)
    assert torch.equal(a, b)
    assert torch.equal(pages.keys[-2:].view(torch.uint8), small.keys.view(torch.uint8)) and not pages.keys[:-2].view(torch.uint8).any()
    for rows in (a, a[:, :, -1:]):
        assert torch.equal(paged_attention_fp8(rows, pages, table, lens, mask="causal"), paged_attention_fp8(rows, small, there, lens, mask="causal"))


# ---- both in a row ----------------------------------------------------------------------------------------------------


def steps(pages, plan, seed, heads=8, dim=128, run=None):
    """Portions and single tokens of three requests: append, attend.  -> outputs and the tokens' rows by request."""
    gen = torch.Generator().manual_seed(seed)
    table_host = np.arange(3 * 8, dtype=np.int32).reshape(3, 8)
    outs, lens = [], [0, 0, 0]
    rope, norm = FastRoPE(dim, 4096, BASE), FastRMSNorm(dim, torch.ones(dim, device=DEV), eps=1e-6)
    for rows, new in plan:
        q, k, v = (torch.randn(3, h, new, dim, generator=gen).to(torch.bfloat16).to(DEV) for h in (heads, pages.kv_heads, pages.kv_heads))
        here = [n + new if i in rows else 0 for i, n in enumerate(lens)]
        lens = [h or n for h, n in zip(here, lens)]
        t = np.where(np.arange(8)[None] < -(-np.asarray(here)[:, None] // pages.page_size), table_host, -1).astype(np.int32)
        kw = dict(block_table_host=t, context_lens_host=np.asarray(here, dtype=np.int32))
        table, ctx = torch.from_numpy(t).to(DEV), torch.tensor(here, dtype=torch.int32, device=DEV)
        q = rotate_append_fp8(q, k, v, pages, table, ctx, rope=rope, query_norm=norm, key_norm=norm, **kw)
        outs.append((q.cpu(), paged_attention_fp8(q, pages, table, ctx, mask="causal", **kw), t, here, new))
    return outs


@gpu
def test_a_run_of_appends_and_attention_as_a_scheduler_makes_it():
    pages = Fp8KvPages.zeros(24, 2, 64, 128)
    plan = [((0,), 100), ((1,), 37), ((0, 1), 1), ((2,), 130), ((0, 1, 2), 1), ((0, 1, 2), 1), ((0, 2), 4), ((1,), 64), ((0, 1, 2), 1)]
    for q, out, table, lens, _ in steps(pages, plan, 3):
        pass
    # the last step's answers against the cache as it is now (nothing was appended behind it)
    check_attention(out, q, Fp8KvPages(*(t.cpu() for t in (pages.keys, pages.values, pages.key_scales, pages.value_scales))), table, lens, True, 128**-0.5, torch.bfloat16)


@gpu
def test_on_another_stream_and_in_a_replayed_graph():
    dim, page = 128, 64
    gen = torch.Generator().manual_seed(5)
    make = lambda h: torch.randn(2, h, 1, dim, generator=gen).to(torch.bfloat16).to(DEV)  # noqa: E731
    q, k, v = make(8), make(2), make(2)
    start = to_gpu(random_pages(8, 2, page, dim, gen))
    table_host, rope = np.arange(8, dtype=np.int32).reshape(2, 4), FastRoPE(dim, 4096, BASE)
    table = torch.from_numpy(table_host).to(DEV)

    def step(pages, lens):
        kw = dict(block_table_host=np.where(np.arange(4)[None] < np.asarray([[4], [4]]), table_host, -1).astype(np.int32), context_lens_host=np.asarray([250, 250], dtype=np.int32))
        x = rotate_append_fp8(q, k, v, pages, table, lens, rope=rope, **kw)
        return paged_attention_fp8(x, pages, table, lens, mask="causal", **kw)

    want = []
    plain = copy_of(start)
    for n in (199, 200, 201, 210):
        want.append(step(plain, torch.tensor([n, n + 30], dtype=torch.int32, device=DEV)).clone())
    other = copy_of(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [step(other, torch.tensor([n, n + 30], dtype=torch.int32, device=DEV)) for n in (199, 200, 201, 210)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    third, lens = copy_of(start), torch.tensor([199, 229], dtype=torch.int32, device=DEV)
    spare = copy_of(start)
    step(spare, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(third, lens)
    for n, w in zip((199, 200, 201, 210), want):
        lens.copy_(torch.tensor([n, n + 30], dtype=torch.int32, device=DEV))
        graph.replay()
        assert torch.equal(out, w), n
    assert torch.equal(third.keys.view(torch.uint8), plain.keys.view(torch.uint8))
