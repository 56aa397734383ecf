"""Attention over pages of 8 bits whose blocks' scales lie far apart: a key that a row does not see, or that weighs nothing, takes nothing from its answer, whatever its size.

The bound counts, for every row, the keys that it sees.  bf16 outputs; p: a key's weight, v: its value, raw: its number without the block's scale.
  - A score is a sum of D exact products, added up in steps of 16, and as many products with fp32 factors: (D / 16 + 6) 2^-22 of sum |q k| scale.  exp2 and the sums: 2^-20 together.
  - A weight is rounded to f16: half a step, 2^-11 of itself, or 2^-25 of the row's largest where it is among the smallest (never by more than all of it).  Ahead of the rounding it may be multiplied by the
    block's scale over one up to 16 times as large (then 2^-21 of the largest weight), or over one of which it is at least 2^-80 (then 2^-105 of the largest p * scale, for each unit of raw).
  - The sum that divides is of the weights before that rounding.  The output is rounded to bf16."""

import math

import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks
from tests.test_gpu_fp8_cache import random_pages, table_of, to_gpu
from tiny_llm_b200 import paged_attention_fp8

DEV = "cuda"
pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def dense(pages, table, n):
    """Numbers and scales of a request in its order: [H, n, D] and [H, n], twice."""
    homes = [int(p) for p in table[: -(-n // pages.page_size)]]
    out = []
    for numbers, scales in ((pages.keys, pages.key_scales), (pages.values, pages.value_scales)):
        out += [numbers.float().double()[homes].transpose(0, 1).flatten(1, 2)[:, :n], scales.double()[homes].transpose(0, 1).flatten(1, 2).repeat_interleave(16, 1)[:, :n]]
    return out


def check(out, q, pages, table, lengths, causal=True, rows=None):
    new, dim = q.shape[2:]
    group = q.shape[1] // pages.kv_heads
    worst = 0.0
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[b].any()
            continue
        k_raw, k_s, v_raw, v_s = dense(pages, table[b], n)
        of = torch.arange(new) if rows is None else torch.as_tensor(rows)
        hidden = torch.arange(n)[None] > (of + n - new)[:, None] if causal else torch.zeros(len(of), n, dtype=torch.bool)
        for h in range(q.shape[1]):
            g = h // group
            k, v, x = k_raw[g] * k_s[g][:, None], v_raw[g] * v_s[g][:, None], q[b, h, of].double()
            s = (x @ k.t() * dim**-0.5).masked_fill(hidden, -math.inf)
            p = torch.softmax(s, -1)
            want = p @ v
            d = (dim / 16 + 6) * 2.0**-22 * (x.abs() @ k.abs().t() * dim**-0.5) + 2.0**-20
            tol = (p * (d + 2.0**-11)) @ v.abs() + (p * d).sum(-1, keepdim=True) * want.abs()
            size = p * v_s[g]
            tol += torch.minimum(2.0**-21 * p.amax(-1, keepdim=True), p) @ v.abs() + torch.minimum(2.0**-105 * size.amax(-1, keepdim=True), size) @ v_raw[g].abs()
            tol += 2.0**-8 * 1.01 * want.abs() + 1e-37
            got = out[b, h, of].cpu().double()
            far = (got - want).abs() / tol
            assert (far <= 1).all(), (b, h, [int(i) for i in (far > 1).any(-1).nonzero()[:8, 0]], float(far.max()))
            worst = max(worst, float(far.max()))
    return worst


def attend(q, pages, table, lengths, causal=True):
    return paged_attention_fp8(q.to(DEV), to_gpu(pages), torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), mask="causal" if causal else None)


def scale_block(pages, table, token, e, side="value_scales"):
    """The scale of the block of a request's token: 2^e."""
    page = pages.page_size
    getattr(pages, side)[int(table[token // page]), :, token % page // 16] = 2.0**e


PORTIONS = [  # lengths, new, heads, kv_heads, dim, page: whole items and pieces, groups of which a CTA holds many tokens or few
    ([400, 400, 400], 400, 16, 2, 128, 128), ([600, 0, 401], 400, 16, 2, 64, 48), ([1300], 700, 4, 4, 128, 64), ([1500], 300, 32, 2, 128, 16), ([700], 64, 8, 1, 64, 64), ([2500], 130, 16, 2, 128, 128),
]


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim,page", PORTIONS)
@pytest.mark.parametrize("side", ["key_scales", "value_scales"])
@pytest.mark.parametrize("apart", [14, 15, 16, 25, 26, 40, 90])
def test_a_portions_rows_that_do_not_see_a_large_block(lengths, new, heads, kv_heads, dim, page, side, apart):
    """The last tokens, and some in the middle of the new ones, have a scale 2^apart times everybody else's."""
    gen = torch.Generator().manual_seed(apart + dim)
    table, count = table_of(lengths, page, 2)
    pages = random_pages(count, kv_heads, page, dim, gen, wide=0.0)
    q = (0.5 * torch.randn(len(lengths), heads, new, dim, generator=gen)).to(BF16)
    low = -6 if apart < 80 else -60
    getattr(pages, side).fill_(2.0**low)
    for b, n in enumerate(lengths):
        if n:
            for token in (n - 1, n - new // 2):
                scale_block(pages, table[b], token, low + apart, side)
    check(attend(q, pages, table, lengths), q, pages, table, lengths, rows=[i for i in range(0, new, 1 + new // 60)] + [new // 2 - 17, new // 2, new - 1])


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim,page", PORTIONS)
@pytest.mark.parametrize("wide", [4.0, 12.0, 30.0])
def test_portions_over_scales_of_every_size(lengths, new, heads, kv_heads, dim, page, wide):
    gen = torch.Generator().manual_seed(int(wide) + dim)
    table, count = table_of(lengths, page, 3)
    pages = random_pages(count, kv_heads, page, dim, gen, wide=0.0)
    pages.value_scales.copy_(torch.exp2(torch.round(wide * torch.randn(pages.value_scales.shape, generator=gen)).clamp(-99, 99)))
    pages.key_scales.copy_(torch.exp2(torch.round(wide / 8 * torch.randn(pages.key_scales.shape, generator=gen) - 8 - wide / 8).clamp(-99, 9)))
    q = (0.5 * torch.randn(len(lengths), heads, new, dim, generator=gen)).to(BF16)
    for causal in (True, False):
        check(attend(q, pages, table, lengths, causal), q, pages, table, lengths, causal, rows=list(range(0, new, 1 + new // 50)) + [new - 1])


def weightless(pages, table, token, e):
    """A token whose score is far below all others (the queries' first entry is positive), with a value of scale 2^e and nothing beside it in its block."""
    page = pages.page_size
    home, slot = int(table[token // page]), token % page
    pages.values.view(torch.uint8)[home, :, slot // 16 * 16 : slot // 16 * 16 + 16] = 0
    pages.values[home, :, slot] = torch.linspace(-448, 448, pages.head_dim).to(torch.float8_e4m3fn)
    pages.value_scales[home, :, slot // 16] = 2.0**e
    pages.keys.view(torch.uint8)[home, :, slot] = 0
    pages.keys.view(torch.uint8)[home, :, slot, 0] = 0xFE  # -448
    pages.key_scales[home, :, slot // 16] = 1.0
    for other in range(slot // 16 * 16, slot // 16 * 16 + 16):  # the keys beside it stay about as large as all others
        if other != slot:
            pages.keys[home, :, other] = (pages.keys[home, :, other].float() / 64).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim,page", PORTIONS[:4])
@pytest.mark.parametrize("e", [8, 20, 90])
def test_a_portions_visible_key_without_weight(lengths, new, heads, kv_heads, dim, page, e):
    gen = torch.Generator().manual_seed(e + dim)
    table, count = table_of(lengths, page, 4)
    pages = random_pages(count, kv_heads, page, dim, gen, wide=0.0)
    pages.value_scales.fill_(2.0**-9)
    q = (0.5 * torch.randn(len(lengths), heads, new, dim, generator=gen)).to(BF16)
    q[..., 0] = 16.0
    for b, n in enumerate(lengths):
        for token in (3, n // 3, n - 40) if n else ():
            weightless(pages, table[b], token, e)
    check(attend(q, pages, table, lengths), q, pages, table, lengths, rows=list(range(0, new, 1 + new // 40)) + [new - 1])


ROWS = [  # lengths, new, heads, kv_heads, dim: one item, clusters, whole items, pieces; 8 and 16 columns; every form of a head
    ([100], 1, 8, 2, 128), ([1011], 1, 32, 8, 128), ([700] * 30, 1, 8, 8, 128), ([9000], 1, 8, 2, 128), ([5000, 16, 0, 40], 1, 8, 8, 64), ([300, 90], 4, 8, 2, 128), ([3000], 4, 8, 4, 64), ([260, 77], 3, 6, 2, 96),
    ([400], 2, 4, 2, 256), ([120], 5, 10, 2, 80),
]


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim", ROWS)
@pytest.mark.parametrize("apart", [3, 4, 5, 14, 20, 25, 40, 100])
def test_a_decoded_tokens_visible_key_without_weight(lengths, new, heads, kv_heads, dim, apart):
    gen = torch.Generator().manual_seed(apart + dim)
    table, count = table_of(lengths, 32, 4)
    pages = random_pages(count, kv_heads, 32, dim, gen, wide=0.0)
    low = -9 if apart < 90 else -60
    pages.value_scales.fill_(2.0**low)
    q = (0.5 * torch.randn(len(lengths), heads, new, dim, generator=gen)).to(BF16)
    q[..., 0] = 16.0
    for b, n in enumerate(lengths):
        for token in (0, n // 3, n - 20) if n > 40 else (n - 1,) if n else ():  # the first, one in the middle, one near the end
            weightless(pages, table[b], token, low + apart)
    check(attend(q, pages, table, lengths), q, pages, table, lengths)


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim", [r for r in ROWS if r[1] > 1])
@pytest.mark.parametrize("side", ["key_scales", "value_scales"])
@pytest.mark.parametrize("apart", [4, 5, 16, 26, 40, 100])
def test_few_tokens_that_do_not_see_a_large_block(lengths, new, heads, kv_heads, dim, side, apart):
    """The last new token begins a block, whose scale is 2^apart times the others'."""
    lengths = [n - n % 16 + 1 if n else 0 for n in lengths]
    gen = torch.Generator().manual_seed(apart + dim)
    table, count = table_of(lengths, 32, 5)
    pages = random_pages(count, kv_heads, 32, dim, gen, wide=0.0)
    low = -6 if apart < 90 else -60
    getattr(pages, side).fill_(2.0**low)
    for b, n in enumerate(lengths):
        if n:
            scale_block(pages, table[b], n - 1, low + apart, side)
    q = (0.5 * torch.randn(len(lengths), heads, new, dim, generator=gen)).to(BF16)
    check(attend(q, pages, table, lengths), q, pages, table, lengths)


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim", ROWS)
@pytest.mark.parametrize("wide", [2.0, 10.0, 30.0])
def test_few_tokens_over_scales_of_every_size(lengths, new, heads, kv_heads, dim, wide):
    gen = torch.Generator().manual_seed(int(wide) + dim)
    table, count = table_of(lengths, 32, 6)
    pages = random_pages(count, kv_heads, 32, dim, gen, wide=0.0)
    pages.value_scales.copy_(torch.exp2(torch.round(wide * torch.randn(pages.value_scales.shape, generator=gen)).clamp(-99, 99)))
    q = (0.5 * torch.randn(len(lengths), heads, new, dim, generator=gen)).to(BF16)
    check(attend(q, pages, table, lengths), q, pages, table, lengths)


def test_nobody_gave_up():
    assert blocks.library().tlb_tc_gave_up() == 0
