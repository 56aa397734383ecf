"""Portions and decoded tokens over scales far apart, at the edges: numbers that are none, pages that are none, captured calls, requests of many blocks, scales of the scores of 0 and below."""

import math

import numpy as np
import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks
from tests.test_gpu_fp8_cache import random_pages, table_of, to_gpu
from tests.test_gpu_fp8_cache_far_scales import BF16, attend, check, scale_block
from tiny_llm_b200 import Fp8KvPages, paged_attention_fp8

DEV = "cuda"
pytestmark = pytest.mark.gpu


def far_pages(gen, count, kv_heads, page, dim, wide=12.0):
    pages = random_pages(count, kv_heads, page, dim, gen, wide=0.0)
    pages.value_scales.copy_(torch.exp2(torch.round(wide * torch.randn(pages.value_scales.shape, generator=gen)).clamp(-60, 60)))
    return pages


@pytest.mark.parametrize("lengths,new", [((1300, 700), 400), ((600, 401), 400), ((301, 150), 3)])
def test_numbers_that_are_none_reach_the_rows_that_see_them(lengths, new):
    page, dim = 64, 128
    gen = torch.Generator().manual_seed(11)
    table, count = table_of(lengths, page, 6)
    pages = far_pages(gen, count, 2, page, dim)
    q = torch.randn(2, 16, new, dim, generator=gen).to(BF16)
    first_bad = [lengths[0] - new // 2, lengths[1] - 1]
    for b, (n, token) in enumerate(zip(lengths, first_bad)):
        home, at = int(table[b, token // page]), token % page // 16
        (pages.key_scales if b else pages.value_scales)[home, 1, at] = math.nan
        home, slot = int(table[b, n // page]) if n % page else -1, n % page
        if home >= 0:
            pages.keys.view(torch.uint8)[home, :, slot:] = 0x7F
            pages.values.view(torch.uint8)[home, :, slot:] = 0xFF
            pages.key_scales[home, :, (slot + 15) // 16 :] = math.nan
            pages.value_scales[home, :, (slot + 15) // 16 :] = math.nan
    q[0, 3, 1, 5], q[1, 9, new - 1, 100] = math.inf, math.nan
    out = attend(q, pages, table, lengths).cpu()
    none = torch.zeros(2, 16, new, dtype=torch.bool)
    none[0, 3, 1] = none[1, 9, new - 1] = True
    for b, (n, token) in enumerate(zip(lengths, first_bad)):
        none[b, 8:, torch.arange(n - new, n) >= token // 16 * 16] = True
    assert torch.equal(out.isnan().any(-1), none) and torch.equal(out.isnan().all(-1), none)
    fine = Fp8KvPages(pages.keys, pages.values, torch.nan_to_num(pages.key_scales, nan=0.0), torch.nan_to_num(pages.value_scales, nan=0.0))
    fine.keys.view(torch.uint8)[(pages.keys.view(torch.uint8) & 0x7F) == 0x7F] = 0
    fine.values.view(torch.uint8)[(pages.values.view(torch.uint8) & 0x7F) == 0x7F] = 0
    calm = q.clone()
    calm[0, 3, 1, 5] = calm[1, 9, new - 1, 100] = 0.0
    again = attend(calm, fine, table, lengths).cpu()
    assert torch.equal(out[~none], again[~none])
    assert torch.equal(again, attend(calm, fine, table, lengths).cpu())


@pytest.mark.parametrize("new,n", [(600, 1500), (2, 900)])
def test_pages_that_are_none_hide_their_keys(new, n):
    page, dim = 32, 128
    table, count = table_of([n], page, 3)
    gen = torch.Generator().manual_seed(4)
    pages = far_pages(gen, count, 2, page, dim, wide=6.0)
    bad = table.copy()
    bad[0, 2], bad[0, 20] = -1, count + 7
    q = (0.5 * torch.randn(1, 16, new, dim, generator=gen)).to(BF16)
    gp = to_gpu(pages)
    out = blocks.fp8_attention(gp.native, gp.index, q.to(DEV), torch.from_numpy(bad).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), dim**-0.5, True).cpu().double()
    homes = [int(p) for p in table[0]]
    k = (pages.keys.float().double()[homes] * pages.key_scales.double()[homes].repeat_interleave(16, -1)[..., None]).transpose(0, 1).flatten(1, 2)[:, :n]
    v = (pages.values.float().double()[homes] * pages.value_scales.double()[homes].repeat_interleave(16, -1)[..., None]).transpose(0, 1).flatten(1, 2)[:, :n]
    hidden = torch.zeros(n, dtype=torch.bool)
    hidden[2 * page : 3 * page], hidden[20 * page : 21 * page] = True, True
    for h in range(0, 16, 5):
        x = q[0, h].double()
        s = (x @ k[h // 8].t() * dim**-0.5).masked_fill(hidden[None] | (torch.arange(n)[None] > torch.arange(n - new, n)[:, None]), -math.inf)
        p = torch.softmax(s, -1)
        want = p @ v[h // 8]
        # scores: 14 x 2^-22 of sum |q k|; weights: 2^-11 of themselves, 2^-21 of the largest; the output's rounding
        d = 2.0**-18 * (x.abs() @ k[h // 8].abs().t() * dim**-0.5) + 2.0**-20
        tol = (p * (d + 2.0**-11)) @ v[h // 8].abs() + (p * d).sum(-1, keepdim=True) * want.abs() + torch.minimum(2.0**-21 * p.amax(-1, keepdim=True), p) @ v[h // 8].abs() + 2.0**-8 * 1.01 * want.abs()
        assert ((out[0, h] - want).abs() <= tol).all(), h


@pytest.mark.parametrize("new,heads,kv_heads,dim", [(512, 16, 2, 64), (130, 16, 2, 128), (3, 8, 2, 128), (1, 8, 8, 64)])
def test_a_captured_call_follows_lengths_and_scales(new, heads, kv_heads, dim):
    """The same launches over scales that are near one another, far apart and near again."""
    page, width = 64, 40
    gen = torch.Generator().manual_seed(7)
    near = random_pages(2 * width, kv_heads, page, dim, gen, wide=0.5)
    far = far_pages(gen, 2 * width, kv_heads, page, dim, wide=10.0)
    pages = to_gpu(near)
    table = np.random.RandomState(1).permutation(2 * width).astype(np.int32).reshape(2, width)
    q = (0.5 * torch.randn(2, heads, new, dim, generator=gen)).to(BF16)
    gq, gt, lens = q.to(DEV), torch.from_numpy(table).to(DEV), torch.tensor([600, 512], dtype=torch.int32, device=DEV)
    full = dict(block_table_host=table, context_lens_host=np.asarray([width * page] * 2, dtype=np.int32))
    paged_attention_fp8(gq, pages, gt, lens, mask="causal", **full)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention_fp8(gq, pages, gt, lens, mask="causal", **full)
    for which, lengths in ((near, [600, 512]), (far, [600, 512]), (far, [2560, 0]), (near, [2560, 700]), (far, [530, 2500])):
        for to, t in zip((pages.keys, pages.values, pages.key_scales, pages.value_scales), (which.keys, which.values, which.key_scales, which.value_scales)):
            to.copy_(t)
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(out, q, which, table, lengths, rows=list(range(0, new, 1 + new // 40)) + [new - 1])
    assert blocks.library().tlb_tc_gave_up() == 0


@pytest.mark.parametrize("apart", [20, 60])
def test_more_blocks_than_a_cta_has_threads(apart):
    """One block far above all others among some 800: scales are looked over in several rounds."""
    new, page, dim, n = 2500, 128, 64, 13_500
    gen = torch.Generator().manual_seed(9)
    table, count = table_of([n, 70], page, 1)
    pages = random_pages(count, 4, page, dim, gen, wide=1.0)
    scale_block(pages, table[0], 13_000, apart - 5)
    q = (0.5 * torch.randn(1, 40, new, dim, generator=gen)).to(BF16)
    out = attend(q, pages, table[:1], [n])
    for g in (0, 3):
        part = Fp8KvPages(*(t[:, g : g + 1].contiguous() for t in (pages.keys, pages.values, pages.key_scales, pages.value_scales)))
        check(out[:, 10 * g : 10 * g + 3], q[:, 10 * g : 10 * g + 3], part, table[:1], [n], rows=list(range(0, 20)) + list(range(1980, 2020)) + list(range(2490, 2500)))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30])
@pytest.mark.parametrize("new", [300, 3])
def test_other_scales_of_the_scores(new, scale):
    page, dim, n = 64, 128, 700
    gen = torch.Generator().manual_seed(3)
    table, count = table_of([n], page, 2)
    pages = far_pages(gen, count, 2, page, dim, wide=8.0)
    q = (0.5 * torch.randn(1, 16, new, dim, generator=gen)).to(BF16)
    out = paged_attention_fp8(q.to(DEV), to_gpu(pages), torch.from_numpy(table).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), scale=scale, mask="causal")
    if scale < 0:  # the same as queries turned around
        same = paged_attention_fp8((-q).to(DEV), to_gpu(pages), torch.from_numpy(table).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), scale=-scale, mask="causal")
        assert torch.equal(out, same)
    else:  # every weight alike
        check(out, torch.zeros_like(q), pages, table, [n], rows=list(range(0, new, 1 + new // 40)))


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim", [([1011], 1, 32, 8, 128), ([5000, 16, 0, 40], 1, 8, 8, 64), ([300, 90], 40, 8, 2, 128), ([260, 77], 3, 6, 2, 96), ([400], 2, 4, 2, 256)])
@pytest.mark.parametrize("wide", [10.0, 30.0])
def test_fp32_over_scales_of_every_size(lengths, new, heads, kv_heads, dim, wide):
    """Weights are two f16 terms, the second one 2^11 times what the first left: 2^-21 of a weight, 2^-36 of the largest; queries two such terms, 2^-21 of the row's largest entry with the rest.  Value scales
    are fp32 factors behind the products."""
    gen = torch.Generator().manual_seed(int(wide) + dim)
    table, count = table_of(lengths, 32, 6)
    pages = far_pages(gen, count, kv_heads, 32, dim, wide)
    q = 0.5 * torch.randn(len(lengths), heads, new, dim, generator=gen)
    out = attend(q, pages, table, lengths).cpu().double()
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[b].any()
            continue
        homes = [int(p) for p in table[b, : -(-n // 32)]]
        k, v = ((x.float().double()[homes] * s.double()[homes].repeat_interleave(16, -1)[..., None]).transpose(0, 1).flatten(1, 2)[:, :n] for x, s in ((pages.keys, pages.key_scales), (pages.values, pages.value_scales)))
        hidden = torch.arange(n)[None] > torch.arange(n - new, n)[:, None]
        for h in range(heads):
            g, x = h // (heads // kv_heads), q[b, h].double()
            p = torch.softmax((x @ k[g].t() * dim**-0.5).masked_fill(hidden, -math.inf), -1)
            want = p @ v[g]
            d = (dim / 16 + 6) * 2.0**-22 * (x.abs() @ k[g].abs().t() * dim**-0.5) + 2.0**-20
            tol = (p * (d + 2.0**-21)) @ v[g].abs() + (p * d).sum(-1, keepdim=True) * want.abs() + torch.minimum(2.0**-36 * p.amax(-1, keepdim=True), p) @ v[g].abs() + 2.0**-23 * want.abs()
            assert ((out[b, h] - want).abs() <= tol).all(), (b, h, float(((out[b, h] - want).abs() / tol).max()))
