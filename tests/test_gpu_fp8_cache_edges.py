"""Calls of the 8-bit cache at the edges of what its documentation allows: rows that begin anywhere, captured launches whose requests grow past the cut into pieces, pages that are
none, wide groups, far positions, two streams, idle slots.  Helpers and tolerances are those of the operators' own tests."""

import math

import numpy as np
import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks
from tests.test_gpu_fp8_cache import attention_tolerance, check_attention, check_side, copy_of, dense, on_host, random_pages, run_append, run_attention, table_of, to_gpu, turned
from tiny_llm_b200 import FastRMSNorm, FastRoPE, Fp8KvPages, paged_attention_fp8, rotate_append_fp8

DEV = "cuda"
pytestmark = pytest.mark.gpu


def odd_rows(x, pad=3):
    """The same tensor with rows that begin on any 2 (or 4) bytes."""
    wide = torch.zeros(*x.shape[:-1], x.shape[-1] + pad, dtype=x.dtype, device=x.device)
    wide[..., 1 : 1 + x.shape[-1]] = x
    return wide[..., 1 : 1 + x.shape[-1]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["tokens", "columns"])
def test_norms_of_keys_far_from_one(dtype, layout):
    def change(q, k, v):
        k[0, :, 0] *= 1e28
        k[0, 3, 1] *= 1e13
        k[1, :, 1] *= 1e-25

    for dim in (64, 144):
        run_append([40, 35], 20, 4, 2, dim, 16, dtype, change=change, layout=layout, seed=dim)


def test_norms_without_an_eps():
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(1, 1, 16, 64, generator=gen) * torch.exp2(torch.arange(-75.0, 69.0, 9.0))[:, None]
    pages = Fp8KvPages.zeros(1, 1, 16, 64)
    g = x.to(DEV)
    rotate_append_fp8(g, g, g, pages, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.full((1,), 16, dtype=torch.int32, device=DEV), key_norm=FastRMSNorm(64, torch.ones(64, device=DEV), eps=0.0))
    y = x[0].double()
    want = y / y.square().mean(-1, keepdim=True).sqrt()
    zero = torch.zeros(1, 1, 16, 64, dtype=torch.float64)
    check_side("keys", on_host(pages.keys), on_host(pages.key_scales), zero, torch.zeros(1, 1, 1, dtype=torch.float64), want[None], np.zeros((1, 1), dtype=np.int32), [16], 16, 16)


@pytest.mark.parametrize("new", [1, 5, 50])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_begin_anywhere(new, dtype):
    lengths, page, dim = [130, 0, 70], 32, 128
    table, count = table_of(lengths, page, 2)
    gen = torch.Generator().manual_seed(new)
    pages = random_pages(count, 2, page, dim, gen)
    q, k, v = (torch.randn(3, h, new, dim, generator=gen).to(dtype).to(DEV) for h in (8, 2, 2))
    args = (torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    even, odd = to_gpu(pages), to_gpu(pages)
    rope = FastRoPE(dim, 4096, 10000)
    a, b = rotate_append_fp8(q, k, v, even, *args, rope=rope), rotate_append_fp8(*(odd_rows(x) for x in (q, k, v)), odd, *args, rope=rope)
    # two kernels: the same definition, so the same numbers but where one lies next to a border
    assert torch.equal(even.values.view(torch.uint8), odd.values.view(torch.uint8)) and torch.equal(even.value_scales, odd.value_scales) and torch.equal(even.key_scales, odd.key_scales)
    assert (even.keys.view(torch.uint8) != odd.keys.view(torch.uint8)).float().mean() < 1e-4
    torch.testing.assert_close(a, b, rtol=2 * torch.finfo(dtype).eps, atol=2.0**-20)
    whole = paged_attention_fp8(q, even, *args, mask="causal")
    assert torch.equal(whole, paged_attention_fp8(odd_rows(q), even, *args, mask="causal"))  # the same kernel, read another way
    assert torch.equal(whole, paged_attention_fp8(q.transpose(1, 2).contiguous().transpose(1, 2), even, *args, mask="causal"))
    assert torch.equal(whole[:1], paged_attention_fp8(q[:1].expand(3, -1, -1, -1), even, *args, mask="causal")[:1])


@pytest.mark.parametrize("new,heads,kv_heads,dim,dtype", [(1, 8, 2, 128, torch.bfloat16), (1, 8, 2, 64, torch.float32), (3, 8, 2, 128, torch.bfloat16), (40, 4, 2, 128, torch.bfloat16), (33, 4, 2, 64, torch.bfloat16)])
def test_a_captured_call_follows_requests_past_the_cut(new, heads, kv_heads, dim, dtype):
    page, width = 64, 80
    gen = torch.Generator().manual_seed(7)
    pages_host = random_pages(2 * width, kv_heads, page, dim, gen)
    pages = to_gpu(pages_host)
    table = np.random.RandomState(1).permutation(2 * width).astype(np.int32).reshape(2, width)
    q = torch.randn(2, heads, new, dim, generator=gen).to(dtype)
    gq, gt, lens = q.to(DEV), torch.from_numpy(table).to(DEV), torch.tensor([60, 50], dtype=torch.int32, device=DEV)
    full = dict(block_table_host=table, context_lens_host=np.asarray([width * page] * 2, dtype=np.int32))  # any lengths are covered
    paged_attention_fp8(gq, pages, gt, lens, mask="causal", **full)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged_attention_fp8(gq, pages, gt, lens, mask="causal", **full)
    with torch.cuda.graph(side):
        other = paged_attention_fp8(gq, pages, gt, lens, mask="causal", **full)
    for lengths in ([60, 50], [5000, 77], [0, 4099], [1100, 1100], [5120, 5120], [new, 0]):
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay(), side.replay()
        torch.cuda.synchronize()
        check_attention(out, q, pages_host, table, lengths, True, dim**-0.5, dtype)
        assert torch.equal(out, other)


@pytest.mark.parametrize("lengths,new", [([5000], 1), ([4000, 16, 0, 1030], 1), ([4500, 20], 4), ([3000], 40), ([2500, 100], 70)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_requests_in_pieces(lengths, new, dtype):
    run_attention(lengths, new, 8, 2, 128, 64, dtype, seed=new)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_that_are_none_hide_their_keys(new):
    """Past the host's checks (a captured launch, another caller of the extension): entries outside the pages are not read."""
    page, dim, n = 32, 128, 300
    table, count = table_of([n], page, 3)
    gen = torch.Generator().manual_seed(4)
    pages = random_pages(count, 2, page, dim, gen)
    bad = table.copy()
    bad[0, 2], bad[0, 5] = -1, count + 7
    q = torch.randn(1, 8, new, dim, generator=gen).to(torch.bfloat16)
    gp = to_gpu(pages)
    out = blocks.fp8_attention(gp.native, gp.index, q.to(DEV), torch.from_numpy(bad).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), dim**-0.5, True)
    # the same with the hidden keys scored far below all others
    k, v = (torch.cat([x[int(p)] for p in table[0]], dim=1)[:, :n].double() for x in pages.dequantize())
    hidden = torch.zeros(n, dtype=torch.bool)
    hidden[2 * page : 3 * page], hidden[5 * page : 6 * page] = True, True
    keep = ~hidden
    for h in range(8):
        x = q[0, h].double()
        s = (x @ k[h // 4].t() * dim**-0.5).masked_fill(hidden[None] | (torch.arange(n)[None] > torch.arange(n - new, n)[:, None]), -torch.inf)
        want = torch.softmax(s, -1) @ v[h // 4]
        # as for attention among the keys that are left: weights off by 2^-12, scores by some 2^-18 of sums of |q k|, outputs by half a step of bf16
        most = (x.abs() @ k[h // 4].abs().t() * dim**-0.5).amax()
        tol = (2.0**-11 + 2.0**-18 * most) * (torch.softmax(s, -1) @ v[h // 4].abs() + want.abs()) + 2.0**-8 * want.abs() + 2.0**-16 * v[h // 4][keep].abs().amax(0)
        assert ((out[0, h].cpu().double() - want).abs() <= tol).all()
    x = torch.randn(1, 2, 40, dim, generator=gen).to(torch.bfloat16).to(DEV)
    before = copy_of(gp)
    turned_q = blocks.fp8_append(gp.native, gp.index, x, x, x, torch.full((1, 10), -1, dtype=torch.int32, device=DEV), torch.tensor([60], dtype=torch.int32, device=DEV))
    assert torch.equal(turned_q, x) and torch.equal(before.keys.view(torch.uint8), gp.keys.view(torch.uint8)) and torch.equal(before.key_scales, gp.key_scales)
    for lens in (39, -3, 10 * page + 1):  # shorter than the step, negative, past the table: as an idle slot
        zeros = blocks.fp8_append(gp.native, gp.index, x, x, x, torch.from_numpy(bad).to(DEV), torch.tensor([lens], dtype=torch.int32, device=DEV))
        assert not zeros.any() and torch.equal(before.keys.view(torch.uint8), gp.keys.view(torch.uint8))


@pytest.mark.parametrize("heads,kv_heads,dim,new", [(40, 1, 64, 1), (40, 1, 128, 7), (300, 1, 128, 1), (300, 1, 32, 2), (64, 2, 256, 3), (7, 7, 128, 41)])
def test_wide_groups(heads, kv_heads, dim, new):
    run_attention([90, 0, 17 + new], new, heads, kv_heads, dim, 16, torch.bfloat16, seed=heads)
    run_append([90, 0, 17 + new], new, heads, kv_heads, dim, 16, torch.bfloat16, seed=heads)


@pytest.mark.parametrize("page", [16, 1024, 4096, 2032])
def test_page_sizes(page):
    run_attention([3000, 31], 2, 4, 2, 64, page, torch.bfloat16, seed=page)
    run_attention([1500, 40], 40, 4, 2, 64, page, torch.bfloat16, seed=page)
    run_append([3000, 31], 20, 4, 2, 64, page, torch.bfloat16, seed=page)


@pytest.mark.parametrize("traditional", [False, True])
@pytest.mark.parametrize("rot", [128, 120])
def test_far_positions_turn_exactly(traditional, rot):
    """Angles of up to a million radians: 24 bits of a turn would be off by a tenth."""
    n, page, dim, new = 1_000_003, 4096, 128, 19
    pages = Fp8KvPages.zeros(245, 1, page, dim)
    table_host = np.arange(245, dtype=np.int32)[None]
    gen = torch.Generator().manual_seed(8)
    x = torch.randn(1, 1, new, dim, generator=gen).to(torch.bfloat16)
    g = x.to(DEV)
    out = rotate_append_fp8(g, g, g, pages, torch.from_numpy(table_host).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), rope=FastRoPE(rot, 4096, 10000, traditional=traditional))
    want = turned(x[0, 0], None, 0.0, rot, traditional, n - new)
    size = x[0, 0].double().abs().amax(-1, keepdim=True)
    assert ((out[0, 0].cpu().double() - want).abs() <= 2.0**-8 * 1.01 * want.abs() + 2.0**-20 * size).all()
    zero = torch.zeros(245, 1, page, dim, dtype=torch.float64)
    scales = torch.zeros(245, 1, page // 16, dtype=torch.float64)
    check_side("keys", on_host(pages.keys), on_host(pages.key_scales), zero, scales, want[None, None], table_host, [n], new, page)


def test_idle_slots_and_other_requests_do_not_change_an_answer():
    gen = torch.Generator().manual_seed(3)
    pages = to_gpu(random_pages(60, 2, 64, 128, gen))
    q = torch.randn(1, 8, 1, 128, generator=gen).to(torch.bfloat16).to(DEV)
    for n in (700, 3000):  # whole, in pieces
        row = torch.arange(48, dtype=torch.int32, device=DEV)
        row[-(-n // 64) :] = -1
        alone = paged_attention_fp8(q, pages, row[None], torch.tensor([n], dtype=torch.int32, device=DEV))
        idle = torch.full((5, 48), -1, dtype=torch.int32, device=DEV)
        idle[3] = row
        beside = paged_attention_fp8(q.expand(5, -1, -1, -1), pages, idle, torch.tensor([0, 0, 0, n, 0], dtype=torch.int32, device=DEV))
        assert torch.equal(beside[3], alone[0]) and not beside[[0, 1, 2, 4]].any()


def test_two_streams_at_once():
    gen = torch.Generator().manual_seed(6)
    runs = []
    for i, (n, new) in enumerate(((4000, 1), (2000, 64))):
        table, count = table_of([n], 64, i)
        pages = to_gpu(random_pages(count, 2, 64, 128, gen))
        q, k, v = (torch.randn(1, h, new, 128, generator=gen).to(torch.bfloat16).to(DEV) for h in (8, 2, 2))
        runs.append((q, k, v, pages, torch.from_numpy(table).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV)))

    def once(run):
        q, k, v, pages, table, lens = run
        x = rotate_append_fp8(q, k, v, pages, table, lens, rope=FastRoPE(128, 4096, 10000))
        return paged_attention_fp8(x, pages, table, lens, mask="causal")

    want = [once(r) for r in runs]  # appending the same tokens again leaves the same numbers
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(once(runs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i]) for i in range(2) for a in got[i])
    assert blocks.library().tlb_tc_gave_up() == 0


@pytest.mark.parametrize("batch,kv_heads", [(1, 1), (1, 8), (2, 8), (3, 8), (5, 8), (9, 8), (20, 8)])
@pytest.mark.parametrize("group,dim,dtype", [(4, 128, torch.bfloat16), (12, 64, torch.bfloat16), (2, 256, torch.bfloat16), (10, 80, torch.float32), (1, 256, torch.float32)])
def test_few_and_more_items(batch, kv_heads, group, dim, dtype):
    """Items that clusters of 8, 7 .. 2 CTAs share, and too many for that; lengths of less than a block a CTA, idle slots, and long ones beside them."""
    lengths = [(700, 0, 33, 16, 210, 5, 129, 1, 64, 300)[i % 10] for i in range(batch)]
    run_attention(lengths, 1, kv_heads * group, kv_heads, dim, 32, dtype, seed=batch + dim)


# ---- portions of so many columns that the 5th-generation tensor cores take them ------------------------------------------


def check_portion(out, q, pages, table, lengths, causal, scale):
    """A weight rounded to f16 (11 significant bits) is off by at most half a step, 2^-11 of itself, and the sum that divides is of the weights before: 2^-11 of sum(p |v|).  The
    shared bound counts 2^-12 of that and 2^-12 of the output, which is less where values cancel: 2^-12 of sum(p |v|) are added here.  Everything else is as there."""
    page, new = pages.page_size, q.shape[2]
    group = q.shape[1] // pages.kv_heads
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        k, v = dense(pages, table[b], n, page)
        for h in range(q.shape[1]):
            x, keys, values = q[b, h].double(), k[h // group], v[h // group]
            s = x @ keys.t() * scale
            if causal:
                s = s.masked_fill(torch.arange(n)[None] > torch.arange(n - new, n)[:, None], -math.inf)
            p = torch.softmax(s, dim=-1)
            want = p @ values
            tol = attention_tolerance(x, keys, values, p, scale, want, torch.bfloat16, q.shape[3]) + 2.0**-12 * (p @ values.abs())
            far = (out[b, h].cpu().double() - want).abs() - tol
            assert (far <= 0).all(), (b, h, float(far.max()), float(tol.mean()))


def run_portion(lengths, new, heads, kv_heads, dim, page, *, causal=True, seed=0, wide=1.0, strength=1.0):
    gen = torch.Generator().manual_seed(seed + 5)
    table, count = table_of(lengths, page, seed)
    pages = random_pages(count, kv_heads, page, dim, gen, wide)
    q = (strength * torch.randn(len(lengths), new, heads, dim, generator=gen)).to(torch.bfloat16).transpose(1, 2)
    out = paged_attention_fp8(q.to(DEV), to_gpu(pages), torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), mask="causal" if causal else None)
    check_portion(out, q, pages, table, lengths, causal, dim**-0.5)


@pytest.mark.parametrize("lengths", [(1300, 0, 700), (600, 0, 401), (400, 400, 400)])
@pytest.mark.parametrize("dim,page", [(128, 128), (64, 48), (128, 16)])
@pytest.mark.parametrize("causal", [True, False])
def test_portions_of_many_columns(lengths, dim, page, causal):
    run_portion(list(lengths), 400, 16, 2, dim, page, causal=causal, seed=dim + page, wide=3.0)


@pytest.mark.parametrize("group,new,n", [(1, 2500, 2600), (5, 517, 2000), (64, 70, 900), (3, 1001, 1001)])
def test_large_portions_of_other_groups(group, new, n):
    run_portion([n], new, 2 * group, 2, 128, 64, seed=group, strength=2.0)


@pytest.mark.parametrize("lengths", [(1300, 700), (600, 401)])
@pytest.mark.parametrize("strided", [False, True])
def test_a_large_portion_over_numbers_that_are_none(lengths, strided):
    """A scale that is none reaches the rows that see its block, a query that is none its own row; what lies behind the last token reaches nobody."""
    new, page, dim = 400, 64, 128
    gen = torch.Generator().manual_seed(11)
    table, count = table_of(lengths, page, 6)
    pages = random_pages(count, 2, page, dim, gen)
    q = torch.randn(2, 16, new, dim, generator=gen).to(torch.bfloat16)
    first_bad = [lengths[0] - 150, lengths[1] - 33]  # tokens in whose blocks a scale is none
    for b, (n, token) in enumerate(zip(lengths, first_bad)):
        home, at = int(table[b, token // page]), token % page // 16
        (pages.key_scales if b else pages.value_scales)[home, 1, at] = math.nan
        home, slot = int(table[b, n // page]) if n % page else -1, n % page
        if home >= 0:
            pages.keys.view(torch.uint8)[home, :, slot:] = 0x7F
            pages.values.view(torch.uint8)[home, :, slot:] = 0xFF
            pages.key_scales[home, :, (slot + 15) // 16 :] = math.nan
            pages.value_scales[home, :, (slot + 15) // 16 :] = math.nan
    q[0, 3, 17, 5], q[1, 9, 399, 100] = math.inf, math.nan
    gq = odd_rows(q.to(DEV)) if strided else q.to(DEV)
    out = paged_attention_fp8(gq, to_gpu(pages), torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), mask="causal").cpu()
    none = torch.zeros(2, 16, new, dtype=torch.bool)
    none[0, 3, 17] = none[1, 9, 399] = True
    for b, (n, token) in enumerate(zip(lengths, first_bad)):
        sees = torch.arange(n - new, n) >= token // 16 * 16
        none[b, 8:, sees] = True
    assert torch.equal(out.isnan().any(-1), none) and torch.equal(out.isnan().all(-1), none)
    # the others as if there were nothing of it
    fine = Fp8KvPages(pages.keys, pages.values, torch.nan_to_num(pages.key_scales, nan=0.0), torch.nan_to_num(pages.value_scales, nan=0.0))
    fine.keys.view(torch.uint8)[(pages.keys.view(torch.uint8) & 0x7F) == 0x7F] = 0
    fine.values.view(torch.uint8)[(pages.values.view(torch.uint8) & 0x7F) == 0x7F] = 0
    calm = q.clone()
    calm[0, 3, 17, 5] = calm[1, 9, 399, 100] = 0.0
    again = paged_attention_fp8(calm.to(DEV), to_gpu(fine), torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), mask="causal").cpu()
    assert torch.equal(out[~none], again[~none])


def test_a_large_portion_hides_pages_that_are_none():
    new, page, dim, n = 600, 32, 128, 1500
    table, count = table_of([n], page, 3)
    gen = torch.Generator().manual_seed(4)
    pages = random_pages(count, 2, page, dim, gen)
    bad = table.copy()
    bad[0, 2], bad[0, 40] = -1, count + 7
    q = torch.randn(1, 16, new, dim, generator=gen).to(torch.bfloat16)
    gp = to_gpu(pages)
    # any lengths are covered by so wide a table: the kernel is chosen for them
    out = blocks.fp8_attention(gp.native, gp.index, q.to(DEV), torch.from_numpy(bad).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), dim**-0.5, True).cpu().double()
    k, v = (torch.cat([x[int(p)] for p in table[0]], dim=1)[:, :n].double() for x in pages.dequantize())
    hidden = torch.zeros(n, dtype=torch.bool)
    hidden[2 * page : 3 * page], hidden[40 * page : 41 * page] = True, True
    for h in range(0, 16, 5):
        x = q[0, h].double()
        s = (x @ k[h // 8].t() * dim**-0.5).masked_fill(hidden[None] | (torch.arange(n)[None] > torch.arange(n - new, n)[:, None]), -torch.inf)
        p = torch.softmax(s, -1)
        want = p @ v[h // 8]
        most = (x.abs() @ k[h // 8].abs().t() * dim**-0.5).amax()
        tol = (2.0**-11 + 2.0**-18 * most) * (p @ v[h // 8].abs() + want.abs()) + 2.0**-8 * want.abs() + 2.0**-16 * v[h // 8][~hidden].abs().amax(0)
        assert ((out[0, h] - want).abs() <= tol).all()


def test_a_captured_large_portion_follows_its_lengths():
    new, page, dim, width = 512, 64, 64, 40
    gen = torch.Generator().manual_seed(7)
    pages_host = random_pages(2 * width, 2, page, dim, gen)
    pages = to_gpu(pages_host)
    table = np.random.RandomState(1).permutation(2 * width).astype(np.int32).reshape(2, width)
    q = torch.randn(2, 16, new, dim, generator=gen).to(torch.bfloat16)
    gq, gt, lens = q.to(DEV), torch.from_numpy(table).to(DEV), torch.tensor([600, 512], dtype=torch.int32, device=DEV)
    full = dict(block_table_host=table, context_lens_host=np.asarray([width * page] * 2, dtype=np.int32))
    graph = torch.cuda.CUDAGraph()
    paged_attention_fp8(gq, pages, gt, lens, mask="causal", **full)
    with torch.cuda.graph(graph):
        out = paged_attention_fp8(gq, pages, gt, lens, mask="causal", **full)
    for lengths in ([600, 512], [2560, 0], [513, 2500]):
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check_portion(out, q, pages_host, table, lengths, True, dim**-0.5)
    assert blocks.library().tlb_tc_gave_up() == 0


@pytest.mark.parametrize("batch", [20, 32, 33])
def test_unlike_requests_in_any_order(batch):
    """More items than SMs: requests are taken by their length, equal ones and idle slots among them."""
    lengths = [(5, 300, 0, 17, 300, 1, 64, 900)[(3 * i) % 8] for i in range(batch)]
    run_attention(lengths, 1, 32, 8, 64, 32, torch.bfloat16, seed=batch)


@pytest.mark.parametrize("bad", [None, 12_900, 13_400])
def test_a_large_portion_far_into_a_long_request(bad):
    """More blocks than a CTA has threads, so that scales are looked over in several rounds; one that is none among the last."""
    new, page, dim, n = 2500, 128, 64, 13_500
    gen = torch.Generator().manual_seed(9)
    table, count = table_of([n, 70], page, 1)
    pages = random_pages(count, 4, page, dim, gen, wide=2.0)
    if bad is not None:
        pages.value_scales[int(table[0, bad // page]), :, bad % page // 16] = math.nan
    q = torch.randn(1, 40, new, dim, generator=gen).to(torch.bfloat16)
    out = paged_attention_fp8(q.to(DEV), to_gpu(pages), torch.from_numpy(table[:1]).to(DEV), torch.tensor([n], dtype=torch.int32, device=DEV), mask="causal").cpu()
    sees = torch.arange(n - new, n) >= (n if bad is None else bad // 16 * 16)
    assert out[0, :, sees].isnan().all() and not out[0, :, ~sees].isnan().any()
    k, v = dense(pages, table[0], n, page)
    v = torch.nan_to_num(v, nan=0.0)
    for h in (0, 13, 39):
        for rows in (slice(0, 40), slice(1200, 1240), slice(2300, 2340)):
            rows = torch.arange(new)[rows][~sees[rows]]
            if not len(rows):
                continue
            x = q[0, h, rows].double()
            s = (x @ k[h // 10].t() * dim**-0.5).masked_fill(torch.arange(n)[None] > (rows + n - new)[:, None], -math.inf)
            p = torch.softmax(s, -1)
            want = p @ v[h // 10]
            tol = attention_tolerance(x, k[h // 10], v[h // 10], p, dim**-0.5, want, torch.bfloat16, dim) + 2.0**-12 * (p @ v[h // 10].abs())
            assert ((out[0, h, rows].double() - want).abs() <= tol).all()
