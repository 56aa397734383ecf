"""The paged cache of 8 bits without a GPU: what its entry points refuse, the pool's and the caches' bookkeeping, the model's wiring."""

import numpy as np
import pytest
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks
from tiny_llm_b200 import BatchingKvCache, FastRMSNorm, FastRoPE, Fp8KvPagedCache, Fp8KvPagedPool, Fp8KvPages, Qwen3ModelWeek3, fp8_cache, paged_attention_fp8, qwen3_week3, rotate_append_fp8
from tiny_llm_b200.paged_kv_cache import TinyKvPagedCache, TinyKvPagedPool
from tiny_llm_b200.synthetic import synthetic_qwen3

F8 = torch.float8_e4m3fn


def numbers(*shape):
    return torch.zeros(*shape, dtype=torch.uint8).view(F8)


@pytest.mark.parametrize("keys,values,ks,vs", [
    (torch.zeros(2, 2, 16, 32), numbers(2, 2, 16, 32), torch.ones(2, 2, 1), torch.ones(2, 2, 1)),
    (numbers(2, 2, 16, 32), numbers(2, 2, 32, 32), torch.ones(2, 2, 1), torch.ones(2, 2, 1)),
    (numbers(2, 2, 24, 32), numbers(2, 2, 24, 32), torch.ones(2, 2, 1), torch.ones(2, 2, 1)),
    (numbers(2, 2, 16, 24), numbers(2, 2, 16, 24), torch.ones(2, 2, 1), torch.ones(2, 2, 1)),
    (numbers(2, 2, 16, 272), numbers(2, 2, 16, 272), torch.ones(2, 2, 1), torch.ones(2, 2, 1)),
    (numbers(2, 2, 32, 32), numbers(2, 2, 32, 32), torch.ones(2, 2, 1), torch.ones(2, 2, 2)),
    (numbers(2, 2, 16, 32), numbers(2, 2, 16, 32), torch.ones(2, 2, 1, dtype=torch.float64), torch.ones(2, 2, 1)),
    (numbers(2, 16, 2, 32).transpose(1, 2), numbers(2, 16, 2, 32).transpose(1, 2), torch.ones(2, 2, 1), torch.ones(2, 2, 1)),
    (numbers(2 * 2 * 16 * 32 + 16).view(torch.uint8)[8 : 8 + 2048].view(F8).view(2, 2, 16, 32), numbers(2, 2, 16, 32), torch.ones(2, 2, 1), torch.ones(2, 2, 1)),
    (numbers(0, 2, 16, 32), numbers(0, 2, 16, 32), torch.ones(0, 2, 1), torch.ones(0, 2, 1)),
])
def test_pages_of_another_form_are_refused(keys, values, ks, vs):
    with pytest.raises(ValueError, match="Fp8KvPages"):
        Fp8KvPages(keys, values, ks, vs)


def test_sizes_of_new_pages():
    for bad in ((0, 2, 16, 32), (1, 2, 24, 32), (1, 2, 16, 8), (1, 2, 16, 512)):
        with pytest.raises(ValueError):
            Fp8KvPages.zeros(*bad, device="cpu")
    pages = Fp8KvPages.zeros(3, 2, 48, 80, device="cpu")
    assert pages.nbytes == 2 * (3 * 2 * 48 * 80 + 4 * 3 * 2 * 3)
    pages.keys.view(torch.uint8)[1, 0, 17, 3] = 0x38  # 1.0
    pages.key_scales[1, 0, 1] = 0.25
    assert pages.dequantize()[0][1, 0, 17, 3] == 0.25 and pages.dequantize([1])[0].sum() == 0.25


def step(B=2, heads=4, kv=2, L=3, D=32, dtype=torch.bfloat16):
    return tuple(torch.zeros(B, h, L, D, dtype=dtype) for h in (heads, kv, kv))


TABLE = torch.tensor([[0, 1], [2, -1]], dtype=torch.int32)
LENS = torch.tensor([20, 5], dtype=torch.int32)


def pages_of(n=4):
    return Fp8KvPages.zeros(n, 2, 16, 32, device="cpu")


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(2, 4, 3, 48, dtype=torch.bfloat16)), "head dimension"),
    (dict(q=torch.zeros(2, 3, 3, 32, dtype=torch.bfloat16)), "divisible"),
    (dict(q=torch.zeros(4, 3, 32, dtype=torch.bfloat16)), "4D"),
    (dict(q=torch.zeros(2, 4, 0, 32, dtype=torch.bfloat16)), "positive"),
    (dict(q=torch.zeros(2, 4, 3, 32, dtype=torch.float16)), "float32 or bfloat16"),
    (dict(table=TABLE.long()), "int32"),
    (dict(table=TABLE[0]), "2D int32"),
    (dict(lens=LENS.long()), "int32"),
    (dict(lens=LENS[:1]), "batch sizes"),
    (dict(table=TABLE[:1]), "batch sizes"),
    (dict(table=torch.tensor([[0, 0], [2, -1]], dtype=torch.int32), late=True), "aliased"),
    (dict(table=torch.tensor([[0, 9], [2, -1]], dtype=torch.int32), late=True), "outside physical"),
    (dict(table=torch.tensor([[0, 1], [2, 3]], dtype=torch.int32), late=True), "sentinel"),
    (dict(lens=torch.tensor([40, 5], dtype=torch.int32), late=True), "not covered"),
    (dict(lens=torch.tensor([20, 2], dtype=torch.int32), late=True), "at least query length"),
    (dict(lens=torch.tensor([-1, 5], dtype=torch.int32), late=True), "nonnegative"),
    (dict(hosts=dict(context_lens_host=np.array([20, 5, 1], dtype=np.int32))), "copies"),
    (dict(hosts=dict(block_table_host=np.array([[0, 1, -1], [2, -1, -1]], dtype=np.int32))), "copies"),
])
def test_steps_that_do_not_fit_are_refused_by_both(change, text, monkeypatch):
    q, k, v = step()
    table, lens, hosts = change.get("table", TABLE), change.get("lens", LENS), change.get("hosts", {})
    q = change.get("q", q)
    for call in (lambda p: paged_attention_fp8(q, p, table, lens, **hosts), lambda p: rotate_append_fp8(q, k, v, p, table, lens, **hosts)):
        pages = pages_of()
        if change.get("late"):  # found by the library, behind the check for a GPU: nothing is launched for any of them
            monkeypatch.setattr(blocks, "fp8_devices", lambda *a: None)
            monkeypatch.setattr(blocks, "_current_device", lambda: pages.index)
            monkeypatch.setattr(blocks, "_raw_stream", lambda device: 0)
            monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
        with pytest.raises(ValueError, match=text):
            call(pages)


def test_what_append_alone_refuses():
    q, k, v = step()
    args = (pages_of(), TABLE, LENS)
    for bad in ((k[:, :, :2], v[:, :, :2]), (k, v[..., :16]), (k[:, :1], v[:, :1])):
        with pytest.raises(ValueError, match="beside the query"):
            rotate_append_fp8(q, *bad, *args)
    with pytest.raises(ValueError, match="same dtype"):
        rotate_append_fp8(q, k.float(), v.float(), *args)
    with pytest.raises(RuntimeError, match="GPU-only"):  # everything is right: the device is not
        rotate_append_fp8(q, k, v, *args, rope=FastRoPE(32, 64), query_norm=FastRMSNorm(32, torch.ones(32)))


def test_masks_of_attention():
    q, _, _ = step()
    for mask in (torch.zeros(3, 20), "window"):
        with pytest.raises(NotImplementedError):
            paged_attention_fp8(q, pages_of(), TABLE, LENS, mask=mask)
    with pytest.raises(RuntimeError, match="GPU-only"):
        paged_attention_fp8(q, pages_of(), TABLE, LENS, mask="causal")


def test_the_extensions_own_entries_look_at_their_tensors():
    q, k, v = step()
    native = pages_of().native
    for bad in (dict(q=q[..., :16]), dict(k=k.float()), dict(v=v[:1]), dict(q=torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16)[..., ::2]), dict(table=TABLE.long()), dict(lens=LENS[:1]),
                dict(table=torch.zeros(2, 4, dtype=torch.int32)[:, ::2])):
        a = {**dict(q=q, k=k, v=v, table=TABLE, lens=LENS), **bad}
        with pytest.raises(RuntimeError):
            blocks.fp8_append(native, -1, a["q"], a["k"], a["v"], a["table"], a["lens"])
    with pytest.raises(RuntimeError, match="GPU-only"):
        blocks.fp8_attention(native, -1, q, TABLE, LENS, 1.0, True)


# ---- the C entries' own checks (no launch is reached) ------------------------------------------------------------------


def test_c_entries_refuse_sizes_and_pointers():
    import ctypes

    lib = blocks.library()
    pages = blocks.Fp8Pages(4096, 8192, 4096, 4096, 4, 2, 16, 32)
    call = lambda **k: blocks._FP8_ATTENTION.pack(*[{**dict(q=16, out=16, table=16, lens=16, qb=0, qh=0, ql=0, scale=1.0, B=1, H=4, L=1, pages=1, causal=1, dtype=2), **k}[n] for n in  # noqa: E731
                                                    ("q", "out", "table", "lens", "qb", "qh", "ql", "scale", "B", "H", "L", "pages", "causal", "dtype")])
    bad_pages = [blocks.Fp8Pages(0, 8192, 4096, 4096, 4, 2, 16, 32), blocks.Fp8Pages(4096, 8192, 4096, 4096, 4, 2, 24, 32), blocks.Fp8Pages(4096, 8192, 4096, 4096, 4, 2, 16, 8),
                 blocks.Fp8Pages(4096, 8192, 4096, 4096, 4, 2, 16, 512), blocks.Fp8Pages(4104, 8192, 4096, 4096, 4, 2, 16, 32), blocks.Fp8Pages(4096, 8192, 4096, 4096, 0, 2, 16, 32)]
    for p in bad_pages:
        assert lib.tlb_fp8_attention(ctypes.addressof(p), call(), None, None, None, 0, None) == -1
        assert lib.tlb_fp8_attention_workspace(ctypes.addressof(p), call(), None) == 0
    for bad in (dict(H=3), dict(H=0), dict(B=-1), dict(L=-1), dict(pages=0), dict(q=0), dict(out=0), dict(table=0), dict(lens=0)):
        assert lib.tlb_fp8_attention(ctypes.addressof(pages), call(**bad), None, None, None, 0, None) == -1, bad
    assert lib.tlb_fp8_attention(ctypes.addressof(pages), call(dtype=1), None, None, None, 0, None) == -2
    assert lib.tlb_fp8_attention(ctypes.addressof(pages), call(B=0, q=0), None, None, None, 0, None) == 0  # nothing to do
    long = blocks.Fp8Pages(4096, 8192, 4096, 4096, 4, 2, 128, 32)
    size = lib.tlb_fp8_attention_workspace(ctypes.addressof(long), call(pages=100), None)
    assert size > 0
    assert lib.tlb_fp8_attention(ctypes.addressof(long), call(pages=100), None, None, 4096, size - 1, None) == -3
    ints = lambda *v: np.array(v, dtype=np.int32).tobytes()  # noqa: E731
    many = blocks.Fp8Pages(4096, 8192, 4096, 4096, 100, 2, 128, 32)
    assert lib.tlb_fp8_attention(ctypes.addressof(many), call(pages=90), ints(128 * 90), ints(*range(90)), None, 0, None) == -3
    for lens, table in ((5, (4,)), (5, (-1,)), (20, (0,)), (-1, (0,)), (0, (0,))):  # outside, none, not covered, negative, an idle request's page
        assert lib.tlb_fp8_attention(ctypes.addressof(pages), call(), ints(lens), ints(*table), None, 0, None) == -1
    for lens, table in (((5, 5), (1, 1)), ((1, 2), (0, 1))):  # twice the same page, shorter than the step
        assert lib.tlb_fp8_attention(ctypes.addressof(pages), call(B=2, L=2), ints(*lens), ints(*table), None, 0, None) == -1
    assert lib.tlb_fp8_attention(ctypes.addressof(pages), call(), ints(5), None, None, 0, None) == -1
    assert lib.tlb_fp8_attention_workspace(ctypes.addressof(long), call(pages=100), np.array([100], dtype=np.int32).tobytes()) == 0  # short for now


def test_sizes_whose_places_an_int_does_not_hold_are_refused():
    import ctypes

    lib = blocks.library()
    attend = lambda pages: blocks._FP8_ATTENTION.pack(16, 16, 16, 16, 0, 0, 0, 1.0, 1, 4, 1, pages, 1, 2)  # noqa: E731
    append = lambda pages: blocks._FP8_APPEND.pack(16, 16, 16, 16, 16, 16, 0, 0, *[0] * 9, 1.0, 0.0, 0.0, 1, 4, 1, pages, 0, 0, 2)  # noqa: E731
    wide, many = blocks.Fp8Pages(4096, 8192, 4096, 4096, 4, 2, 128, 32), blocks.Fp8Pages(4096, 8192, 4096, 4096, 1 << 28, 2, 128, 32)
    for pages, width in ((wide, (1 << 23) + 1), (many, 1)):
        assert lib.tlb_fp8_attention(ctypes.addressof(pages), attend(width), None, None, None, 0, None) == -1
        assert lib.tlb_fp8_append(ctypes.addressof(pages), append(width), None, None, None) == -1


# ---- pool and caches ----------------------------------------------------------------------------------------------------


@pytest.fixture
def appended(monkeypatch):
    """Appends that only record what they are given."""
    seen = []

    def fake(query, key, value, pages, block_table, context_lens, *, rope=None, query_norm=None, key_norm=None, block_table_host=None, context_lens_host=None):
        fp8_cache.validate_paged_metadata(context_lens_host, block_table_host, pages.page_size, pages.num_pages, query.shape[2])
        seen.append((query.shape[2], block_table.tolist(), context_lens.tolist()))
        return query

    monkeypatch.setattr(fp8_cache, "rotate_append_fp8", fake)
    return seen


def rows(L, B=1):
    return torch.zeros(B, 4, L, 32, dtype=torch.bfloat16), torch.zeros(B, 2, L, 32, dtype=torch.bfloat16), torch.zeros(B, 2, L, 32, dtype=torch.bfloat16)


def test_a_request_fills_pages_in_order_and_gives_them_back(appended):
    pool = Fp8KvPagedPool(page_size=16)
    a, b = Fp8KvPagedCache(pool), Fp8KvPagedCache(pool)
    q, meta = a.rotate_append_paged(*rows(20))
    assert meta.context_lens_host.tolist() == [20] and meta.block_table_host.tolist() == [[0, 1]] and meta.pages is pool.pages
    b.rotate_append_paged(*rows(5))
    a.rotate_append_paged(*rows(13))
    assert a.page_ids == [0, 1, 3] and a.page_lens == [16, 16, 1] and b.page_ids == [2]
    a.rewind(2)
    assert a.page_ids == [0, 1] and a.offset == 31
    a.rotate_append_paged(*rows(1))
    assert a.page_ids == [0, 1] and appended[-1] == (1, [[0, 1]], [32])
    a.release(), b.release()
    assert not pool.used_page_ids and a.offset == 0
    pool.reset()
    assert pool.pages is None and pool.storage_nbytes == 0


def test_growth_carries_numbers_and_scales_over(appended):
    pool = Fp8KvPagedPool(page_size=16)
    a = Fp8KvPagedCache(pool)
    a.rotate_append_paged(*rows(60))
    assert pool.capacity == 4
    pool.pages.keys.view(torch.uint8)[:4] = 7
    pool.pages.value_scales[:4] = 0.5
    old = pool.slab_version
    a.rotate_append_paged(*rows(10))
    assert pool.capacity == 8 and pool.slab_version != old and pool.copied_pages_on_growth == 4
    assert (pool.pages.keys.view(torch.uint8)[:4] == 7).all() and not pool.pages.keys.view(torch.uint8)[4:].any() and (pool.pages.value_scales[:4] == 0.5).all()


def test_a_step_that_fails_leaves_everything_as_it_was(appended, monkeypatch):
    pool = Fp8KvPagedPool(page_size=16, max_pages=3)
    a, b = Fp8KvPagedCache(pool), Fp8KvPagedCache(pool)
    table = BatchingKvCache(3)
    table.add_request(a, 0), table.add_request(b, 2)
    table.rotate_append_paged(*rows(16, 3))
    assert appended[-1] == (16, [[0], [-1], [1]], [16, 0, 16])
    before = (a._snapshot_state(), b._snapshot_state(), pool.num_allocated_pages, set(pool.used_page_ids))
    with pytest.raises(RuntimeError, match="exhausted"):
        table.rotate_append_paged(*rows(1, 3))
    assert before == (a._snapshot_state(), b._snapshot_state(), pool.num_allocated_pages, set(pool.used_page_ids))
    with pytest.raises(ValueError, match="existing pages"):
        a.rotate_append_paged(torch.zeros(1, 4, 1, 64), torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 1, 64))
    assert before[0] == a._snapshot_state()


def test_mixed_pools_lengths_and_widths_are_refused(appended):
    pool, other = Fp8KvPagedPool(page_size=16), Fp8KvPagedPool(page_size=16)
    table = BatchingKvCache(2, max_seq_len=20)
    with pytest.raises(ValueError, match="active requests"):
        table.rotate_append_paged(*rows(1, 2))
    table.add_request(Fp8KvPagedCache(pool), 0), table.add_request(Fp8KvPagedCache(other), 1)
    with pytest.raises(ValueError, match="one page pool"):
        table.rotate_append_paged(*rows(1, 2))
    table.kv_caches[1] = TinyKvPagedCache(TinyKvPagedPool(16))
    with pytest.raises(ValueError, match="one page pool"):
        table.rotate_append_paged(*rows(1, 2))
    table.kv_caches[1] = None
    with pytest.raises(ValueError, match="batch size"):
        table.rotate_append_paged(*rows(1, 3))
    with pytest.raises(ValueError, match="max_seq_len"):
        table.rotate_append_paged(*rows(21, 2))
    with pytest.raises(ValueError, match="multiple"):
        Fp8KvPagedPool(page_size=24)
    with pytest.raises(ValueError, match="8-bit pool"):
        Fp8KvPagedCache(TinyKvPagedPool(16))
    for call in (table.kv_caches[0].update_and_fetch, table.kv_caches[0].update_and_fetch_paged):
        with pytest.raises(NotImplementedError):
            call(*rows(1)[1:])


# ---- the model ------------------------------------------------------------------------------------------------------------


def test_the_models_option(cpu_ext):
    ns = synthetic_qwen3("tiny", seed=0)
    model = Qwen3ModelWeek3(ns, page_size=16, kv_cache="e4m3")
    assert all(isinstance(p, Fp8KvPagedPool) for p in model.page_pools) and all(isinstance(c, Fp8KvPagedCache) for c in model.create_kv_cache())
    assert isinstance(Qwen3ModelWeek3(ns).create_kv_cache()[0], TinyKvPagedCache)
    with pytest.raises(NotImplementedError):
        model.decode_engine(1)
    for bad in (dict(kv_cache="int8"), dict(kv_cache="e4m3", enable_paged_attention=False), dict(kv_cache="e4m3", page_size=8)):
        with pytest.raises(ValueError):
            Qwen3ModelWeek3(ns, **bad)


def test_a_models_steps_append_and_attend_at_the_caches_positions(cpu_ext, appended, monkeypatch):
    ns = synthetic_qwen3("tiny", seed=0)
    model = Qwen3ModelWeek3(ns, page_size=16, kv_cache="e4m3")
    seen = []
    monkeypatch.setattr(qwen3_week3, "paged_attention_fp8", lambda q, pages, table, lens, **k: seen.append((tuple(q.shape), lens.tolist(), k["mask"])) or q)
    cache = model.create_kv_cache()
    model(torch.arange(20, dtype=torch.int32)[None], 0, cache, logits_to_keep=1)
    model(torch.tensor([[3]], dtype=torch.int32), torch.tensor([20]), cache, logits_to_keep=1)
    assert seen == [((1, 4, 20, 32), [20], "causal")] * 2 + [((1, 4, 1, 32), [21], "causal")] * 2
    with pytest.raises(ValueError, match="number of tokens"):
        model(torch.tensor([[3]], dtype=torch.int32), 20, cache)
    tables = [BatchingKvCache(3, max_seq_len=64) for _ in cache]
    for c, t in zip(cache, tables):
        t.add_request(c, 1)
    model(torch.zeros(3, 1, dtype=torch.int32), [0, 21, 0], tables, logits_to_keep=1)
    assert seen[-1] == ((3, 4, 1, 32), [0, 22, 0], "causal")
    for t in tables:
        t.remove_request(1)
    assert all(not p.used_page_ids for p in model.page_pools)
