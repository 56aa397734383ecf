"""A Qwen3 model over a cache of 8 bits: every append and every attention it makes, against 64 bits on the model's own inputs; the scheduler; the command line.

The helpers and tolerances are those of the operators' own tests."""

import numpy as np
import pytest
import torch

from tests.test_gpu_fp8_cache import check_attention, check_side, on_host, turned
from tiny_llm_b200 import BatchingKvCache, Fp8KvPages, Qwen3ModelWeek3, batch_generate, fp8_cache, greedy_generate_ids, qwen3_week3
from tiny_llm_b200.cli import main
from tiny_llm_b200.synthetic import synthetic_qwen3

DEV = "cuda"
pytestmark = pytest.mark.gpu


def host(pages):
    return Fp8KvPages(*(t.cpu() for t in (pages.keys, pages.values, pages.key_scales, pages.value_scales)))


@pytest.fixture
def watched(monkeypatch):
    """The model's appends and attention, checked as they are made; -> how many of each."""
    count = {"append": 0, "attend": 0}
    append, attend = fp8_cache.rotate_append_fp8, qwen3_week3.paged_attention_fp8

    def checked_append(query, key, value, pages, table, lens, *, rope, query_norm, key_norm, **hosts):
        before = host(pages)
        out = append(query, key, value, pages, table, lens, rope=rope, query_norm=query_norm, key_norm=key_norm, **hosts)
        lengths, new = hosts["context_lens_host"].tolist(), query.shape[2]
        eps, k64 = key_norm.eps, torch.zeros(key.shape, dtype=torch.float64)
        assert rope.base == 10000, "the helper's base"
        weight = key_norm.weight.to(query.dtype).cpu()
        for b, n in enumerate(lengths):
            for h in range(key.shape[1]):
                if n:
                    k64[b, h] = turned(key[b, h].cpu(), weight, eps, rope.dims, rope.traditional, n - new)
        check_side("keys", on_host(pages.keys), on_host(pages.key_scales), on_host(before.keys), on_host(before.key_scales), k64, hosts["block_table_host"], lengths, new, pages.page_size)
        check_side("values", on_host(pages.values), on_host(pages.value_scales), on_host(before.values), on_host(before.value_scales), value.cpu().double(), hosts["block_table_host"],
                   lengths, new, pages.page_size)
        count["append"] += 1
        return out

    def checked_attend(query, pages, table, lens, *, scale, mask, block_table_host, context_lens_host):
        out = attend(query, pages, table, lens, scale=scale, mask=mask, block_table_host=block_table_host, context_lens_host=context_lens_host)
        assert mask == "causal"
        check_attention(out, query.cpu(), host(pages), block_table_host, context_lens_host.tolist(), True, scale, query.dtype)
        count["attend"] += 1
        return out

    monkeypatch.setattr(fp8_cache, "rotate_append_fp8", checked_append)
    monkeypatch.setattr(qwen3_week3, "paged_attention_fp8", checked_attend)
    return count


def make(**more):
    ns = synthetic_qwen3("tiny-d128", seed=0, device=DEV, realistic=True)
    ns.args.rope_theta = 10000
    return Qwen3ModelWeek3(ns, page_size=32, kv_cache="e4m3", **more)


def test_portions_single_tokens_and_a_batch(watched):
    model = make()
    gen = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 512, (200,), generator=gen, dtype=torch.int32).to(DEV)
    first, second = model.create_kv_cache(), model.create_kv_cache()
    at = 0
    for n in (70, 1, 33, 9):  # a portion, a token, portions that end inside a block
        logits = model(ids[at : at + n][None], at, first, logits_to_keep=1)
        at += n
    model(ids[:17][None], 0, second, logits_to_keep=1)
    tables = [BatchingKvCache(3, max_seq_len=256) for _ in first]
    for table, a, b in zip(tables, first, second):
        table.add_request(a, 2), table.add_request(b, 0)
    for k in range(3):
        logits = model(torch.stack([ids[20 + k], ids[0], ids[150 + k]])[:, None], [17 + k, 0, at + k], tables, logits_to_keep=1)
    assert torch.isfinite(logits).all() and watched == {"append": 2 * 8, "attend": 2 * 8}
    for table in tables:
        table.remove_request(0), table.remove_request(2)
    assert all(not p.used_page_ids for p in model.page_pools)


def test_a_rewound_request_goes_on(watched):
    model = make()
    ids = torch.arange(60, dtype=torch.int32, device=DEV)
    cache = model.create_kv_cache()
    model(ids[:50][None], 0, cache, logits_to_keep=1)
    for c in cache:
        c.rewind(13)
    model(ids[37:60][None], 37, cache, logits_to_keep=1)
    assert cache[0].offset == 60 and watched["attend"] == 4


def test_the_scheduler_runs_requests_of_unlike_length(watched):
    model = make()
    prompts = [list(range(3, 3 + n)) for n in (5, 40, 70, 18)]
    answers = dict(batch_generate(model, None, prompts, max_seq_len=128, batch_size=2, prefill_step=32, verbose=False, device=torch.device(DEV), max_new_tokens=[6] * 4))
    assert sorted(answers) == [0, 1, 2, 3] and all(len(text.split()) == 6 for text in answers.values())
    assert all(not p.used_page_ids for p in model.page_pools)


def test_half_the_memory_of_the_16_bit_cache():
    ns = synthetic_qwen3("tiny-d128", seed=0, device=DEV, realistic=True)
    sizes = {}
    for kind in ("bf16", "e4m3"):
        model = Qwen3ModelWeek3(ns, page_size=32, kv_cache=kind)
        model.use_decode_graph = False
        cache = model.create_kv_cache()
        model(torch.arange(100, dtype=torch.int32, device=DEV)[None], 0, cache, logits_to_keep=1)
        sizes[kind] = model.page_pools[0].storage_nbytes
    assert sizes["e4m3"] == sizes["bf16"] // 2 * (1 + 1 / 512)  # 4 bytes for every 16 x 128


def test_generation_and_command_line(capsys):
    model = make()
    out = greedy_generate_ids(model, [5, 17, 3], 8, device=torch.device(DEV))
    assert len(out) == 8
    assert main(["generate", "--synthetic", "tiny-d128", "--prompt-ids", "5,17,3", "--max-new-tokens", "8", "--kv-cache", "e4m3"]) == 0
    assert len(capsys.readouterr().out.split()) == 8
    assert main(["batch", "--synthetic", "tiny-d128", "--prompt-ids", "5,17,3;9,9,4,1", "--batch-size", "2", "--max-new-tokens", "4", "--quiet", "--kv-cache", "e4m3"]) == 0
    with pytest.raises(SystemExit):
        main(["generate", "--synthetic", "tiny-d128", "--prompt-ids", "5", "--loader", "week2", "--kv-cache", "e4m3"])
    with pytest.raises(SystemExit):
        main(["generate", "--synthetic", "voluzen:WC", "--prompt-ids", "5", "--kv-cache", "e4m3"])
