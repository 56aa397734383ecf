"""A step over the 8-bit cache is only put in line: the host waits for the device nowhere in it."""

import pytest
import torch

from tests.test_gpu_fp8_cache import check_attention
from tiny_llm_b200 import BatchingKvCache, FastRMSNorm, FastRoPE, Fp8KvPagedCache, Fp8KvPagedPool, Fp8KvPages, paged_attention_fp8

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [1, 40])
def test_a_step_of_a_batch_waits_for_nothing(new):
    heads, kv_heads, dim = 8, 2, 128
    gen = torch.Generator(device=DEV).manual_seed(new)
    pool = Fp8KvPagedPool(page_size=32)
    pool.reserve(64, kv_heads, dim)
    batch = BatchingKvCache(3)
    for slot in (0, 2):
        batch.add_request(Fp8KvPagedCache(pool), slot)
    norm = FastRMSNorm(dim, torch.ones(dim, dtype=torch.bfloat16, device=DEV), eps=1e-6)
    more = dict(rope=FastRoPE(dim, 4096, 10000), query_norm=norm, key_norm=norm)
    steps = [tuple(torch.randn(3, h, new, dim, generator=gen, device=DEV).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads)) for _ in range(5)]

    def step(q, k, v):
        x, meta = batch.rotate_append_paged(q, k, v, **more)
        return x, meta, paged_attention_fp8(x, meta.pages, meta.block_table, meta.context_lens, mask="causal", block_table_host=meta.block_table_host, context_lens_host=meta.context_lens_host)

    step(*steps[0])
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        answers = [step(*s) for s in steps[1:]]
    finally:
        torch.cuda.set_sync_debug_mode("default")
    x, meta, out = answers[-1]
    assert meta.block_table.cpu().tolist() == meta.block_table_host.tolist() and meta.context_lens.cpu().tolist() == meta.context_lens_host.tolist() == [5 * new, 0, 5 * new]
    pages = Fp8KvPages(*(t.cpu() for t in (meta.pages.keys, meta.pages.values, meta.pages.key_scales, meta.pages.value_scales)))
    check_attention(out, x.cpu(), pages, meta.block_table_host, [5 * new, 0, 5 * new], True, dim**-0.5, torch.bfloat16)
