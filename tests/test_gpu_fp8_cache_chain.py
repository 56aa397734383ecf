"""Appends to the 8-bit cache and attention over it, launch behind launch: each reads what the one in front has just written, scales that grow among it."""

import numpy as np
import pytest
import torch

from tiny_llm_b200 import FastRoPE, Fp8KvPages, paged_attention_fp8, rotate_append_fp8

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requests,new,page,dtype", [(1, 1, 128, torch.bfloat16), (24, 1, 128, torch.bfloat16), (24, 1, 16, torch.float32), (2, 40, 128, torch.bfloat16), (1, 130, 64, torch.bfloat16)])
def test_a_chain_of_steps_is_what_it_is_when_each_launch_is_waited_for(requests, new, page, dtype):
    heads, kv_heads, dim, steps, start = 16, 8, 128, 30, 600
    gen = torch.Generator(device=DEV).manual_seed(requests + new)
    make = lambda h: torch.randn(steps, requests, h, new, dim, generator=gen, device=DEV)  # noqa: E731
    # most steps need a larger scale than the one before, in another order for every request and head
    grow = torch.exp2(torch.randint(-3, 4, (steps, requests, kv_heads, 1, 1), generator=gen, device=DEV) + 0.5 * torch.arange(steps, device=DEV)[:, None, None, None, None])
    q, k, v = make(heads).to(dtype), (make(kv_heads) * grow).to(dtype), (make(kv_heads) * grow).to(dtype)
    last = start + steps * new
    width = -(-last // page)
    full = np.random.RandomState(1).permutation(requests * width).astype(np.int32).reshape(requests, width)
    hosts = []
    for i in range(steps):
        n = start + (i + 1) * new
        table = np.where(np.arange(width)[None] < -(-n // page), full, -1).astype(np.int32)
        hosts.append((table, np.full(requests, n, dtype=np.int32)))
    tables, lens = ([torch.from_numpy(h[j]).to(DEV) for h in hosts] for j in range(2))
    numbers = [(torch.randn(requests * width, kv_heads, page, dim, generator=gen, device=DEV) * 60).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.exp2(torch.randint(-9, -5, (requests * width, kv_heads, page // 16), generator=gen, device=DEV).float()) for _ in range(2)]
    rope = FastRoPE(dim, 4096, 10000)

    def run(waiting):
        pages = Fp8KvPages(*(t.clone() for t in (*numbers, *scales)))
        out = []
        for i, (table, n) in enumerate(hosts):
            where = dict(block_table_host=table, context_lens_host=n)
            if waiting:
                torch.cuda.synchronize()
            x = rotate_append_fp8(q[i], k[i], v[i], pages, tables[i], lens[i], rope=rope, **where)
            if waiting:
                torch.cuda.synchronize()
            out.append(paged_attention_fp8(x, pages, tables[i], lens[i], mask="causal", **where))
        torch.cuda.synchronize()
        return torch.stack(out), pages.keys.view(torch.uint8), pages.values.view(torch.uint8), pages.key_scales, pages.value_scales

    want = run(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))
