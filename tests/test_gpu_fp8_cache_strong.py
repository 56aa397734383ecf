"""Attention over pages of 8 bits with scores of 2^20 and far more: they are rounded once, like their maxima, so that equal scores have equal weights and none is above its own maximum."""

import pytest
import torch

from tests.test_gpu_fp8_cache import table_of, to_gpu
from tiny_llm_b200 import Fp8KvPages, paged_attention_fp8

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,new,heads,kv_heads,dim", [([400, 0, 700], 1, 8, 2, 128), ([3000], 1, 8, 8, 64), ([300], 3, 4, 2, 96), ([90, 500], 8, 8, 2, 128), ([700, 400], 300, 16, 2, 128), ([2000], 130, 16, 2, 64)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("size", [2.0**21, 1.3e9, -7.7e11, 3e18])
def test_equal_scores_and_one_above_them(lengths, new, heads, kv_heads, dim, dtype, size):
    page = 32
    gen = torch.Generator().manual_seed(dim + new)
    table, count = table_of(lengths, page, 3)
    pages = Fp8KvPages.zeros(count, kv_heads, page, dim, device="cpu")
    pages.keys[..., 0] = torch.tensor(1.0).to(torch.float8_e4m3fn)
    pages.values.copy_((torch.randn(pages.values.shape, generator=gen) * 60).clamp(-448, 448).to(torch.float8_e4m3fn))
    pages.key_scales.fill_(0.25), pages.value_scales.fill_(2.0**-5)
    q = torch.zeros(len(lengths), heads, new, dim)
    q[..., 0] = size * (1 + 0.3 * torch.rand(len(lengths), heads, new, generator=gen))
    q = q.to(dtype)
    args = (torch.from_numpy(table).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))
    even = paged_attention_fp8(q.to(DEV), to_gpu(pages), *args, mask="causal").cpu().double()
    chosen = {}
    for b, n in enumerate(lengths):
        if n:  # of all that every row sees
            chosen[b] = (n - new) // 3
            pages.keys[int(table[b, chosen[b] // page]), :, chosen[b] % page, 0] = torch.tensor(2.0 if size > 0 else 0.5).to(torch.float8_e4m3fn)
    one = paged_attention_fp8(q.to(DEV), to_gpu(pages), *args, mask="causal").cpu().double()
    for b, n in enumerate(lengths):
        if n == 0:
            assert not even[b].any() and not one[b].any()
            continue
        homes = [int(p) for p in table[b, : -(-n // page)]]
        v = (pages.values.float().double()[homes].transpose(0, 1).flatten(1, 2)[:, :n] * 2.0**-5).repeat_interleave(heads // kv_heads, 0)
        # weights are all the same number, whose rounding the sum that divides does not share (f16: 2^-11); sums in fp32; the output's own rounding
        weight = 2.0**-11 if dtype == torch.bfloat16 else 2.0**-21
        sums = v.cumsum(1)[:, n - new :], v.abs().cumsum(1)[:, n - new :]
        keys = torch.arange(n - new + 1, n + 1, dtype=torch.float64)[None, :, None]
        want = sums[0] / keys
        assert ((even[b] - want).abs() <= (weight + 2.0**-18) * sums[1] / keys + torch.finfo(dtype).eps / 2 * 1.01 * want.abs()).all(), b
        want = v[:, chosen[b], None]
        assert ((one[b] - want).abs() <= (weight + 2.0**-18 + torch.finfo(dtype).eps / 2 * 1.01) * want.abs()).all(), b
