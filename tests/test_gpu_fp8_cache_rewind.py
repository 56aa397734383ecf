"""What a rewind of an 8-bit cache leaves of the dropped tokens: nothing at the beginning of a block, the block's scale inside one."""

import math

import pytest
import torch

from tiny_llm_b200 import Fp8KvPagedCache, Fp8KvPagedPool, FastRoPE, paged_attention_fp8

DEV = "cuda"
pytestmark = pytest.mark.gpu
HEADS, KV, DIM, PAGE = 4, 2, 64, 32
ROPE = FastRoPE(DIM, 4096, 10000)


def tokens(n, seed, size=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return tuple((size * torch.randn(1, h, n, DIM, generator=gen, device=DEV)).to(torch.bfloat16) for h in (HEADS, KV, KV))


def fresh():
    return Fp8KvPagedCache(Fp8KvPagedPool(page_size=PAGE))


def numbers(cache):
    """What the request's numbers stand for: keys and values [tokens, H, D]."""
    sides = cache.pool.pages.dequantize(cache.page_ids)
    return [x.transpose(1, 2).flatten(0, 1)[: cache.offset] for x in sides]


def attend(cache, q, meta):
    return paged_attention_fp8(q, meta.pages, meta.block_table, meta.context_lens, mask="causal", block_table_host=meta.block_table_host, context_lens_host=meta.context_lens_host)


@pytest.mark.parametrize("keep", [0, 16, 32, 48])
@pytest.mark.parametrize("bad", [1e30, math.nan, math.inf])
def test_at_the_beginning_of_a_block_nothing_is_left(keep, bad):
    seen, never = fresh(), fresh()
    first, more = tokens(max(keep, 1), 1), tokens(9, 2)
    for c in (seen, never):
        if keep:
            c.rotate_append_paged(*first, rope=ROPE)
    q, k, v = tokens(7, 3)
    k[:, :, 2, 5] = v[:, :, 2, 5] = bad
    seen.rotate_append_paged(q, k, v, rope=ROPE)
    seen.rewind(7)
    assert seen.offset == keep
    (a, meta_a), (b, meta_b) = (c.rotate_append_paged(*more, rope=ROPE) for c in (seen, never))
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(numbers(seen), numbers(never)))
    assert torch.equal(attend(seen, a, meta_a), attend(never, b, meta_b))


@pytest.mark.parametrize("size", [4.0, 300.0, 1e30])
def test_inside_a_block_its_scale_is_left(size):
    """As if the dropped tokens had come along: the numbers that stay are off by half a step of that scale at the most (once for the first rounding, once for the second)."""
    seen, never = fresh(), fresh()
    first, more = tokens(21, 1), tokens(9, 2)
    for c in (seen, never):
        c.rotate_append_paged(*first)
    large = tokens(3, 3, size)
    seen.rotate_append_paged(*large)
    scales = [s[seen.page_ids[0], :, 1].clone() for s in (seen.pool.pages.key_scales, seen.pool.pages.value_scales)]
    seen.rewind(3)
    assert seen.offset == 21
    seen.rotate_append_paged(*more), never.rotate_append_paged(*more)
    for got, want, scale, after, x in zip(numbers(seen), numbers(never), scales, (seen.pool.pages.key_scales, seen.pool.pages.value_scales), (1, 2)):
        assert torch.equal(after[seen.page_ids[0], :, 1], scale)  # what the large tokens asked for is more than the later ones'
        assert torch.equal(got[:16], want[:16])  # another block
        exact = torch.cat([first[x], more[x]], dim=2)[0].transpose(0, 1).double()
        block = slice(16, 30)
        step = torch.maximum(exact[block].abs() * 2.0**-4, scale.double()[None, :, None] * 2.0**-10)
        assert ((got[block].double() - exact[block]).abs() <= 2 * step * (1 + 2.0**-8)).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_dropped_number_that_is_none_stays_until_its_block_begins_anew(bad):
    cache = fresh()
    first = tokens(21, 1)
    cache.rotate_append_paged(*first)
    q, k, v = tokens(3, 3)
    k[:, 1, 1, 0] = bad
    cache.rotate_append_paged(q, k, v)
    cache.rewind(3)
    cache.rotate_append_paged(*tokens(1, 4))
    keys, values = numbers(cache)
    assert keys[16:, 1].isnan().all() and not keys[:, 0].isnan().any() and not keys[:16].isnan().any() and not values.isnan().any()
    cache.rewind(6)  # to the block's beginning, and what it held once more
    cache.rotate_append_paged(*(x[:, :, 16:] for x in first))
    clean = fresh()
    clean.rotate_append_paged(*first)
    assert all(torch.equal(a, b) for a, b in zip(numbers(cache), numbers(clean)))
