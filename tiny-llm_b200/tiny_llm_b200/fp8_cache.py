"""A paged key/value cache of 8 bits: e4m3 numbers with one scale, a power of two, for each 16 tokens of a head.

``Fp8KvPages`` is the storage (the page layout of ``TinyKvPagedPool``, one byte a number), ``rotate_append_fp8`` puts a step's keys and values
into it, with the norm and the rotation that queries and keys pass on the way, and ``paged_attention_fp8`` is ``paged_attention`` over it.  The block
table and the context lengths are those of the 16-bit cache: a request's tokens fill its pages in order, ``context_lens`` count the step's own
tokens, 0 marks an idle slot.

``Fp8KvPagedPool`` and ``Fp8KvPagedCache`` are the page allocator and a request's cache over such pages (``Qwen3ModelWeek3(..., kv_cache="e4m3")``); both sides of the
bookkeeping are those of ``TinyKvPagedPool`` and ``TinyKvPagedCache``."""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from extensions_b200.tiny_llm_ext_b200 import blocks

from .attention import validate_paged_metadata
from .paged_kv_cache import _SLAB_VERSIONS, TinyKvPagedCache, TinyKvPagedPool

TOKENS = 16  # that share a scale
_DTYPES = (torch.float32, torch.bfloat16)
_INT32 = np.dtype(np.int32)


class Fp8KvPages:
    """``keys`` and ``values`` (``torch.float8_e4m3fn``) ``[P, H_kv, page_size, D]``, ``key_scales`` and ``value_scales`` (fp32)
    ``[P, H_kv, page_size / 16]``; ``page_size`` and ``D`` are multiples of 16, ``D`` at most 256.  A number stands for itself times its block's
    scale, a power of two; where that is NaN (an infinity or a NaN was stored), every number of the block is.  Numbers by themselves are finite: pages that
    something else than ``rotate_append_fp8`` fills have to keep to that where a request's tokens are."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor, value_scales: torch.Tensor):
        for name, t in (("keys", keys), ("values", values)):
            if t.dtype != torch.float8_e4m3fn or t.dim() != 4 or t.shape != keys.shape or min(t.shape) <= 0:
                raise ValueError(f"Fp8KvPages: {name} must be float8_e4m3fn [P, H_kv, page_size, D], keys and values alike")
        pages, heads, size, dim = keys.shape
        if size % TOKENS or dim % 16 or dim > 256:
            raise ValueError(f"Fp8KvPages: page_size must be a multiple of {TOKENS}, D a multiple of 16 up to 256, got {size} and {dim}")
        for name, t in (("key_scales", key_scales), ("value_scales", value_scales)):
            if t.dtype != torch.float32 or t.shape != (pages, heads, size // TOKENS):
                raise ValueError(f"Fp8KvPages: {name} must be float32 {(pages, heads, size // TOKENS)}, one for each {TOKENS} tokens of a head")
        if any(t.device != keys.device or not t.is_contiguous() for t in (keys, values, key_scales, value_scales)) or keys.data_ptr() % 16 or values.data_ptr() % 16:
            raise ValueError("Fp8KvPages: tensors must be contiguous, on one device, the numbers on a boundary of 16 bytes")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, size, dim
        self.index = keys.get_device()
        self.native = blocks.Fp8Pages(keys.data_ptr(), values.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(), pages, heads, size, dim)

    @staticmethod
    def zeros(num_pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> "Fp8KvPages":
        if min(num_pages, kv_heads, page_size, head_dim) <= 0 or page_size % TOKENS:
            raise ValueError(f"Fp8KvPages: page_size must be a multiple of {TOKENS} and every size positive")
        numbers = [torch.zeros((num_pages, kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2)]
        return Fp8KvPages(*numbers, *(torch.zeros((num_pages, kv_heads, page_size // TOKENS), dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def device(self) -> torch.device:
        return self.keys.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.keys, self.values, self.key_scales, self.value_scales))

    def grown(self, num_pages: int, live: int) -> "Fp8KvPages":
        """Room for ``num_pages``, with the first ``live`` ones as they are here."""
        new = Fp8KvPages.zeros(num_pages, self.kv_heads, self.page_size, self.head_dim, device=self.device)
        for to, old in ((new.keys.view(torch.uint8), self.keys.view(torch.uint8)), (new.values.view(torch.uint8), self.values.view(torch.uint8)), (new.key_scales, self.key_scales),
                        (new.value_scales, self.value_scales)):
            to[:live] = old[:live]
        return new

    def dequantize(self, pages=slice(None), dtype: torch.dtype = torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """(keys, values) that the numbers of ``pages`` (an index into the first dimension) stand for."""
        wide = lambda numbers, scales: (numbers.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * scales[pages].repeat_interleave(TOKENS, -1)[..., None]).to(dtype)  # noqa: E731
        return wide(self.keys, self.key_scales), wide(self.values, self.value_scales)


def _step(op: str, pages: Fp8KvPages, query: torch.Tensor, block_table: torch.Tensor, context_lens: torch.Tensor, block_table_host, context_lens_host):
    """Checks of a step's shapes and metadata -> (the query's shape, block table, context lengths, the host's lengths and table as bytes, and as arrays)."""
    shape, rows = query.shape, block_table.shape
    if len(shape) != 4:
        raise ValueError(f"{op}: query must be 4D [B, H_q, L, D]")
    B, heads, L, D = shape
    if B <= 0 or heads <= 0 or L <= 0 or D <= 0:
        raise ValueError(f"{op}: dimensions must be positive")
    if D != pages.head_dim:
        raise ValueError(f"{op}: query and pages must have the same head dimension")
    if heads % pages.kv_heads:
        raise ValueError(f"{op}: query heads must be divisible by K/V heads")
    if query.dtype not in _DTYPES:
        raise ValueError(f"{op}: supports float32 or bfloat16 inputs")
    counts = context_lens.shape
    if len(rows) != 2 or len(counts) != 1 or block_table.dtype != torch.int32 or context_lens.dtype != torch.int32:
        raise ValueError(f"{op}: block_table must be 2D int32 and context_lens 1D int32")
    if rows[0] != B or counts[0] != B or rows[1] <= 0:
        raise ValueError(f"{op}: query, block_table, and context_lens batch sizes must match, with at least one page slot")
    if context_lens_host is None:
        context_lens_host = context_lens.detach().cpu().numpy()
    if block_table_host is None:
        block_table_host = block_table.detach().cpu().numpy()
    lens, table = np.asarray(context_lens_host), np.asarray(block_table_host)
    if lens.shape != counts or table.shape != rows:
        raise ValueError(f"{op}: context_lens_host and block_table_host must be copies of the tensors")
    if lens.dtype != _INT32 or table.dtype != _INT32:  # the library's check is for int32
        validate_paged_metadata(lens, table, pages.page_size, pages.num_pages, L)
        lens, table = lens.astype(_INT32), table.astype(_INT32)
    # a copy of a few kilobytes costs less than numpy's .ctypes
    bytes_of = table.tobytes() if table.nbytes <= 8192 or not table.flags.c_contiguous else table.ctypes.data
    return (shape, block_table if block_table.is_contiguous() else block_table.contiguous(), context_lens if context_lens.is_contiguous() else context_lens.contiguous(), lens.tobytes(),
            bytes_of, (lens, table))


def _refused(op: str, pages: Fp8KvPages, hosts: tuple, L: int) -> None:
    """What the library found in the lengths or the table, as an exception of ``paged_attention``."""
    validate_paged_metadata(*hosts, pages.page_size, pages.num_pages, L)
    raise RuntimeError(blocks.library().tlb_last_error().decode() or op)


def rotate_append_fp8(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, pages: Fp8KvPages, block_table: torch.Tensor, context_lens: torch.Tensor, *, rope=None,
                      query_norm=None, key_norm=None, block_table_host: np.ndarray | None = None, context_lens_host: np.ndarray | None = None) -> torch.Tensor:
    """Append a step's ``key`` and ``value [B, H_kv, L, D]`` to the pages at positions ``context_lens - L ..``; -> the queries ``[B, H_q, L, D]`` to attend with.

    ``query_norm`` and ``key_norm`` (``FastRMSNorm``) and ``rope`` (``FastRoPE``, turned by a token's position) are applied on the way, the keys' in 64 bits
    ahead of their one rounding.  Any strides will do; float32 or bfloat16.  A block of 16 tokens of a head has one scale: it grows where the new
    tokens need it to, and the block's earlier numbers are rounded to it again."""
    shape, table, lens, lens_host, table_host, hosts = _step("rotate_append_fp8", pages, query, block_table, context_lens, block_table_host, context_lens_host)
    B, _, L, D = shape
    theirs = key.shape
    if theirs != (B, pages.kv_heads, L, D) or theirs != value.shape:
        raise ValueError("rotate_append_fp8: key and value must be [B, H_kv, L, D] beside the query")
    dtype = query.dtype
    if key.dtype != dtype or value.dtype != dtype:
        raise ValueError("rotate_append_fp8: query, key, and value must have the same dtype")
    blocks.fp8_devices("rotate_append_fp8", pages.index, query, key, value, table, lens)
    rot, base, interleaved = 0, 1.0, False
    if rope is not None:
        rot, base, interleaved = rope.dims, rope.base, rope.traditional
        if rot % 2 or not 0 < rot <= D or not base > 0:
            raise ValueError(f"rotate_append_fp8: cannot rotate {rot} of {D} entries")
    weights = []
    for norm in (query_norm, key_norm):
        if norm is None:
            weights += (None, 0.0)
            continue
        weight = norm.weight
        if weight.dtype != dtype or weight.get_device() != pages.index or not weight.is_contiguous():
            weight = norm._weight_as(dtype, query.device)
        if weight.shape != (D,):
            raise ValueError(f"rotate_append_fp8: a norm of {tuple(weight.shape)} for heads of {D}")
        weights += (weight, norm.eps)
    out = blocks.fp8_append_of(pages.native, pages.index, query, key, value, table, lens, *weights, rot, base, interleaved, lens_host, table_host)
    if out is None:
        _refused("rotate_append_fp8", pages, hosts, L)
    return out


def paged_attention_fp8(query: torch.Tensor, pages: Fp8KvPages, block_table: torch.Tensor, context_lens: torch.Tensor, scale: float | None = None,
                        mask: torch.Tensor | str | None = None, *, block_table_host: np.ndarray | None = None, context_lens_host: np.ndarray | None = None) -> torch.Tensor:
    """``paged_attention`` over pages of 8 bits: ``query [B, H_q, L, D]`` (float32 or bfloat16, any strides) -> the same shape and dtype, laid out token by token.
    ``mask``: None or ``"causal"``; ``scale``: ``D ** -0.5`` by default.  Rows of idle slots come out as zeros."""
    if isinstance(mask, torch.Tensor) or mask not in (None, "causal"):
        raise NotImplementedError("Paged attention only supports mask=None or causal")
    shape, table, lens, lens_host, table_host, hosts = _step("paged_attention_fp8", pages, query, block_table, context_lens, block_table_host, context_lens_host)
    factor = shape[3] ** -0.5 if scale is None else float(scale)
    blocks.fp8_devices("paged_attention_fp8", pages.index, query, table, lens)
    if torch.cuda.is_current_stream_capturing():  # a captured call is replayed for other lengths
        validate_paged_metadata(*hosts, pages.page_size, pages.num_pages, shape[2])
        lens_host = table_host = None
    out = blocks.fp8_attention_of(pages.native, pages.index, query, table, lens, factor, mask == "causal", lens_host, table_host)
    if out is None:
        _refused("paged_attention_fp8", pages, hosts, shape[2])
    return out


@dataclass
class Fp8KvMetadata:
    """What attention over an 8-bit cache needs for one layer; the ``*_host`` fields are the copies the tensors were made from."""

    pages: Fp8KvPages
    block_table: torch.Tensor
    context_lens: torch.Tensor
    block_table_host: np.ndarray
    context_lens_host: np.ndarray


class Fp8KvPagedPool(TinyKvPagedPool):
    """A layer's pages of 8 bits: the allocator of ``TinyKvPagedPool`` over ``Fp8KvPages``, which are made with the first tokens (or ``reserve``) and grow
    geometrically.  ``max_pages``: an append that needs more fails instead."""

    def __init__(self, page_size: int = 128, max_pages: int | None = None):
        if page_size <= 0 or page_size % TOKENS:
            raise ValueError(f"an 8-bit page holds a multiple of {TOKENS} tokens, got {page_size}")
        super().__init__(page_size=page_size)
        self.pages: Fp8KvPages | None = None
        self.max_pages = max_pages

    @property
    def capacity(self) -> int:
        return 0 if self.pages is None else self.pages.num_pages

    @property
    def key_pages(self):
        raise AttributeError("an 8-bit pool has .pages")

    value_pages = key_pages

    @property
    def storage_nbytes(self) -> int:
        return 0 if self.pages is None else self.pages.nbytes

    def read_page(self, page_id: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values ``[1, H, page_size, D]`` (fp32) that a page's numbers stand for."""
        if self.pages is None:
            raise ValueError(f"Page {page_id} has no storage")
        if not 0 <= page_id < self.num_pages:
            raise ValueError(f"Page {page_id} is out of range")
        return self.pages.dequantize(slice(page_id, page_id + 1))

    def reserve(self, num_pages: int, heads: int, head_dim: int, dtype=None, device="cuda") -> None:
        """Room for ``num_pages`` (one counted growth; live pages are carried over)."""
        if self.pages is not None and (self.pages.kv_heads, self.pages.head_dim) != (heads, head_dim):
            raise ValueError("keys and values must match the existing pages")
        if self.capacity >= num_pages:
            return
        if self.max_pages is not None and num_pages > self.max_pages:
            raise RuntimeError(f"page pool exhausted: {num_pages} pages wanted, the pool is fixed at {self.max_pages}")
        if self.pages is None:
            self.pages = Fp8KvPages.zeros(num_pages, heads, self.page_size, head_dim, device=device)
        else:
            live = min(self.num_pages, self.capacity)
            self.copied_pages_on_growth += live
            self.copied_bytes_on_growth += self.pages.nbytes // self.pages.num_pages * live
            self.pages = self.pages.grown(num_pages, live)
        self.storage_growths += 1
        self.slab_version = next(_SLAB_VERSIONS)

    def ensure_room(self, fresh_pages: int, heads: int, head_dim: int, device) -> None:
        """Make sure ``fresh_pages`` allocations will find storage."""
        wanted = self.num_pages + max(0, fresh_pages - len(self.free_page_ids))
        if wanted > self.capacity or self.pages is None:
            self.reserve(max(wanted, min(max(4, wanted, self.capacity * 2), self.max_pages or 1 << 62)), heads, head_dim, device=device)
        elif (self.pages.kv_heads, self.pages.head_dim) != (heads, head_dim):
            raise ValueError("keys and values must match the existing pages")

    def reset(self) -> None:
        super().reset()
        self.pages = None

    def _snapshot_state(self) -> tuple:
        return (*super()._snapshot_state(), self.pages)

    def _restore_state(self, state: tuple) -> None:
        super()._restore_state(state[:-1])
        if self.pages is not state[-1]:
            self.pages = state[-1]
            self.slab_version = next(_SLAB_VERSIONS)

    def _ensure_page_storage(self, key, value) -> None:
        raise NotImplementedError("an 8-bit pool is filled by rotate_append_paged")

    def can_batch_decode_append(self, keys, slots) -> bool:
        return False


class Fp8KvPagedCache(TinyKvPagedCache):
    """A request's pages in an ``Fp8KvPagedPool``.

    ``rewind`` to the beginning of a block of 16 tokens, or of the request, leaves nothing of the dropped tokens.  Inside a block it is bookkeeping alone, and a rewind of
    16 bits' caches is more than that: the block keeps the scale that the dropped tokens made it take, and the numbers of the tokens that stay are rounded to it, as if all had come
    together.  So a dropped token far larger than these costs them their small bits (or all of them), and a dropped infinity or NaN makes the block's numbers none for good:
    ``rewind`` further then, to the block's beginning, and append what it held again."""

    def __init__(self, pool: Fp8KvPagedPool):
        if not isinstance(pool, Fp8KvPagedPool):
            raise ValueError("an 8-bit cache needs an 8-bit pool")
        super().__init__(pool)

    def _device(self):
        return self.pool.pages.device if self.pool.pages is not None else torch.device("cpu")

    def update_and_fetch(self, key, value, mask_length=None, mask=None):
        raise NotImplementedError("an 8-bit cache is filled by rotate_append_paged")

    update_and_fetch_paged = update_and_fetch

    def rotate_append_paged(self, query, key, value, *, rope=None, query_norm=None, key_norm=None) -> tuple[torch.Tensor, Fp8KvMetadata]:
        """``rotate_append_fp8`` of the request's next tokens (``[1, H, L, D]``) -> (queries, what ``paged_attention_fp8`` needs)."""
        return append_step([self], query, key, value, rope=rope, query_norm=query_norm, key_norm=key_norm)


def append_step(slots: list, query, key, value, *, rope=None, query_norm=None, key_norm=None) -> tuple[torch.Tensor, Fp8KvMetadata]:
    """One launch for a step of all ``slots`` (``Fp8KvPagedCache``, or None where idle) of one pool; all or nothing."""
    live = [s for s in slots if s is not None]
    if not live:
        raise ValueError("Cannot build paged metadata without active requests")
    pool = live[0].pool
    if any(not isinstance(s, Fp8KvPagedCache) or s.pool is not pool for s in live):
        raise ValueError("Paged batch caches must share one page pool")
    if query.dim() != 4 or key.dim() != 4 or key.shape != value.shape or key.shape[0] != len(slots) or min(key.shape) <= 0:
        raise ValueError("K/V chunks must be 4D [B, H, S, D], a row for every slot")
    heads, count, dim = key.shape[1:]
    theirs, mine = pool._snapshot_state(), [s._snapshot_state() for s in live]
    try:
        for s in live:
            room = s.page_size - s.page_lens[-1] if s.page_ids else 0
            pool.ensure_room(max(0, -(-(count - room) // s.page_size)), heads, dim, key.device)
            s.append_slots(count)
        # table and lengths side by side: one copy, which nobody waits for (the host would else wait for the device in every layer)
        width = max(s.num_pages for s in live)
        both = np.full((width + 1) * len(slots), -1, dtype=np.int32)
        table, lens = both[: width * len(slots)].reshape(len(slots), width), both[width * len(slots) :]
        lens[:] = 0
        for b, s in enumerate(slots):
            if s is not None:
                table[b, : s.num_pages], lens[b] = s.page_ids, s.offset
        there = torch.from_numpy(both).to(key.device, non_blocking=True)
        meta = Fp8KvMetadata(pool.pages, there[: width * len(slots)].view(len(slots), width), there[width * len(slots) :], table, lens)
        out = rotate_append_fp8(query, key, value, pool.pages, meta.block_table, meta.context_lens, rope=rope, query_norm=query_norm, key_norm=key_norm, block_table_host=table,
                                context_lens_host=lens)
    except Exception:
        pool._restore_state(theirs)
        for s, state in zip(live, mine):
            s._restore_state(state)
        raise
    return out, meta
