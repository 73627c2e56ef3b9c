"""A serving step over paged caches, driven from the device: pages from request lengths, new
rows into their slots, attention over block tables, and drafted tokens against the target's
probabilities. Lengths and tables stay on the device, so a captured step serves later ones.

The reference has the same steps for one sequence at a time, on the host (paramecia-model/src/
qwen3_next.rs: append_quantized :431-509, the SDPA :2492-2605, truncate and checkpoint hooks
:2755-2762, 4291-4375). Tensors are torch device tensors; every kernel is libpkv's.
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import lib
from .kv_cache import KvCacheError, _at, _call, _device, _past_32_bits, _stream, _take

_PAGES = {torch.float16: _lib.QUANT_F16, torch.bfloat16: _lib.QUANT_BF16}


@functools.lru_cache(maxsize=256)
def _attend_bytes(n: int, tokens: int, heads: int, kv_heads: int, dim: int) -> int:
    return lib().pkv_pages_attend_workspace(n, tokens, heads, kv_heads, dim)


@functools.lru_cache(maxsize=256)
def _verify_bytes(n: int, vocab: int) -> int:
    return lib().pkv_verify_drafts_workspace(n, vocab)


class PageMap(NamedTuple):
    """What map_pages gives: for each row of the step its slot (int64, -1: no row) and position,
    for each request its rows [starts[b], starts[b + 1]) and its keys, and the status: 0, or
    with nothing moved 1 (the stack lacks pages) or 3 (lengths that do not fit)."""
    slots: torch.Tensor
    positions: torch.Tensor
    starts: torch.Tensor
    totals: torch.Tensor
    status: torch.Tensor


def map_pages(lens: torch.Tensor, add: torch.Tensor, tables: torch.Tensor, held: torch.Tensor,
              free_pages: torch.Tensor, free_count: torch.Tensor, page_tokens: int,
              max_tokens: int, out: Optional[PageMap] = None) -> PageMap:
    """Request lengths to pages and slots (pkv_pages_map). lens, add: int32 [n], the tokens that
    each request keeps and gets; tables [n, max_pages], held [n], free_pages [capacity] and
    free_count [1], all int32, are updated: pages that a request no longer needs go back onto
    the stack, pages that it lacks come from its top. page_tokens: a power of two from 32 on.
    Returns the PageMap of a step of up to max_tokens rows (out: one to be written again)."""
    dev = _device()
    n = lens.shape[0] if lens.dim() == 1 else 0
    if n == 0 or tables.dim() != 2 or free_pages.dim() != 1:
        raise KvCacheError("map_pages expects lens [n], tables [n, max_pages] and free_pages [capacity]")
    max_pages, capacity = tables.shape[1], free_pages.shape[0]
    if (n | max_pages | capacity | page_tokens | max_tokens) >> 31:
        _past_32_bits("n, max_pages, capacity, page_tokens and max_tokens", n, max_pages, capacity, page_tokens, max_tokens)
    i32 = torch.int32
    lens, add = _take(lens, "lens", (n,), dev, i32), _take(add, "add", (n,), dev, i32)
    _take(tables, "tables", (n, max_pages), dev, i32, writes=True)
    _take(held, "held", (n,), dev, i32, writes=True)
    _take(free_pages, "free_pages", (capacity,), dev, i32, writes=True)
    _take(free_count, "free_count", (1,), dev, i32, writes=True)
    if out is None:
        slots, positions, starts, totals, status = lens.new_empty(3 * max_tokens + 2 * n + 2).split_with_sizes(
            (2 * max_tokens, max_tokens, n + 1, n, 1))
        out = PageMap(slots.view(torch.int64), positions, starts, totals, status)
    else:
        for t, name, size, dtype in zip(out, PageMap._fields, (max_tokens, max_tokens, n + 1, n, 1),
                                        (torch.int64, i32, i32, i32, i32)):
            _take(t, name, (size,), dev, dtype, writes=True)
    _call(lib().pkv_pages_map(lens.data_ptr(), add.data_ptr(), n, tables.data_ptr(), max_pages,
                              held.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
                              capacity, page_tokens, out.slots.data_ptr(),
                              out.positions.data_ptr(), max_tokens, out.starts.data_ptr(),
                              out.totals.data_ptr(), out.status.data_ptr(), _stream()))
    return out


def _planes(k_pages: torch.Tensor, v_pages: torch.Tensor, dev: int):
    """The pages' encoding and shape, refused unless both are contiguous pages of 16-bit rows."""
    quant = _PAGES.get(k_pages.dtype)
    if quant is None or k_pages.dim() != 4:
        raise KvCacheError("pages are float16 or bfloat16 [n_pages, page_tokens, kv heads, head_dim]")
    shape = k_pages.shape
    if (shape[0] | shape[1] | shape[2] | shape[3]) >> 31:
        _past_32_bits("the pages' sizes", *shape)
    _take(k_pages, "k_pages", shape, dev, k_pages.dtype, writes=True)
    _take(v_pages, "v_pages", shape, dev, k_pages.dtype, writes=True)
    return quant, shape


def append_pages(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_pages: torch.Tensor,
                 v_pages: torch.Tensor) -> None:
    """New rows into their slots (pkv_pages_append): k, v [tokens, kv heads, head_dim] f32 (any
    token stride: slices of a projection), slots int64 [tokens] as map_pages gives them (a
    negative one: no row); k_pages, v_pages [n_pages, page_tokens, kv heads, head_dim]."""
    dev = _device()
    quant, (n_pages, page, heads, dim) = _planes(k_pages, v_pages, dev)
    n = slots.numel()
    rows, strides = [], []
    for t, name in ((k, "k"), (v, "v")):
        if (t.get_device() != dev or t.dtype is not torch.float32 or t.shape != (n, heads, dim) or
                t.stride(2) != 1 or t.stride(1) != dim or (t.stride(0) < heads * dim and n > 1)):
            t = _take(t, name, (n, heads, dim), dev)
        rows.append(t)
        strides.append(t.stride(0) if n > 1 else heads * dim)
    slots = _take(slots, "slots", (n,), dev, torch.int64)
    _call(lib().pkv_pages_append(quant, rows[0].data_ptr(), rows[1].data_ptr(), strides[0], strides[1],
                                 slots.data_ptr(), n, k_pages.data_ptr(), v_pages.data_ptr(),
                                 n_pages * page, heads, dim, _stream()))


def attend_pages(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 tables: torch.Tensor, lens: torch.Tensor, scale: float,
                 starts: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of the new tokens of n requests over their pages (pkv_pages_attend): q
    [tokens, heads, head_dim] f32 (any token and head strides), request b's rows [starts[b],
    starts[b + 1]) (starts None: one row each), the last of its lens[b] keys, whose pages
    tables[b] names (int32 [n, max_pages]). window: how many keys up to its own a token sees (0:
    all), sinks: the first keys that it sees all the same. Returns out [tokens, heads, head_dim];
    rows of no request are left as they were (zeros if out is not given)."""
    dev = _device()
    expects = "attend_pages expects q [tokens, heads, head_dim], heads a multiple of the pages', and tables [n, max_pages]"
    if q.dim() != 3 or tables.dim() != 2:
        raise KvCacheError(expects)
    (tokens, heads, width), (n, max_pages) = q.shape, tables.shape
    if (window | sinks | n | max_pages | tokens | heads) >> 31:
        _past_32_bits("window, sinks, n, max_pages, tokens and heads", window, sinks, n, max_pages, tokens, heads)
    quant, (n_pages, page, kv_heads, dim) = _planes(k_pages, v_pages, dev)
    if width != dim or heads == 0 or kv_heads == 0 or heads % kv_heads:
        raise KvCacheError(expects)
    st, sh, sd = q.stride()
    if (q.get_device() != dev or q.dtype is not torch.float32 or sd != 1 or sh < dim or sh % 4 or st % 4 or
            st < (heads - 1) * sh + dim or q.data_ptr() % 16):
        _take(q, "q", q.shape, dev)
        q = q.clone(memory_format=torch.contiguous_format)
        st, sh, sd = q.stride()
    tables = _take(tables, "tables", (n, max_pages), dev, torch.int32)
    lens = _take(lens, "lens", (n,), dev, torch.int32)
    starts = _take(starts, "starts", (n + 1,), dev, torch.int32)
    if out is None:
        out = (torch.empty if starts is None else torch.zeros)((tokens, heads, dim), dtype=torch.float32, device=q.device)
    else:
        _take(out, "out", (tokens, heads, dim), dev, writes=True)
    need = _attend_bytes(n, tokens, heads, kv_heads, dim)
    # torch's allocator orders the workspace with the stream, and gives each graph its own
    ws = out.new_empty(need, dtype=torch.uint8) if need else None
    _call(lib().pkv_pages_attend(quant, q.data_ptr(), st, sh, k_pages.data_ptr(), v_pages.data_ptr(), n_pages,
                                 page, tables.data_ptr(), max_pages, lens.data_ptr(), _at(starts), n,
                                 tokens, heads, kv_heads, dim, scale, window, sinks, out.data_ptr(), _at(ws),
                                 need, _stream()))
    return out


def verify_drafts(target_probs: torch.Tensor, drafts: torch.Tensor, uniforms: torch.Tensor,
                  draft_probs: Optional[torch.Tensor] = None, n_drafts: Optional[torch.Tensor] = None):
    """Drafted tokens against the target's probabilities (pkv_verify_drafts): target_probs [n,
    k + 1, vocab] f32, drafts int32 [n, k], uniforms [n, k + 1] f32 in [0, 1), draft_probs [n, k,
    vocab] f32 (None: the drafts were certain, as a greedy drafter's are), n_drafts int32 [n]
    (None: k each). Returns (tokens [n, k + 1], accepted [n]) int32: the accepted drafts, the
    token that follows them, then -1. A request goes on with lens + accepted + 1 tokens."""
    dev = _device()
    if target_probs.dim() != 3 or target_probs.shape[1] == 0:
        raise KvCacheError("verify_drafts expects target_probs [n, k + 1, vocab]")
    n, rows, vocab = target_probs.shape
    k = rows - 1
    if (n | k | vocab) >> 31:
        _past_32_bits("n, k and vocab", n, k, vocab)
    target_probs = _take(target_probs, "target_probs", (n, rows, vocab), dev)
    draft_probs = _take(draft_probs, "draft_probs", (n, k, vocab), dev)
    drafts = _take(drafts, "drafts", (n, k), dev, torch.int32)
    uniforms = _take(uniforms, "uniforms", (n, rows), dev)
    n_drafts = _take(n_drafts, "n_drafts", (n,), dev, torch.int32)
    tokens, accepted = drafts.new_empty((n, rows)), drafts.new_empty(n)
    need = _verify_bytes(n, vocab)
    ws = drafts.new_empty(need, dtype=torch.uint8) if need else None
    _call(lib().pkv_verify_drafts(target_probs.data_ptr(), vocab, _at(draft_probs), vocab, drafts.data_ptr(),
                                  _at(n_drafts), uniforms.data_ptr(), n, k, vocab, tokens.data_ptr(),
                                  accepted.data_ptr(), _at(ws), need, _stream()))
    return tokens, accepted
