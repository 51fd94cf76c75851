"""The pages of a latent cache: append, store, extend, fork, free, compact and copy, and the plan of
a step over them.

A pool is one or more caches [num_pages, page_size, ...] that share their page ids (latent,
rotary and index keys; the layers of a model), and int32 state on the device:

* ``block_table`` [slots, max_blocks]: page of each block of a sequence, -1 where it has none
  (what ``flash_attention_paged``, ``sparse_flash_attention_triton`` and
  ``lightning_indexer_paged`` read),
* ``seq_lengths`` [slots]: tokens of each sequence, 0 for an empty slot,
* ``ref_counts`` [num_pages]: sequences that hold a page, 0 for a free one.

The calls that change the state read it and return a new one; the data of the pages is moved in
place.  None waits for the GPU.  Free pages are taken lowest id first.  A request that cannot be
met (an id out of range, a slot in use, a length past the block table, no page left) leaves its
sequence as it was and is reported by ``check_device_errors``.  No counterpart in the reference,
whose paged layout takes the table as given (sparse_flash_attention_triton.py:393-402).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _host as H
from ._lib import (APPEND_MAX_ENTRIES, BIND_APPEND, BIND_PLAN, BIND_STORE, BIND_UPKEEP, BatchPlanParams, CacheStoreParams, DSA_DTYPE_BF16, DSA_DTYPE_FP16, DSA_DTYPE_FP32, PAGES_COMPACT, PAGES_COPY,
                   PAGES_EXTEND, PAGES_FORK, PAGES_FREE, ROTARY_CODES, CacheAppendParams, PageCache,
                   PagesParams, binding, check, lib, ptr, remember, report_ptr)

_ROTATED = {torch.bfloat16: DSA_DTYPE_BF16, torch.float16: DSA_DTYPE_FP16, torch.float32: DSA_DTYPE_FP32}


def _int32(t, what, dim, dev):
    """A contiguous int32 device tensor of `dim` dims."""
    if not torch.is_tensor(t) or t.dtype != torch.int32 or t.dim() != dim:
        raise ValueError(f"{what} must be an int32 tensor of {dim} dim{'s' if dim > 1 else ''}")
    H.require_cuda(t)
    if t.device != dev:
        raise ValueError("all tensors must be on one device")
    return t.contiguous()


def _row_bytes(t: torch.Tensor, first: int, what: str) -> int:
    """Bytes of the contiguous trailing dims from `first` on."""
    width = 1
    for i in range(t.dim() - 1, first - 1, -1):
        if t.shape[i] > 1 and t.stride(i) != width:
            raise ValueError(f"{what} needs contiguous rows")
        width *= t.shape[i]
    return width * t.element_size()


def _page_strides(t: torch.Tensor, row: int, what: str):
    """(page, row) strides in bytes; rows, strides and base are whole 16-byte pieces."""
    size = t.element_size()
    row_stride = t.stride(1) * size if t.shape[1] > 1 else row
    page_stride = t.stride(0) * size if t.shape[0] > 1 else row_stride * t.shape[1]
    if row < 16 or row % 16 or row_stride % 16 or page_stride % 16:
        raise ValueError(f"{what} needs rows and strides of whole 16-byte pieces")
    if H.self_overlap(t):
        raise ValueError(f"{what} must not be an expanded tensor")
    return page_stride, row_stride


def _check_caches(caches, dev, num_pages=None):
    """(num_pages, page_size) that all caches share."""
    page_size = None
    for i, c in enumerate(caches):
        if c.dim() < 3:
            raise ValueError(f"cache {i} must be [num_pages, page_size, ...]")
        H.require_cuda(c)
        if c.device != dev:
            raise ValueError("all tensors must be on one device")
        num_pages = c.shape[0] if num_pages is None else num_pages
        page_size = c.shape[1] if page_size is None else page_size
        if c.shape[0] != num_pages or c.shape[1] != page_size:
            raise ValueError(f"cache {i} is {tuple(c.shape[:2])}, expected pages of {(num_pages, page_size)}")
    if num_pages is not None and num_pages < 1 or page_size is not None and page_size < 1:
        raise ValueError("the caches must not be empty")
    return num_pages, page_size


def _append_plan(tokens, caches, block_table, starts, counts, table, rotary):
    """Check the arguments and fill in what their shapes decide: (parameters, which tokens have
    to be copied first)."""
    if not 1 <= len(tokens) <= APPEND_MAX_ENTRIES or len(tokens) != len(caches):
        raise ValueError(f"tokens and caches must be lists of equal length, 1..{APPEND_MAX_ENTRIES}")
    if len(rotary) != len(tokens):
        raise ValueError("rotary must have one entry per cache")
    H.require_cuda(*tokens, *caches, block_table)
    dev = caches[0].device
    if tokens[0].dim() != 4:
        raise ValueError("tokens must be [B, S, 1, width]")
    B, S = tokens[0].shape[:2]
    num_pages, page_size = _check_caches(caches, dev)
    bt = _int32(block_table, "block_table", 2, dev)
    if bt.shape[0] != B or bt.shape[1] < 1:
        raise ValueError("block_table must be [B, max_blocks]")
    if _int32(starts, "starts", 1, dev).numel() != B or (
            counts is not None and _int32(counts, "counts", 1, dev).numel() != B):
        raise ValueError(f"starts and counts must have {B} entries")
    p = CacheAppendParams()
    if any(r is not None for r in rotary):
        if table is None:
            raise ValueError("rotary rows need a table (rotary_table)")
        if table.dim() != 2 or table.dtype != torch.float32 or table.shape[0] < 1:
            raise ValueError("table must be a float32 [max_positions, dim] tensor (rotary_table)")
        H.require_cuda(table)
        if table.device != dev:
            raise ValueError("all tensors must be on one device")
        dim = table.shape[1]
        if dim % 8 or not 8 <= dim <= 256:
            raise ValueError(f"the table's dim must be a multiple of 8 up to 256, got {dim}")
        p.max_positions, p.dim = table.shape[0], dim
    copy = []
    for i, (t, c, r) in enumerate(zip(tokens, caches, rotary)):
        if t.dim() != 4 or c.dim() != 4 or t.shape[:3] != (B, S, 1) or c.shape[2] != 1 \
                or t.shape[3] != c.shape[3]:
            raise ValueError(f"tokens {i} must be {(B, S, 1, c.shape[-1])}, got {tuple(t.shape)}")
        if t.dtype != c.dtype or t.device != dev:
            raise ValueError(f"tokens {i} must have its cache's dtype and device")
        size, width = c.element_size(), c.shape[3]
        row = _row_bytes(c, 2, f"cache {i}")
        e = p.rows[i]
        e.page_stride, e.row_stride = _page_strides(c, row, f"cache {i}")
        e.width_bytes = row
        fits = (width == 1 or t.stride(3) == 1) and not any(
            t.shape[d] > 1 and t.stride(d) * size % 16 for d in (0, 1))
        copy.append(not fits)
        steps = t.stride()[:2] if fits else (S * width, width)
        e.src_batch_stride = steps[0] * size if B > 1 else 0
        e.src_token_stride = steps[1] * size if S > 1 else 0
        if r is not None:
            layout, offset = r
            if layout not in ("interleaved", "half"):
                raise ValueError(f"unsupported rotary layout {layout!r}")
            if c.dtype not in _ROTATED:
                raise ValueError(f"rotated rows must be bf16, fp16 or fp32, got {c.dtype}")
            step = 16 // size
            if offset < 0 or offset % step or offset + dim > width \
                    or dim % (2 * step if layout == "half" else step):
                raise ValueError(f"offset {offset} and dim {dim} must be whole 16-byte pieces "
                                 f"within {width} values")
            e.rotary, e.offset, e.dtype = ROTARY_CODES[layout], int(offset), _ROTATED[c.dtype]
    p.batch, p.s, p.num_pages, p.page_size = B, S, num_pages, page_size
    p.max_blocks, p.entries = bt.shape[1], len(tokens)
    return bytes(p), copy


def paged_cache_append(tokens, caches, block_table, starts, counts=None, table=None, rotary=None):
    """Write new tokens into their pages, in up to four caches at once; returns ``caches``.

    ``tokens[i]`` [B, S, 1, width] goes into ``caches[i]`` [num_pages, page_size, 1, width] of the
    same dtype: token s < ``counts[b]`` (default S) of batch b to position ``starts[b]`` + s, by
    ``block_table`` [B, max_blocks].  ``rotary[i]`` is None or (layout, offset): those rows are
    rotated on the way by ``table`` (:func:`rotary_table`) at their position, as
    ``rotary_embedding`` would.  A token without a page, or past the table, is left out and
    reported.  Rows are whole 16-byte pieces; neither the tokens nor two caches share memory with
    rows that are written.
    """
    tokens, caches = list(tokens), list(caches)
    args = (tokens, caches, block_table, starts, counts, table, rotary)
    fast = binding()
    if fast is not None and fast.append(*args):
        return caches
    rotary = [None] * len(tokens) if rotary is None else list(rotary)
    template, copy = _append_plan(tokens, caches, block_table, starts, counts, table, rotary)
    index = caches[0].get_device()
    if H.current_device() != index:
        with torch.cuda.device(index):
            return paged_cache_append(tokens, caches, block_table, starts, counts, table, rotary)
    p = CacheAppendParams.from_buffer_copy(template)
    keep = []
    for e, t, c, again in zip(p.rows, tokens, caches, copy):
        src, dst = t.data_ptr(), c.data_ptr()
        if again or src % 16:
            t = t.clone(memory_format=torch.contiguous_format)
            keep.append(t)
            src, size = t.data_ptr(), t.element_size()
            e.src_batch_stride, e.src_token_stride = t.stride(0) * size, t.stride(1) * size
        if dst % 16:
            raise ValueError("caches need 16-byte aligned bases")
        e.src, e.cache = src, dst
    if p.dim:
        table = table.contiguous()
        if table.data_ptr() % 16:
            table = table.clone()
        p.table = table.data_ptr()
    bt, st = block_table.contiguous(), starts.contiguous()
    ct = None if counts is None else counts.contiguous()
    p.block_table, p.starts, p.counts = bt.data_ptr(), st.data_ptr(), ptr(ct)
    p.error_flag = report_ptr(index)
    check(lib().dsa_cache_append(p, H.raw_stream(index)), "dsa_cache_append")
    if not keep and bt is block_table and st is starts and ct is counts \
            and (table is args[5] or not p.dim):
        remember(BIND_APPEND, index, *args, template, b"", 0)
    return caches


def _pool_plan(op, caches, block_table, seq_lengths, ref_counts, first, second, page_size):
    """Check the arguments of an upkeep call and fill in what their shapes decide: (parameters,
    the caches' array, workspace bytes)."""
    copy = op == PAGES_COPY
    if copy:
        if not caches:
            raise ValueError("paged_cache_copy needs at least one cache")
        dev = caches[0].device
        num_pages = None
    else:
        H.require_cuda(block_table)
        dev = block_table.device
        bt = _int32(block_table, "block_table", 2, dev)
        num_pages = _int32(ref_counts, "ref_counts", 1, dev).numel()
        if bt.numel() == 0 or num_pages == 0:
            raise ValueError("block_table and ref_counts must not be empty")
        if op != PAGES_COMPACT and _int32(seq_lengths, "seq_lengths", 1, dev).numel() != bt.shape[0]:
            raise ValueError(f"seq_lengths must have {bt.shape[0]} entries, got {seq_lengths.numel()}")
    num_pages, size = _check_caches(caches, dev, num_pages)
    if size is not None and page_size is not None and size != page_size:
        raise ValueError(f"page_size {page_size} does not match the caches' {size}")
    size = page_size if size is None else size
    if size is None:
        if op in (PAGES_FORK, PAGES_EXTEND):
            raise ValueError("page_size is required without caches")
        size = 1   # not looked at
    if size < 1:
        raise ValueError(f"page_size must be positive, got {size}")
    p = PagesParams()
    p.op, p.num_pages, p.page_size, p.num_caches = op, num_pages, size, len(caches)
    if op != PAGES_COMPACT:
        names = {PAGES_COPY: ("src_pages", "dst_pages"), PAGES_FORK: ("parents", "children"),
                 PAGES_EXTEND: ("counts", ""), PAGES_FREE: ("rows", "")}[op]
        p.n = _int32(first, names[0], 1, dev).numel()
        if second is not None and _int32(second, names[1], 1, dev).numel() != p.n:
            raise ValueError(f"{names[0]} and {names[1]} must have equal lengths")
        if op == PAGES_EXTEND and p.n != bt.shape[0]:
            raise ValueError(f"counts must have {bt.shape[0]} entries, got {p.n}")
    if not copy:
        p.slots, p.max_blocks = bt.shape
        p.workspace_bytes = lib().dsa_pages_workspace_size(op, p.n, p.slots, num_pages)
    array = (PageCache * len(caches))()
    for i, (e, c) in enumerate(zip(array, caches)):
        e.row_bytes = _row_bytes(c, 2, f"cache {i}")
        e.page_stride, e.row_stride = _page_strides(c, e.row_bytes, f"cache {i}")
    return bytes(p), bytes(array), max(p.workspace_bytes, 4)


def _upkeep(op, caches, block_table=None, seq_lengths=None, ref_counts=None, first=None, second=None,
            page_size=None):
    """Run one call of ``dsa_pages``; returns the new (block_table, seq_lengths, ref_counts)."""
    page_size = None if page_size is None else int(page_size)
    state = (block_table, seq_lengths, ref_counts)
    args = (op, caches, *state, first, second, page_size)
    fast = binding()
    if fast is not None:
        done = fast.upkeep(*args)
        if done is not None:
            return done
    template, cache_template, ws_bytes = _pool_plan(op, caches, *state, first, second, page_size)
    lead = caches[0] if block_table is None else block_table
    index = lead.get_device()
    if H.current_device() != index:
        with torch.cuda.device(index):
            return _upkeep(op, caches, *state, first, second, page_size)
    p = PagesParams.from_buffer_copy(template)
    out = [None, None, None]
    if op != PAGES_COPY:
        state = [None if t is None else t.contiguous() for t in state]
        out = [None if t is None else torch.empty_like(t) for t in state]
        p.block_table, p.seq_lengths, p.ref_counts = [ptr(t) for t in state]
        p.block_table_out, p.seq_lengths_out, p.ref_counts_out = [ptr(t) for t in out]
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=lead.device)
        p.workspace = ws.data_ptr()
    if first is not None:
        first = first.contiguous()
        p.first = first.data_ptr()
    if second is not None:
        second = second.contiguous()
        p.second = second.data_ptr()
    if caches:
        array = (PageCache * len(caches)).from_buffer_copy(cache_template)
        for e, c in zip(array, caches):
            e.data = c.data_ptr()
            if e.data % 16:
                raise ValueError("caches need 16-byte aligned bases")
        p.caches = array
    p.error_flag = report_ptr(index)
    check(lib().dsa_pages(p, H.raw_stream(index)), "dsa_pages")
    if all(a is b for a, b in zip(args[2:7], (*state, first, second))):
        remember(BIND_UPKEEP, index, *args, template, cache_template, ws_bytes)
    return tuple(out)


def paged_cache_copy(caches, src_pages, dst_pages):
    """Copy pages ``src_pages[i]`` [n] to ``dst_pages[i]`` in every cache (a negative id skips the
    pair); returns ``caches``.  No page may be both written and read, or written twice."""
    caches = list(caches)
    _upkeep(PAGES_COPY, caches, first=src_pages, second=dst_pages)
    return caches


def paged_cache_extend(block_table, seq_lengths, ref_counts, counts, page_size):
    """Grow sequence r by ``counts[r]`` [slots] tokens, with the pages that takes.  Rows are served
    in order; one that the pages left cannot serve takes none of them, and those after it are
    served all the same.  Returns the new (block_table, seq_lengths, ref_counts)."""
    return _upkeep(PAGES_EXTEND, [], block_table, seq_lengths, ref_counts, counts, page_size=page_size)


def paged_cache_fork(caches, block_table, seq_lengths, ref_counts, parents, children, page_size=None):
    """Make the empty slots ``children[i]`` [n] copies of the sequences ``parents[i]``: they share
    the parents' full pages, and a partly filled last page is copied (its filled rows, in every
    cache) to a page of the child's own.  A full block without a page in the parent has none in the
    child and is reported.  Returns the new (block_table, seq_lengths, ref_counts).  ``page_size`` is
    needed where ``caches`` is empty."""
    return _upkeep(PAGES_FORK, list(caches), block_table, seq_lengths, ref_counts, parents, children,
                   page_size)


def paged_cache_free(block_table, seq_lengths, ref_counts, rows):
    """Empty the slots ``rows`` [n]: their pages lose one holder each.  Returns the new
    (block_table, seq_lengths, ref_counts)."""
    return _upkeep(PAGES_FREE, [], block_table, seq_lengths, ref_counts, rows)


def paged_cache_compact(caches, block_table, ref_counts):
    """Move the live pages to the lowest ids, so that the pool's tail is free: the k-th live page
    past the first n_live ids goes to the k-th free id among those, in every cache.  Returns the
    new (block_table, ref_counts)."""
    out = _upkeep(PAGES_COMPACT, list(caches), block_table, None, ref_counts)
    return out[0], out[2]


def _store_plan(tokens, caches, slot_map):
    """Check the arguments and fill in what their shapes decide: (parameters, which tokens have to be
    copied first)."""
    if not 1 <= len(tokens) <= APPEND_MAX_ENTRIES or len(tokens) != len(caches):
        raise ValueError(f"tokens and caches must be lists of equal length, 1..{APPEND_MAX_ENTRIES}")
    if not torch.is_tensor(slot_map) or slot_map.dtype not in (torch.int64, torch.int32) or slot_map.dim() != 1:
        raise ValueError("slot_map must be an int64 or int32 tensor of 1 dim")
    H.require_cuda(*tokens, *caches, slot_map)
    dev, T = caches[0].device, slot_map.numel()
    if slot_map.device != dev:
        raise ValueError("all tensors must be on one device")
    p = CacheStoreParams()
    p.num_pages, p.page_size = _check_caches(caches, dev)
    p.tokens, p.entries = T, len(tokens)
    copy = []
    for i, (t, c) in enumerate(zip(tokens, caches)):
        if t.dim() != 3 or c.dim() != 4 or c.shape[2] != 1 or tuple(t.shape) != (T, 1, c.shape[3]):
            raise ValueError(f"tokens {i} must be {(T, 1, c.shape[-1])}, got {tuple(t.shape)}")
        if t.dtype != c.dtype or t.device != dev:
            raise ValueError(f"tokens {i} must have its cache's dtype and device")
        row, size = _row_bytes(c, 2, f"cache {i}"), c.element_size()
        e = p.rows[i]
        e.page_stride, e.row_stride = _page_strides(c, row, f"cache {i}")
        e.width_bytes = row
        copy.append(c.shape[3] > 1 and t.stride(2) != 1 or T > 1 and t.stride(0) * size % 16 != 0)
        e.src_token_stride = row if copy[-1] or T == 1 else t.stride(0) * size
    return bytes(p), copy


def paged_cache_store(tokens, caches, slot_map):
    """Write packed tokens to their slots, in up to four caches at once; returns ``caches``.

    ``tokens[i]`` [T, 1, width] goes into ``caches[i]`` [num_pages, page_size, 1, width] of the same
    dtype: token t to row ``slot_map[t]`` (int64 or int32) % page_size of page ``slot_map[t]`` //
    page_size, as ``paged_batch_plan`` makes them.  A negative slot leaves its token out; so does one
    past the pool, which is reported.  No two tokens have one slot; rows are whole 16-byte pieces, and
    neither the tokens nor two caches share memory with rows that are written.
    """
    tokens, caches = list(tokens), list(caches)
    args = (tokens, caches, slot_map)
    fast = binding()
    if fast is not None and fast.store(*args):
        return caches
    template, copy = _store_plan(tokens, caches, slot_map)
    index = caches[0].get_device()
    if H.current_device() != index:
        with torch.cuda.device(index):
            return paged_cache_store(tokens, caches, slot_map)
    p = CacheStoreParams.from_buffer_copy(template)
    keep = []
    for e, t, c, again in zip(p.rows, tokens, caches, copy):
        if again or t.data_ptr() % 16:
            t = t.clone(memory_format=torch.contiguous_format)
            keep.append(t)
            e.src_token_stride = e.width_bytes
        if c.data_ptr() % 16:
            raise ValueError("caches need 16-byte aligned bases")
        e.src, e.cache = t.data_ptr(), c.data_ptr()
    slots = slot_map.to(torch.int64).contiguous()
    p.slots = slots.data_ptr()
    p.error_flag = report_ptr(index)
    check(lib().dsa_cache_store(p, H.raw_stream(index)), "dsa_cache_store")
    if not keep and slots is slot_map:
        remember(BIND_STORE, index, *args, template, b"", 0)
    return caches


class PagedBatchPlan(NamedTuple):
    """What :func:`paged_batch_plan` makes; int32, but for ``slot_map``."""
    block_table: torch.Tensor      # [B, max_blocks]
    key_lengths: torch.Tensor      # [B]
    query_ends: torch.Tensor       # [B] new tokens up to the request's last (TND lengths)
    token_rows: torch.Tensor       # [T] request of each token, -1 behind the last
    positions: torch.Tensor        # [T], 0 behind the last
    slot_map: torch.Tensor         # [T] int64, -1 behind the last
    group_starts: torch.Tensor     # [max_groups + 1]
    prefix_lengths: torch.Tensor   # [max_groups]


def _batch_plan(block_table, seq_lengths, rows, counts, page_size, num_tokens, max_groups, min_prefix):
    """Check the arguments and fill in what their shapes decide."""
    H.require_cuda(block_table)
    dev = block_table.device
    bt = _int32(block_table, "block_table", 2, dev)
    if bt.numel() == 0:
        raise ValueError("block_table must not be empty")
    if _int32(seq_lengths, "seq_lengths", 1, dev).numel() != bt.shape[0]:
        raise ValueError(f"seq_lengths must have {bt.shape[0]} entries, got {seq_lengths.numel()}")
    batch = _int32(rows, "rows", 1, dev).numel()
    if _int32(counts, "counts", 1, dev).numel() != batch:
        raise ValueError(f"counts must have {batch} entries (as rows has), got {counts.numel()}")
    for value, name, least in ((page_size, "page_size", 1), (num_tokens, "num_tokens", 0), (max_groups, "max_groups", 0),
                               (min_prefix, "min_prefix", 0)):
        if not least <= value <= 0x7fffffff:
            raise ValueError(f"{name} must be {least}..{0x7fffffff}, got {value}")
    if bt.shape[1] * page_size > 0x7fffffff:
        raise ValueError(f"{bt.shape[1]} blocks of {page_size} tokens pass 32 bits")
    p = BatchPlanParams()
    p.batch, p.page_size, p.num_tokens = batch, page_size, num_tokens
    p.slots, p.max_blocks = bt.shape
    p.max_groups, p.min_prefix = max_groups, min_prefix
    p.workspace_bytes = lib().dsa_batch_plan_workspace_size(batch)
    return bytes(p)


def paged_batch_plan(block_table, seq_lengths, rows, counts, page_size, num_tokens, max_groups=None, min_prefix=1):
    """The plan of a step, from the lengths of its requests, without waiting for them: request b is slot
    ``rows[b]`` [B] of the pool's state with ``counts[b]`` new tokens, which ``seq_lengths`` counts
    already (``paged_cache_extend``).  Returns a :class:`PagedBatchPlan`:

    * ``block_table``, ``key_lengths``: the requests' pages (-1 behind their lengths) and lengths, for
      attention and the indexer;
    * ``query_ends``: the new tokens up to each request's last, the cumulative lengths of TND calls;
    * ``token_rows``, ``positions``, ``slot_map``: of the ``num_tokens`` places of the packed new tokens,
      one request behind another, the request, the position (for ``rotary_embedding``) and the slot, page *
      page_size + row (for ``paged_cache_store``); -1, 0 and -1 behind the last token;
    * ``group_starts``, ``prefix_lengths``: groups of neighbouring requests with at least
      max(``min_prefix``, page_size) tokens in common, in whole pages that both had before this step (for
      ``flash_attention_shared_prefix``); a request that shares less with the one before it begins a
      group.  The first ``max_groups`` (default B) are listed.

    A request that cannot be (a slot out of range, a count past its length) has length 0, and its tokens
    keep their places, with -1, 0 and -1 as behind the last; a token without a page has slot -1, and tokens
    past ``num_tokens`` are left out; all are reported by ``check_device_errors``.  A slot that is in ``rows``
    twice with new tokens gives them the same places of the cache twice, which ``paged_cache_store`` does not take.
    """
    page_size, num_tokens, min_prefix = int(page_size), int(num_tokens), int(min_prefix)
    if max_groups is None:
        max_groups = rows.numel() if torch.is_tensor(rows) else 0
    max_groups = int(max_groups)
    args = (block_table, seq_lengths, rows, counts, page_size, num_tokens, max_groups, min_prefix)
    fast = binding()
    if fast is not None:
        done = fast.plan(*args)
        if done is not None:
            return PagedBatchPlan(*done)
    template = _batch_plan(*args)
    index = block_table.get_device()
    if H.current_device() != index:
        with torch.cuda.device(index):
            return paged_batch_plan(*args)
    p = BatchPlanParams.from_buffer_copy(template)
    given = [t.contiguous() for t in (block_table, seq_lengths, rows, counts)]
    p.block_table, p.seq_lengths, p.rows, p.counts = [t.data_ptr() for t in given]
    batch = p.batch
    make = lambda *shape, dtype=torch.int32: torch.empty(shape, dtype=dtype, device=block_table.device)
    plan = PagedBatchPlan(make(batch, block_table.shape[1]), make(batch), make(batch), make(num_tokens), make(num_tokens),
                          make(num_tokens, dtype=torch.int64), make(max_groups + 1), make(max_groups))
    ws_bytes = max(p.workspace_bytes, 4)
    ws = make(ws_bytes, dtype=torch.uint8)
    p.block_table_out, p.key_lengths, p.query_ends = [t.data_ptr() for t in plan[:3]]
    p.token_rows, p.positions, p.slot_map = [t.data_ptr() for t in plan[3:6]]
    p.group_starts, p.prefix_lengths = [t.data_ptr() for t in plan[6:]]
    p.workspace = ws.data_ptr()
    p.error_flag = report_ptr(index)
    check(lib().dsa_batch_plan(p, H.raw_stream(index)), "dsa_batch_plan")
    if all(a is b for a, b in zip(args, given)):
        remember(BIND_PLAN, index, *args, template, b"", ws_bytes)
    return plan
