"""flash_attention_paged: attention of new tokens over the whole paged latent cache, and
flash_attention_shared_prefix: the same for a batch whose rows share their first pages.

The dense counterpart of ``sparse_flash_attention_triton`` with ``layout_kv="PA_BSND"``
(sparse_flash_attention_triton.py:483-641): every visible key of a sequence is attended, so
there are no indices.  It serves decode steps of contexts that are no longer than the
indexer's top-k, and layers without an indexer.  No counterpart in the reference.  MLA-absorb,
one key head: value = key_cache[..., :D].
"""
from __future__ import annotations

import torch

from . import _host as H
from ._lib import (BIND_ATTN, BIND_SHARED, AttnPagedParams, AttnSharedParams, binding, check, lib, remember,
                   report_ptr)

_VALID_D = (128, 256, 512)
_D_ROPE = 64
# Cycles of one multiprocessor that sharing has to save, as it takes two launches more, one of them to
# be waited for, and a larger join: times 19, 20 and 14 at D = 512, 256 and 128.  Of 300 calls of 4 to 64 rows, 8 to
# 80 heads and 1024 to 32768 shared keys 61 save more: 57 gain up to 18 us, 4 lose, 1.8 us of 36 at most.  With
# nothing saved sharing would cost 9 to 14 us.
_LEAST_SAVING = 250000
_LEAST_TIMES = {128: 14, 256: 20, 512: 19}
_MAX_SCALE = torch.finfo(torch.float32).max


def _tma_strides(t: torch.Tensor):
    """Strides over (batch, token, head) if TMA can address the tensor (contiguous last dim,
    16-byte steps), else None.  A size-1 dim's own stride means nothing."""
    if t.stride(-1) != 1 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in (0, 1, 2)):
        return None
    return [t.stride(i) if t.shape[i] > 1 else t.shape[-1] for i in (0, 1, 2)]


def _cache_strides(t: torch.Tensor, what: str):
    """Strides over (page, row) of a cache [num_pages, page_size, 1, width]; a cache is never
    copied, so one that TMA cannot address is refused."""
    if t.stride(-1) != 1 or any(t.shape[i] > 1 and t.stride(i) % 8 for i in (0, 1)):
        raise ValueError(f"{what} needs a contiguous last dim and 16-byte strides")
    width = t.shape[-1]
    row = t.stride(1) if t.shape[1] > 1 else width
    return (t.stride(0) if t.shape[0] > 1 else row * t.shape[1]), row


def _plan(query, query_rope, key_cache, key_rope_cache, block_table, scale_value, sparse_mode, counted):
    """Check the arguments and fill in what their shapes decide: (parameters, strides fit,
    statistics' shape, workspace bytes).  `counted`: with a count of queries per sequence."""
    if sparse_mode not in (0, 3):
        raise ValueError("Only sparse_mode 0 (full) / 3 (rightDownCausal) supported")
    if not abs(scale_value) <= _MAX_SCALE:
        raise ValueError(f"scale_value must be finite in float32, got {scale_value}")
    if query.dim() != 4 or query_rope.dim() != 4:
        raise ValueError("query and query_rope must be [B, S1, N1, D]")
    if key_cache.dim() != 4 or key_rope_cache.dim() != 4:
        raise ValueError("key_cache and key_rope_cache must be [num_pages, page_size, 1, D]")
    B, S1, N1, D = query.shape
    num_pages, page, n2, dk = key_cache.shape
    if D not in _VALID_D or dk != D:
        raise ValueError(f"query and key_cache must share a D of {_VALID_D}, got {D} and {dk}")
    if not 1 <= N1 <= 128:
        raise ValueError(f"N1 must be 1..128, got {N1}")
    if tuple(query_rope.shape) != (B, S1, N1, _D_ROPE):
        raise ValueError(f"query_rope must be {(B, S1, N1, _D_ROPE)}, got {tuple(query_rope.shape)}")
    if n2 != 1 or tuple(key_rope_cache.shape) != (num_pages, page, 1, _D_ROPE):
        raise ValueError("Only N2=1 (MQA) is supported, with key_rope_cache "
                         f"[num_pages, page_size, 1, {_D_ROPE}]")
    if num_pages < 1 or page < 8 or page % 8:
        raise ValueError(f"page_size ({page}) must be a multiple of 8 and the cache not empty")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != B \
            or block_table.shape[1] < 1:
        raise ValueError("block_table must be an int32 [B, max_blocks] tensor")
    dtype = H.dtype_code(query)
    if not query.dtype == query_rope.dtype == key_cache.dtype == key_rope_cache.dtype:
        raise ValueError("query, query_rope and the caches must share their dtype")
    H.require_cuda(query, query_rope, key_cache, key_rope_cache, block_table)
    if not all(t.device == query.device for t in (query_rope, key_cache, key_rope_cache, block_table)):
        raise ValueError("all tensors must be on one device")
    p = AttnPagedParams()
    p.k_page_stride, p.k_row_stride = _cache_strides(key_cache, "key_cache")
    p.kr_page_stride, p.kr_row_stride = _cache_strides(key_rope_cache, "key_rope_cache")
    qs, qrs = _tma_strides(query), _tma_strides(query_rope)
    # a few tokens share their keys if their heads lie one step apart; queries that lie otherwise
    # are copied rather than each token's keys read anew (with counts per sequence none share):
    # 32 x 2 tokens of 64 heads, D 256, 8192 .. 65536 keys: 194 us against 290 token by token
    # (178 without a copy); 8 x 2 of them over 500 .. 4000 keys: 39 against 28
    if N1 > 1 and not counted and lib().dsa_attn_paged_shares_keys(S1, N1):
        qs, qrs = [None if st is None or st[1] != N1 * st[2] else st for st in (qs, qrs)]
    contiguous = lambda w: (S1 * N1 * w, N1 * w, w)
    p.q_batch_stride, p.q_token_stride, p.q_head_stride = qs or contiguous(D)
    p.qr_batch_stride, p.qr_token_stride, p.qr_head_stride = qrs or contiguous(_D_ROPE)
    p.batch, p.s1, p.n1, p.d = B, S1, N1, D
    p.num_pages, p.page_size, p.max_blocks = num_pages, page, block_table.shape[1]
    p.scale, p.sparse_mode, p.dtype = scale_value, int(sparse_mode), dtype
    p.workspace_bytes = lib().dsa_attn_paged_workspace_size(B, S1, N1, D)
    return bytes(p), qs is not None, qrs is not None, (B, 1, S1, N1), max(p.workspace_bytes, 16)


def _copied(t: torch.Tensor) -> torch.Tensor:
    return t.clone(memory_format=torch.contiguous_format)


def _call(params, p, entry, name, tensors, stats, index, q_fits, qr_fits, stat_shape, ws_bytes):
    """Fill `p`, the attention's part of `params`, in and call the entry: (results, whether the tables
    and lengths went in as they were given)."""
    query, query_rope, key_cache, key_rope_cache, block_table, act_k_given, act_q_given = tensors
    dev = query.device
    B, _, S1, _ = stat_shape
    act_k, act_q = act_k_given, act_q_given
    if not H.is_i32_vector(act_k, B, index):
        act_k = H.lens_tensor(act_k, B, p.max_blocks * p.page_size, dev).contiguous()
    if act_q is not None and not H.is_i32_vector(act_q, B, index):
        act_q = H.lens_tensor(act_q, B, S1, dev).contiguous()
    out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    alloc = torch.empty if stats else torch.zeros
    smax = alloc(stat_shape, dtype=torch.float32, device=dev)
    ssum = alloc(stat_shape, dtype=torch.float32, device=dev)
    if B == 0 or S1 == 0:
        return (out, smax, ssum), False
    q = query if q_fits and query.data_ptr() % 16 == 0 else _copied(query)
    qr = query_rope if qr_fits and query_rope.data_ptr() % 16 == 0 else _copied(query_rope)
    if q is not query:
        p.q_batch_stride, p.q_token_stride, p.q_head_stride = q.stride()[:3]
    if qr is not query_rope:
        p.qr_batch_stride, p.qr_token_stride, p.qr_head_stride = qr.stride()[:3]
    kc, krc = key_cache.data_ptr(), key_rope_cache.data_ptr()
    if (kc | krc) % 16:
        raise ValueError("key_cache and key_rope_cache need 16-byte aligned bases")
    bt = block_table.contiguous()
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    p.query, p.query_rope, p.key_cache, p.key_rope_cache = q.data_ptr(), qr.data_ptr(), kc, krc
    p.block_table, p.act_k, p.out, p.workspace = bt.data_ptr(), act_k.data_ptr(), out.data_ptr(), ws.data_ptr()
    if act_q is not None:
        p.act_q = act_q.data_ptr()
    if stats:
        p.softmax_max, p.softmax_sum = smax.data_ptr(), ssum.data_ptr()
    p.error_flag = report_ptr(index)
    check(entry(params, H.raw_stream(index)), name)
    return (out, smax, ssum), bt is block_table and act_k is act_k_given and act_q is act_q_given


def flash_attention_paged(
    query: torch.Tensor,
    query_rope: torch.Tensor,
    key_cache: torch.Tensor,
    key_rope_cache: torch.Tensor,
    block_table: torch.Tensor,
    actual_seq_lengths_key=None,
    scale_value: float = 1.0,
    actual_seq_lengths_query=None,
    sparse_mode: int = 0,
    return_softmax_lse: bool = False,
):
    """Attention of ``query`` [B, S1, N1, D] (N1 1..128; D 128, 256 or 512; bf16 / fp16) and
    ``query_rope`` [B, S1, N1, 64] over ``key_cache`` [num_pages, page_size, 1, D] and
    ``key_rope_cache`` [num_pages, page_size, 1, 64], page_size a multiple of 8.

    ``block_table`` [B, max_blocks] int32: key position t of batch b is row t % page_size of
    page ``block_table[b, t // page_size]``; a negative entry holds no keys.
    ``actual_seq_lengths_key`` counts each batch's keys, the new tokens' own among them
    (default: max_blocks * page_size).  ``sparse_mode`` 0: every row of a batch sees all of
    its keys; 3: row s sees the keys before act_k - act_q + s + 1 (rightDownCausal).  Rows past
    ``actual_seq_lengths_query`` (default S1) and rows without keys give zeros.

    Returns (attention_out, softmax_max, softmax_sum); the statistics are (B, 1, S1, N1) fp32,
    zeros when ``return_softmax_lse`` is False.  Strided inputs (views of a joint projection or
    of a joint cache) are read in place.
    """
    args = (query, query_rope, key_cache, key_rope_cache, block_table, actual_seq_lengths_key,
            actual_seq_lengths_query, float(scale_value), sparse_mode, bool(return_softmax_lse))
    fast = binding()
    if fast is not None:
        done = fast.attn(*args)
        if done is not None:
            return done
    index = query.get_device()
    if index >= 0 and H.current_device() != index:
        with torch.cuda.device(index):
            return flash_attention_paged(query, query_rope, key_cache, key_rope_cache, block_table,
                                         actual_seq_lengths_key, scale_value, actual_seq_lengths_query,
                                         sparse_mode, return_softmax_lse)
    plan = _plan(query, query_rope, key_cache, key_rope_cache, block_table, float(scale_value), sparse_mode,
                 actual_seq_lengths_query is not None)
    template, q_fits, qr_fits, stat_shape, ws_bytes = plan
    p = AttnPagedParams.from_buffer_copy(template)
    done, as_given = _call(p, p, lib().dsa_attn_paged, "dsa_attn_paged", args[:7], bool(return_softmax_lse), index, *plan[1:])
    if as_given:
        remember(BIND_ATTN, index, *args, template, bytes((not q_fits, not qr_fits)), ws_bytes)
    return done


def _one_matrix(t: torch.Tensor, strides):
    """Whether all heads of a [B, S1, N1, D] tensor lie one step apart, across tokens and rows."""
    b, s, n, d = t.shape
    step = strides[2] if n > 1 else strides[1] if s > 1 else strides[0] if b > 1 else d
    return (s == 1 or strides[1] == n * step) and (b == 1 or strides[0] == s * n * step)


def _shared_plan(query, query_rope, key_cache, key_rope_cache, block_table, group_starts, prefix_lengths,
                 scale_value, sparse_mode, counted=True):
    """As _plan, for flash_attention_shared_prefix."""
    for t, what in ((group_starts, "group_starts"), (prefix_lengths, "prefix_lengths")):
        if not torch.is_tensor(t) or t.dtype != torch.int32 or t.dim() != 1:
            raise ValueError(f"{what} must be an int32 tensor of 1 dim")
    template, q_fits, qr_fits, stat_shape, _ = _plan(query, query_rope, key_cache, key_rope_cache, block_table, scale_value,
                                                     sparse_mode, counted)
    H.require_cuda(group_starts, prefix_lengths)
    if group_starts.device != query.device or prefix_lengths.device != query.device:
        raise ValueError("all tensors must be on one device")
    groups = prefix_lengths.numel()
    if group_starts.numel() != groups + 1:
        raise ValueError(f"group_starts must have {groups + 1} entries (one more than prefix_lengths), "
                         f"got {group_starts.numel()}")
    p = AttnSharedParams()
    p.attn = AttnPagedParams.from_buffer_copy(template)
    B, S1, N1, D = query.shape
    p.groups, p.least_saving = groups, _LEAST_SAVING * _LEAST_TIMES[D]
    if lib().dsa_attn_shared_looks(p, counted):
        # pieces of a prefix are runs of heads of neighbouring tokens; queries that lie otherwise are copied
        qs, qrs = _tma_strides(query), _tma_strides(query_rope)
        q_fits, qr_fits = [st is not None and _one_matrix(t, st) for t, st in ((query, qs), (query_rope, qrs))]
        contiguous = lambda w: (S1 * N1 * w, N1 * w, w)
        p.attn.q_batch_stride, p.attn.q_token_stride, p.attn.q_head_stride = qs if q_fits else contiguous(D)
        p.attn.qr_batch_stride, p.attn.qr_token_stride, p.attn.qr_head_stride = qrs if qr_fits else contiguous(_D_ROPE)
    p.attn.workspace_bytes = lib().dsa_attn_shared_workspace_size(B, S1, N1, D, groups)
    return bytes(p), q_fits, qr_fits, stat_shape, max(p.attn.workspace_bytes, 16)


def flash_attention_shared_prefix(
    query: torch.Tensor,
    query_rope: torch.Tensor,
    key_cache: torch.Tensor,
    key_rope_cache: torch.Tensor,
    block_table: torch.Tensor,
    group_starts: torch.Tensor,
    prefix_lengths: torch.Tensor,
    actual_seq_lengths_key=None,
    scale_value: float = 1.0,
    actual_seq_lengths_query=None,
    sparse_mode: int = 0,
    return_softmax_lse: bool = False,
):
    """:func:`flash_attention_paged` for a batch whose rows share their first pages in groups (forks
    of a sequence, requests with one system prompt): the keys that a group shares are read and
    multiplied once for as many of its tokens as 64 or 128 heads hold.

    ``group_starts`` [G + 1] int32, not decreasing, within 0 .. B: group g is the rows
    ``group_starts[g]`` .. ``group_starts[g + 1]`` - 1.  ``prefix_lengths`` [G] int32: the first
    tokens that all rows of the group have in common, for which their rows of ``block_table`` name
    the same pages (those of the group's first row with keys are read); whole pages are shared, at
    most as many as every row of the group with keys sees.  Rows outside all groups share
    nothing.  ``paged_batch_plan`` makes both.

    The other arguments and the results are those of :func:`flash_attention_paged`.  Whether a group's
    prefix is shared is decided on the GPU, by what that saves of the tokens that see a key (padding
    and idle rows are no work): nothing is where a token has more than 64 heads (it fills a piece by
    itself), or in calls that are small or whose tables are.  Where the tables are wide and nothing is
    shared in the end, a call takes 3 to 6 us more than :func:`flash_attention_paged` (up to 25 with 64
    rows of several tokens or of 64 heads).  G
    should be near the number of groups: the pieces are of 128 heads where B * S1 * N1 / G exceeds 64.
    Starts that divide no batch of B rows share nothing; where they are looked at they are
    reported by ``check_device_errors``.
    """
    args = (query, query_rope, key_cache, key_rope_cache, block_table, actual_seq_lengths_key, actual_seq_lengths_query,
            float(scale_value), sparse_mode, bool(return_softmax_lse), group_starts, prefix_lengths)
    fast = binding()
    if fast is not None:
        done = fast.shared(*args)
        if done is not None:
            return done
    index = query.get_device()
    if index >= 0 and H.current_device() != index:
        with torch.cuda.device(index):
            return flash_attention_shared_prefix(query, query_rope, key_cache, key_rope_cache, block_table,
                                                 group_starts, prefix_lengths, actual_seq_lengths_key, scale_value,
                                                 actual_seq_lengths_query, sparse_mode, return_softmax_lse)
    plan = _shared_plan(query, query_rope, key_cache, key_rope_cache, block_table, group_starts, prefix_lengths,
                        float(scale_value), sparse_mode, actual_seq_lengths_query is not None)
    template, q_fits, qr_fits, _, ws_bytes = plan
    p = AttnSharedParams.from_buffer_copy(template)
    starts, prefixes = group_starts.contiguous(), prefix_lengths.contiguous()
    p.group_starts, p.prefix_lengths = starts.data_ptr(), prefixes.data_ptr()
    done, as_given = _call(p, p.attn, lib().dsa_attn_shared, "dsa_attn_shared", args[:7], bool(return_softmax_lse),
                           index, *plan[1:])
    if as_given and starts is group_starts and prefixes is prefix_lengths:
        remember(BIND_SHARED, index, *args, template, bytes((not q_fits, not qr_fits)), ws_bytes)
    return done
