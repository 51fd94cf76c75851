"""flash_attention_paged: attention of new tokens over the whole paged latent cache.

The dense counterpart of ``sparse_flash_attention_triton`` with ``layout_kv="PA_BSND"``
(sparse_flash_attention_triton.py:483-641): every visible key of a sequence is attended, so
there are no indices.  It serves decode steps of contexts that are no longer than the
indexer's top-k, and layers without an indexer.  No counterpart in the reference.  MLA-absorb,
one key head: value = key_cache[..., :D].
"""
from __future__ import annotations

import torch

from . import _host as H
from ._lib import BIND_ATTN, AttnPagedParams, binding, check, lib, remember, report_ptr

_VALID_D = (128, 256, 512)
_D_ROPE = 64
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
    dev = query.device
    B, _, S1, _ = stat_shape
    p = AttnPagedParams.from_buffer_copy(template)
    act_k = actual_seq_lengths_key
    if not H.is_i32_vector(act_k, B, index):
        act_k = H.lens_tensor(act_k, B, p.max_blocks * p.page_size, dev).contiguous()
    act_q = actual_seq_lengths_query
    if act_q is not None and not H.is_i32_vector(act_q, B, index):
        act_q = H.lens_tensor(act_q, B, S1, dev).contiguous()
    out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    alloc = torch.empty if return_softmax_lse else torch.zeros
    smax = alloc(stat_shape, dtype=torch.float32, device=dev)
    ssum = alloc(stat_shape, dtype=torch.float32, device=dev)
    if B == 0 or S1 == 0:
        return out, smax, ssum
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
    if return_softmax_lse:
        p.softmax_max, p.softmax_sum = smax.data_ptr(), ssum.data_ptr()
    p.error_flag = report_ptr(index)
    check(lib().dsa_attn_paged(p, H.raw_stream(index)), "dsa_attn_paged")
    if bt is block_table and act_k is actual_seq_lengths_key and act_q is actual_seq_lengths_query:
        remember(BIND_ATTN, index, *args, template, bytes((not q_fits, not qr_fits)), ws_bytes)
    return out, smax, ssum
