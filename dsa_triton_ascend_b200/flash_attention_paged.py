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
from ._lib import AttnPagedParams, check, lib, ptr, report_flag, stream_ptr

_VALID_D = (128, 256, 512)
_D_ROPE = 64


def _strided(t: torch.Tensor, dims) -> tuple:
    """``t`` with a contiguous last dim, 16-byte steps and a 16-byte base (copied if it has
    none), and its strides over ``dims`` (a size-1 dim's own stride means nothing)."""
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
        t.shape[i] == 1 or t.stride(i) % 8 == 0 for i in dims)
    if not ok:
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    width = -(-t.shape[-1] // 8) * 8
    return t, [t.stride(i) if t.shape[i] > 1 else width for i in dims]


def _cache_strides(t: torch.Tensor, what: str):
    """Strides over (page, row) of a cache [num_pages, page_size, 1, width]; a cache is never
    copied, so one that TMA cannot address is refused."""
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(
            t.shape[i] > 1 and t.stride(i) % 8 for i in (0, 1)):
        raise ValueError(f"{what} needs a contiguous last dim, 16-byte strides and a 16-byte base")
    width = t.shape[-1]
    row = t.stride(1) if t.shape[1] > 1 else width
    return (t.stride(0) if t.shape[0] > 1 else row * t.shape[1]), row


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
    if sparse_mode not in (0, 3):
        raise ValueError("Only sparse_mode 0 (full) / 3 (rightDownCausal) supported")
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
    dev = query.device
    if not all(t.device == dev for t in (query_rope, key_cache, key_rope_cache, block_table)):
        raise ValueError("all tensors must be on one device")
    kp, kr = _cache_strides(key_cache, "key_cache")
    rp, rr = _cache_strides(key_rope_cache, "key_rope_cache")

    with torch.cuda.device(dev):
        max_blocks = block_table.shape[1]
        act_k = H.lens_tensor(actual_seq_lengths_key, B, max_blocks * page, dev).contiguous()
        act_q = None
        if actual_seq_lengths_query is not None:
            act_q = H.lens_tensor(actual_seq_lengths_query, B, S1, dev).contiguous()
        out = torch.empty((B, S1, N1, D), dtype=query.dtype, device=dev)
        alloc = torch.empty if return_softmax_lse else torch.zeros
        smax = alloc((B, 1, S1, N1), dtype=torch.float32, device=dev)
        ssum = alloc((B, 1, S1, N1), dtype=torch.float32, device=dev)
        if B == 0 or S1 == 0:
            return out, smax, ssum
        q, qs = _strided(query, (0, 1, 2))
        qr, qrs = _strided(query_rope, (0, 1, 2))
        bt = block_table.contiguous()
        ws_bytes = lib().dsa_attn_paged_workspace_size(B, S1, N1, D)
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
        p = AttnPagedParams()
        p.query, p.query_rope, p.key_cache, p.key_rope_cache = ptr(q), ptr(qr), ptr(key_cache), ptr(key_rope_cache)
        p.block_table, p.act_q, p.act_k, p.out = ptr(bt), ptr(act_q), ptr(act_k), ptr(out)
        if return_softmax_lse:
            p.softmax_max, p.softmax_sum = ptr(smax), ptr(ssum)
        p.error_flag = ptr(report_flag(dev))
        p.workspace, p.workspace_bytes = ptr(ws), ws_bytes
        p.batch, p.s1, p.n1, p.d = B, S1, N1, D
        p.num_pages, p.page_size, p.max_blocks = num_pages, page, max_blocks
        p.q_batch_stride, p.q_token_stride, p.q_head_stride = qs
        p.qr_batch_stride, p.qr_token_stride, p.qr_head_stride = qrs
        p.k_page_stride, p.k_row_stride = kp, kr
        p.kr_page_stride, p.kr_row_stride = rp, rr
        p.scale = float(scale_value)
        p.sparse_mode = int(sparse_mode)
        p.dtype = dtype
        check(lib().dsa_attn_paged(p, stream_ptr(dev)), "dsa_attn_paged")
    return out, smax, ssum
