"""ctypes binding of libdsa_b200.so (the sm_100a kernels).

The library is loaded from this package directory.  There is no fallback: if the
library is missing or cannot be loaded, every operator raises.
"""
from __future__ import annotations

import ctypes
import os
import threading

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libdsa_b200.so")

DSA_OK = 0
DSA_ERR_INVALID_ARG = 1
DSA_ERR_CUDA = 2
DSA_ERR_TMA_DESCRIPTOR = 3
DSA_ERR_TOO_LARGE = 4
SFA_FWD_NOALLOC_SCRATCH_BYTES = 16 << 20   # DSA_SFA_FWD_NOALLOC_SCRATCH_BYTES
DSA_DTYPE_BF16 = 0
DSA_DTYPE_FP16 = 1
DSA_DTYPE_FP32 = 2
DSA_DTYPE_FP8_E4M3 = 3

_ERR_TEXT = {
    DSA_ERR_INVALID_ARG: "invalid argument",
    DSA_ERR_CUDA: "CUDA launch error",
    DSA_ERR_TMA_DESCRIPTOR: "TMA descriptor rejected (misaligned or oversized tensor)",
    DSA_ERR_TOO_LARGE: "request exceeds the library's fixed scratch array",
}

_p = ctypes.c_void_p
_i64 = ctypes.c_int64


class SfaFwdParams(ctypes.Structure):
    _fields_ = [
        ("q", _p), ("q_rope", _p), ("key", _p), ("key_rope", _p),
        ("sparse_indices", _p), ("act_q", _p), ("act_k", _p), ("q_row_base", _p),
        ("k_row_base", _p), ("block_table", _p), ("out", _p), ("softmax_max", _p),
        ("softmax_sum", _p), ("error_flag", _p), ("workspace", _p), ("workspace_bytes", _i64),
        ("num_rows", _i64), ("batch", _i64), ("n1", _i64), ("d", _i64), ("topk", _i64),
        ("sparse_block_size", _i64), ("kv_rows", _i64), ("page_size", _i64),
        ("max_blocks", _i64), ("s2_cap", _i64),
        ("scale", ctypes.c_float), ("sparse_mode", ctypes.c_int32), ("dtype", ctypes.c_int32),
    ]


class SfaBwdParams(ctypes.Structure):
    _fields_ = [
        ("q", _p), ("q_rope", _p), ("key", _p), ("key_rope", _p), ("d_out", _p), ("out", _p),
        ("softmax_max", _p), ("softmax_sum", _p), ("sparse_indices", _p), ("act_q", _p),
        ("act_k", _p), ("q_row_base", _p), ("k_row_base", _p), ("block_table", _p),
        ("dq", _p), ("dqr", _p), ("dk", _p), ("dkr", _p), ("dv", _p),
        ("dk_acc", _p), ("dkr_acc", _p), ("dv_acc", _p), ("error_flag", _p),
        ("workspace", _p), ("workspace_bytes", _i64),
        ("num_rows", _i64), ("batch", _i64), ("n1", _i64), ("d", _i64), ("topk", _i64),
        ("sparse_block_size", _i64), ("kv_rows", _i64), ("page_size", _i64),
        ("max_blocks", _i64), ("s2_cap", _i64),
        ("scale", ctypes.c_float), ("sparse_mode", ctypes.c_int32), ("dtype", ctypes.c_int32),
        ("defer_cast", ctypes.c_int32), ("accumulate", ctypes.c_int32),
        ("teacher", _p),
    ]


class LiParams(ctypes.Structure):
    _fields_ = [
        ("query", _p), ("key", _p), ("weights", _p), ("act_q", _p), ("act_k", _p),
        ("q_row_base", _p), ("k_row_base", _p), ("out_indices", _p), ("out_values", _p),
        ("error_flag", _p), ("workspace", _p), ("workspace_bytes", _i64),
        ("q_rows", _i64), ("batch", _i64), ("n1", _i64), ("n2", _i64), ("d", _i64),
        ("kv_rows", _i64), ("sparse_count", _i64), ("s2_row", _i64), ("s2_cap", _i64),
        ("q_len_max", _i64), ("q_len_dense", _i64),
        ("sparse_mode", ctypes.c_int32), ("dtype", ctypes.c_int32), ("weights_dtype", ctypes.c_int32),
        ("block_table", _p), ("page_size", _i64), ("max_blocks", _i64), ("key_scale", _p),
    ]


class SliParams(ctypes.Structure):
    _fields_ = [
        ("query", _p), ("key", _p), ("query_rope", _p), ("key_rope", _p), ("query_index", _p),
        ("key_index", _p), ("weights", _p), ("sparse_indices", _p), ("softmax_max", _p),
        ("softmax_sum", _p), ("act_q", _p), ("act_k", _p), ("d_query_index", _p),
        ("d_key_index", _p), ("d_weights", _p), ("dki_acc", _p), ("loss", _p),
        ("error_flag", _p), ("workspace", _p), ("workspace_bytes", _i64),
        ("batch", _i64), ("s1", _i64), ("s2", _i64), ("n1", _i64), ("d", _i64),
        ("n_index", _i64), ("d_index", _i64), ("topk", _i64),
        ("scale", ctypes.c_float), ("dtype", ctypes.c_int32), ("weights_dtype", ctypes.c_int32),
        ("teacher", _p),
    ]


class DenseIndexerParams(ctypes.Structure):
    _fields_ = [
        ("query", _p), ("key", _p), ("query_rope", _p), ("key_rope", _p), ("query_index", _p),
        ("key_index", _p), ("weights", _p), ("softmax_max", _p), ("softmax_sum", _p),
        ("index_max", _p), ("index_sum", _p), ("act_q", _p), ("act_k", _p),
        ("d_query_index", _p), ("d_key_index", _p), ("d_weights", _p), ("loss", _p),
        ("workspace", _p), ("workspace_bytes", _i64),
        ("batch", _i64), ("s1", _i64), ("s2", _i64), ("n1", _i64), ("n2", _i64), ("d", _i64),
        ("d_rope", _i64), ("n_index", _i64), ("d_index", _i64),
        ("scale", ctypes.c_float), ("dtype", ctypes.c_int32), ("weights_dtype", ctypes.c_int32),
    ]


class AttnPagedParams(ctypes.Structure):
    _fields_ = [
        ("query", _p), ("query_rope", _p), ("key_cache", _p), ("key_rope_cache", _p),
        ("block_table", _p), ("act_q", _p), ("act_k", _p), ("out", _p), ("softmax_max", _p),
        ("softmax_sum", _p), ("error_flag", _p), ("workspace", _p), ("workspace_bytes", _i64),
        ("batch", _i64), ("s1", _i64), ("n1", _i64), ("d", _i64), ("num_pages", _i64),
        ("page_size", _i64), ("max_blocks", _i64),
        ("q_batch_stride", _i64), ("q_token_stride", _i64), ("q_head_stride", _i64),
        ("qr_batch_stride", _i64), ("qr_token_stride", _i64), ("qr_head_stride", _i64),
        ("k_page_stride", _i64), ("k_row_stride", _i64),
        ("kr_page_stride", _i64), ("kr_row_stride", _i64),
        ("scale", ctypes.c_float), ("sparse_mode", ctypes.c_int32), ("dtype", ctypes.c_int32),
    ]


class AttnSharedParams(ctypes.Structure):
    _fields_ = [("attn", AttnPagedParams), ("group_starts", _p), ("prefix_lengths", _p), ("groups", _i64),
                ("least_saving", _i64)]


class RotaryParams(ctypes.Structure):
    _fields_ = [
        ("x", _p), ("out", _p), ("positions", _p), ("table", _p), ("error_flag", _p),
        ("batch", _i64), ("s", _i64), ("heads", _i64), ("head_dim", _i64), ("offset", _i64),
        ("dim", _i64), ("max_positions", _i64),
        ("x_batch_stride", _i64), ("x_token_stride", _i64), ("x_head_stride", _i64),
        ("out_batch_stride", _i64), ("out_token_stride", _i64), ("out_head_stride", _i64),
        ("half_layout", ctypes.c_int32), ("inverse", ctypes.c_int32), ("dtype", ctypes.c_int32),
    ]


class RotaryAxesParams(ctypes.Structure):
    _fields_ = [("rotary", RotaryParams), ("axes", ctypes.c_int32), ("axis_of", ctypes.c_uint8 * 128)]


ROTARY_MAX_AXES = 4                                     # DSA_ROTARY_MAX_AXES
ROTARY_CODES = {None: 0, "interleaved": 1, "half": 2}   # DSA_ROTARY_*
APPEND_MAX_ENTRIES = 4                                  # DSA_APPEND_MAX_ENTRIES
PAGES_COPY, PAGES_FORK, PAGES_EXTEND, PAGES_FREE, PAGES_COMPACT = range(5)   # DSA_PAGES_*


class CacheRows(ctypes.Structure):
    _fields_ = [
        ("src", _p), ("cache", _p), ("src_batch_stride", _i64), ("src_token_stride", _i64),
        ("page_stride", _i64), ("row_stride", _i64), ("width_bytes", _i64), ("offset", _i64),
        ("rotary", ctypes.c_int32), ("dtype", ctypes.c_int32),
    ]


class CacheAppendParams(ctypes.Structure):
    _fields_ = [
        ("rows", CacheRows * APPEND_MAX_ENTRIES), ("block_table", _p), ("starts", _p),
        ("counts", _p), ("table", _p), ("error_flag", _p), ("batch", _i64), ("s", _i64),
        ("num_pages", _i64), ("page_size", _i64), ("max_blocks", _i64), ("max_positions", _i64),
        ("dim", _i64), ("entries", ctypes.c_int32),
    ]


class PageCache(ctypes.Structure):
    _fields_ = [("data", _p), ("page_stride", _i64), ("row_stride", _i64), ("row_bytes", _i64)]


class PagesParams(ctypes.Structure):
    _fields_ = [
        ("block_table", _p), ("seq_lengths", _p), ("ref_counts", _p), ("block_table_out", _p),
        ("seq_lengths_out", _p), ("ref_counts_out", _p), ("first", _p), ("second", _p),
        ("caches", ctypes.POINTER(PageCache)), ("error_flag", _p), ("workspace", _p),
        ("workspace_bytes", _i64), ("n", _i64), ("slots", _i64), ("max_blocks", _i64),
        ("num_pages", _i64), ("page_size", _i64), ("num_caches", ctypes.c_int32),
        ("op", ctypes.c_int32),
    ]


class BatchPlanParams(ctypes.Structure):
    _fields_ = [
        ("block_table", _p), ("seq_lengths", _p), ("rows", _p), ("counts", _p), ("block_table_out", _p),
        ("key_lengths", _p), ("query_ends", _p), ("token_rows", _p), ("positions", _p),
        ("slot_map", _p), ("group_starts", _p), ("prefix_lengths", _p), ("error_flag", _p),
        ("workspace", _p), ("workspace_bytes", _i64), ("batch", _i64), ("slots", _i64),
        ("max_blocks", _i64), ("page_size", _i64), ("num_tokens", _i64), ("max_groups", _i64),
        ("min_prefix", _i64),
    ]


class CacheStoreParams(ctypes.Structure):
    _fields_ = [
        ("rows", CacheRows * APPEND_MAX_ENTRIES), ("slots", _p), ("error_flag", _p), ("tokens", _i64),
        ("num_pages", _i64), ("page_size", _i64), ("entries", ctypes.c_int32),
    ]


_lock = threading.Lock()
_lib = None
_err_bufs: dict = {}
_error_views: dict = {}
_report_ptrs: dict = {}


def lib() -> ctypes.CDLL:
    """Load (once) and return the CUDA library; raises if it is missing."""
    global _lib
    if _lib is None:
        with _lock:
            if _lib is None:
                if not os.path.exists(LIB_PATH):
                    raise RuntimeError(
                        f"{LIB_PATH} is missing: build it with `python -m dsa_triton_ascend_b200.build`"
                        " (there is no CPU fallback)")
                l = ctypes.CDLL(LIB_PATH)
                l.dsa_version.restype = ctypes.c_int
                l.dsa_sfa_fwd.argtypes = [ctypes.POINTER(SfaFwdParams), _p]
                l.dsa_sfa_fwd.restype = ctypes.c_int
                l.dsa_sfa_fwd_workspace_size.argtypes = [_i64, _i64, _i64]
                l.dsa_sfa_fwd_workspace_size.restype = _i64
                l.dsa_sfa_fwd_fast_workspace_size.argtypes = [_i64] * 5
                l.dsa_sfa_fwd_fast_workspace_size.restype = _i64
                l.dsa_sfa_fwd_noalloc.argtypes = [ctypes.POINTER(SfaFwdParams), _p]
                l.dsa_sfa_fwd_noalloc.restype = ctypes.c_int
                l.dsa_sfa_bwd.argtypes = [ctypes.POINTER(SfaBwdParams), _p]
                l.dsa_sfa_bwd.restype = ctypes.c_int
                l.dsa_sfa_bwd_cast.argtypes = [ctypes.POINTER(SfaBwdParams), _p]
                l.dsa_sfa_bwd_cast.restype = ctypes.c_int
                l.dsa_sfa_bwd_workspace_size.argtypes = [_i64, _i64, _i64]
                l.dsa_sfa_bwd_workspace_size.restype = _i64
                l.dsa_li_score_topk.argtypes = [ctypes.POINTER(LiParams), _p]
                l.dsa_li_score_topk.restype = ctypes.c_int
                l.dsa_li_workspace_size.argtypes = [_i64, _i64, _i64]
                l.dsa_li_workspace_size.restype = _i64
                l.dsa_sli_grad.argtypes = [ctypes.POINTER(SliParams), _p]
                l.dsa_sli_grad.restype = ctypes.c_int
                l.dsa_sli_cast.argtypes = [ctypes.POINTER(SliParams), _p]
                l.dsa_sli_cast.restype = ctypes.c_int
                l.dsa_sli_workspace_size.argtypes = [_i64, _i64, _i64]
                l.dsa_sli_workspace_size.restype = _i64
                for fn in (l.dsa_dense_indexer_softmax_lse, l.dsa_dense_indexer_grad_kl_loss):
                    fn.argtypes = [ctypes.POINTER(DenseIndexerParams), _p]
                    fn.restype = ctypes.c_int
                l.dsa_dense_indexer_workspace_size.argtypes = [_i64] * 4
                l.dsa_dense_indexer_workspace_size.restype = _i64
                l.dsa_attn_paged.argtypes = [ctypes.POINTER(AttnPagedParams), _p]
                l.dsa_attn_paged.restype = ctypes.c_int
                l.dsa_attn_paged_workspace_size.argtypes = [_i64] * 4
                l.dsa_attn_paged_workspace_size.restype = _i64
                l.dsa_attn_paged_shares_keys.argtypes = [_i64] * 2
                l.dsa_attn_paged_shares_keys.restype = ctypes.c_int
                l.dsa_attn_shared.argtypes = [ctypes.POINTER(AttnSharedParams), _p]
                l.dsa_attn_shared.restype = ctypes.c_int
                l.dsa_attn_shared_looks.argtypes = [ctypes.POINTER(AttnSharedParams), ctypes.c_int]
                l.dsa_attn_shared_looks.restype = ctypes.c_int
                l.dsa_attn_shared_workspace_size.argtypes = [_i64] * 5
                l.dsa_attn_shared_workspace_size.restype = _i64
                l.dsa_rotary.argtypes = [ctypes.POINTER(RotaryParams), _p]
                l.dsa_rotary.restype = ctypes.c_int
                l.dsa_rotary_axes.argtypes = [ctypes.POINTER(RotaryAxesParams), _p]
                l.dsa_rotary_axes.restype = ctypes.c_int
                l.dsa_rotary_table.argtypes = [_p, _i64, _i64, ctypes.POINTER(ctypes.c_double),
                                               ctypes.c_double, _p]
                l.dsa_rotary_table.restype = ctypes.c_int
                l.dsa_cache_append.argtypes = [ctypes.POINTER(CacheAppendParams), _p]
                l.dsa_cache_append.restype = ctypes.c_int
                l.dsa_pages.argtypes = [ctypes.POINTER(PagesParams), _p]
                l.dsa_pages.restype = ctypes.c_int
                l.dsa_pages_workspace_size.argtypes = [ctypes.c_int32, _i64, _i64, _i64]
                l.dsa_pages_workspace_size.restype = _i64
                l.dsa_batch_plan.argtypes = [ctypes.POINTER(BatchPlanParams), _p]
                l.dsa_batch_plan.restype = ctypes.c_int
                l.dsa_batch_plan_workspace_size.argtypes = [_i64]
                l.dsa_batch_plan_workspace_size.restype = _i64
                l.dsa_cache_store.argtypes = [ctypes.POINTER(CacheStoreParams), _p]
                l.dsa_cache_store.restype = ctypes.c_int
                _lib = l
    return _lib


_binding = None


def binding():
    """The compiled path of the serving operators' repeated calls (csrc/binding.cpp), or None
    where it is not built, or was built for another torch; the operators' own Python path calls the
    same entries."""
    global _binding
    if _binding is None:
        _binding = False
        try:
            from . import _binding as module
        except ImportError:
            return None
        if getattr(module, "TORCH_VERSION", None) != torch.__version__:
            return None
        entries = tuple(ctypes.cast(getattr(lib(), name), ctypes.c_void_p).value for name in (
            "dsa_attn_paged", "dsa_rotary", "dsa_cache_append", "dsa_pages", "dsa_attn_shared", "dsa_rotary_axes",
            "dsa_batch_plan", "dsa_cache_store"))
        module.connect(entries, check)
        _binding = module
    return _binding or None


def remember(op: int, index: int, *call) -> None:
    """Keep the plan of a call's signature for the compiled path: the operator's arguments, its
    parameters, extra bytes and workspace bytes."""
    module = binding()
    if module is not None:
        module.set_report(index, report_ptr(index))
        module.keep(op, *call)


# Op of csrc/binding.cpp
BIND_ATTN, BIND_ROTARY, BIND_APPEND, BIND_UPKEEP, BIND_SHARED, BIND_AXES, BIND_PLAN, BIND_STORE = range(8)


def check(rc: int, what: str) -> None:
    if rc != DSA_OK:
        raise RuntimeError(f"{what}: {_ERR_TEXT.get(rc, 'error')} (code {rc})")


def _flags(device) -> torch.Tensor:
    """Per-device pair of int32: error_flag and report_flag."""
    key = torch.device(device).index
    if key is None:   # "cuda" is the current device: one pair, whichever way it is named
        key = torch.cuda.current_device()
    buf = _err_bufs.get(key)
    if buf is None:
        buf = torch.zeros(2, dtype=torch.int32, device=torch.device("cuda", key))
        _err_bufs[key] = buf
    return buf


def error_flag(device: torch.device) -> torch.Tensor:
    """Per-device int32 the kernels OR their error bits into.  Kernels of the sparse path give
    up their work while a bit is set.  Kept per device, as making a view costs each call 1.4 us."""
    index = torch.device(device).index
    flag = _error_views.get(index)
    if flag is None:
        flag = _flags(device)[:1]
        if index is not None:   # "cuda" alone is whichever device is current
            _error_views[index] = flag
    return flag


def report_flag(device: torch.device) -> torch.Tensor:
    """Per-device int32 for operators that report a request they cannot meet (a page that is
    not in the pool, no page left) and go on: such a bit stops no other kernel."""
    return _flags(device)[1:]


def report_ptr(index: int) -> int:
    """Address of :func:`report_flag` of device `index`."""
    p = _report_ptrs.get(index)
    if p is None:
        p = _report_ptrs[index] = report_flag(torch.device("cuda", index)).data_ptr()
    return p


def check_device_errors(device=None) -> None:
    """Synchronise and raise if any kernel reported a device-side error."""
    dev = torch.device("cuda" if device is None else device)
    buf = _flags(dev)
    torch.cuda.synchronize(dev)
    error, report = buf.tolist()
    v = error | report
    if v:
        buf.zero_()
        raise RuntimeError(f"dsa kernel reported device error bits 0x{v:x} "
                           "(bit1: bounded wait timed out, bit2: an index or position outside its "
                           "tensor, bit3: misaligned shared memory, bit4: no free page left)")


def ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def stream_ptr(device) -> int:
    return torch.cuda.current_stream(device).cuda_stream
