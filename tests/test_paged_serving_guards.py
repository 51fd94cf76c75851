"""Refusals of the paged serving operators, before any GPU work (CPU only)."""
import ctypes
import os

import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from dsa_triton_ascend_b200 import _host as H
from dsa_triton_ascend_b200 import _lib


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def attn(**kw):
    args = dict(query=t(2, 1, 8, 512), query_rope=t(2, 1, 8, 64), key_cache=t(4, 16, 1, 512),
                key_rope_cache=t(4, 16, 1, 64), block_table=i(2, 2))
    args.update(kw)
    return dsa.flash_attention_paged(**args)


@pytest.mark.parametrize("kw,msg", [
    (dict(sparse_mode=1), "sparse_mode"),
    (dict(query=t(2, 8, 512)), r"\[B, S1, N1, D\]"),
    (dict(query=t(2, 1, 8, 384)), "share a D"),
    (dict(key_cache=t(4, 16, 1, 256)), "share a D"),
    (dict(query=t(2, 1, 129, 512), query_rope=t(2, 1, 129, 64)), "N1"),
    (dict(query_rope=t(2, 1, 8, 32)), "query_rope"),
    (dict(query_rope=t(2, 1, 4, 64)), "query_rope"),
    (dict(key_cache=t(4, 16, 2, 512)), "MQA"),
    (dict(key_rope_cache=t(4, 8, 1, 64)), "MQA"),
    (dict(key_cache=t(4, 12, 1, 512), key_rope_cache=t(4, 12, 1, 64)), "multiple of 8"),
    (dict(key_cache=t(0, 16, 1, 512), key_rope_cache=t(0, 16, 1, 64)), "not empty"),
    (dict(block_table=i(3, 2)), "block_table"),
    (dict(block_table=i(2, 0)), "block_table"),
    (dict(block_table=i(2, 2).long()), "block_table"),
    (dict(query=t(2, 1, 8, 512, dtype=torch.float16)), "dtype"),
    (dict(query=t(2, 1, 8, 512, dtype=torch.float32)), "dtype"),
    (dict(), "CUDA"),
])
def test_flash_attention_paged(kw, msg):
    with pytest.raises(ValueError, match=msg):
        attn(**kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(layout="neox"), "layout"),
    (dict(x=t(2, 64)), r"\[B, S, N, H\]"),
    (dict(x=t(2, 3, 4, 64, dtype=torch.float64)), "dtype"),
    (dict(table=t(8, 64)), "table"),
    (dict(table=t(8, 63, dtype=torch.float32)), "even"),
    (dict(table=t(8, 512, dtype=torch.float32), x=t(2, 3, 4, 512)), "256"),
    (dict(offset=1), "exceed"),
    (dict(offset=-1), "exceed"),
    (dict(positions=i(2, 4)), "positions"),
    (dict(positions=t(2, 3, dtype=torch.float32)), "int32 or int64"),
    (dict(), "CUDA"),
])
def test_rotary_embedding(kw, msg):
    args = dict(x=t(2, 3, 4, 64), table=t(8, 64, dtype=torch.float32), positions=i(2, 3))
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        dsa.rotary_embedding(**args)


@pytest.mark.parametrize("args,kw,msg", [
    ((0, 64), {}, "max_positions"), ((8, 63), {}, "even"), ((8, 258), {}, "even"),
    ((8, 64), dict(base=1.0), "base"), ((8, 64), dict(scaling="x"), "scaling"),
    ((8, 64), dict(scaling="linear", factor=0.0), "factor"), ((8, 2), dict(scaling="ntk", factor=2.0), "ntk"),
    ((8, 64), dict(scaling="yarn", beta_fast=0.5), "yarn"), ((8, 64), dict(device="cpu"), "CUDA"),
])
def test_rotary_table(args, kw, msg):
    with pytest.raises(ValueError, match=msg):
        dsa.rotary_table(*args, **kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(tokens=[]), "lists"),
    (dict(tokens=[t(2, 3, 1, 64)] * 5, caches=[t(4, 8, 1, 64)] * 5), "lists"),
    (dict(rotary=[None, None]), "one entry"),
    (dict(), "CUDA"),
])
def test_paged_cache_append(kw, msg):
    args = dict(tokens=[t(2, 3, 1, 64)], caches=[t(4, 8, 1, 64)], block_table=i(2, 2), starts=i(2))
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        dsa.paged_cache_append(**args)


def test_paged_cache_bookkeeping():
    for call in (lambda: dsa.paged_cache_copy([], i(1), i(1)),
                 lambda: dsa.paged_cache_copy([t(4, 8, 1, 64)], i(1), i(1)),
                 lambda: dsa.paged_cache_extend(i(2, 2), i(2), i(4), i(2), 8),
                 lambda: dsa.paged_cache_fork([], i(2, 2), i(2), i(4), i(1), i(1), page_size=8),
                 lambda: dsa.paged_cache_free(i(2, 2), i(2), i(4), i(1)),
                 lambda: dsa.paged_cache_compact([], i(2, 2), i(4))):
        with pytest.raises(ValueError, match="CUDA|at least one"):
            call()


def test_overlap_of_views():
    a = torch.zeros(4, 8)
    assert not H.overlap(a, a) and not H.overlap(a[:2], a[2:]) and H.overlap(a[:3], a[2:])
    assert not H.overlap(a, torch.zeros(4, 8)) and not H.overlap(a[:0], a)
    assert not H.self_overlap(a) and not H.self_overlap(a.t()) and not H.self_overlap(a[:, ::2])
    assert H.self_overlap(a[:1].expand(4, 8)) and not H.self_overlap(a[:1])
    assert H.self_overlap(torch.as_strided(a, (3, 3), (2, 1)))


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    return ctypes.CDLL(_lib.LIB_PATH)


def _call(lib, name, params):
    f = getattr(lib, name)
    f.restype = ctypes.c_int
    f.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    return f(ctypes.addressof(params) if params is not None else None, None)


def test_c_entries_refuse_bad_arguments(lib):
    """The entry points look at the arguments on the host; the fake pointers are never touched."""
    fake = 1 << 20
    for name in ("dsa_attn_paged", "dsa_rotary", "dsa_cache_append", "dsa_pages"):
        assert _call(lib, name, None) == 1

    def attn_params(**kw):
        p = _lib.AttnPagedParams()
        for f in ("query", "query_rope", "key_cache", "key_rope_cache", "block_table", "act_k", "out", "workspace"):
            setattr(p, f, fake)
        p.batch, p.s1, p.n1, p.d, p.num_pages, p.page_size, p.max_blocks = 2, 1, 16, 512, 4, 16, 2
        p.workspace_bytes = 1 << 40
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for kw in (dict(n1=129), dict(n1=0), dict(page_size=12), dict(num_pages=0), dict(max_blocks=0), dict(sparse_mode=2),
               dict(out=0), dict(key_cache=fake + 8), dict(q_head_stride=4), dict(k_page_stride=-8), dict(batch=-1),
               dict(batch=1 << 31), dict(max_blocks=1 << 30), dict(softmax_max=fake), dict(d=384, dtype=0)):
        assert _call(lib, "dsa_attn_paged", attn_params(**kw)) == 1, kw
    assert _call(lib, "dsa_attn_paged", attn_params(batch=0)) == 0

    def rotary_params(**kw):
        p = _lib.RotaryParams()
        for f in ("x", "out", "positions", "table"):
            setattr(p, f, fake)
        p.batch, p.s, p.heads, p.head_dim, p.dim, p.max_positions = 1, 2, 4, 64, 64, 8
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for kw in (dict(x=0), dict(dim=63), dict(dim=258, head_dim=300), dict(offset=1), dict(offset=-1), dict(max_positions=0),
               dict(batch=-1), dict(dtype=3)):
        assert _call(lib, "dsa_rotary", rotary_params(**kw)) == 1, kw
    assert _call(lib, "dsa_rotary", rotary_params(s=0)) == 0

    def append_params(entry=None, **kw):
        p = _lib.CacheAppendParams()
        p.block_table = p.starts = p.table = fake
        p.batch, p.s, p.num_pages, p.page_size, p.max_blocks, p.entries, p.dim, p.max_positions = 1, 2, 4, 8, 2, 1, 64, 8
        e = p.rows[0]
        e.src = e.cache = fake
        e.width_bytes, e.row_stride, e.page_stride = 128, 128, 1024
        for k, v in (entry or {}).items():
            setattr(e, k, v)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for entry, kw in ((None, dict(entries=0)), (None, dict(entries=5)), (None, dict(starts=0)), (dict(src=0), {}),
                      (dict(cache=fake + 4), {}), (dict(width_bytes=24), {}), (dict(row_stride=24), {}),
                      (dict(rotary=3), {}), (dict(rotary=1), dict(table=0)), (dict(rotary=1, offset=4), {}),
                      (dict(rotary=1, offset=8), {}), (dict(rotary=2), dict(dim=8)), (dict(rotary=1, dtype=3), {}),
                      (None, dict(max_blocks=1 << 30)), (None, dict(batch=-1))):
        assert _call(lib, "dsa_cache_append", append_params(entry, **kw)) == 1, (entry, kw)
    assert _call(lib, "dsa_cache_append", append_params(batch=0)) == 0

    def pages_params(**kw):
        p = _lib.PagesParams()
        for f in ("block_table", "seq_lengths", "ref_counts", "block_table_out", "seq_lengths_out", "ref_counts_out",
                  "first", "second", "workspace"):
            setattr(p, f, fake)
        p.op, p.n, p.slots, p.max_blocks, p.num_pages, p.page_size = _lib.PAGES_FORK, 1, 2, 2, 4, 8
        p.workspace_bytes = 1 << 40
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for kw in (dict(op=5), dict(op=-1), dict(n=-1), dict(slots=0), dict(num_pages=0), dict(page_size=0), dict(second=0),
               dict(workspace_bytes=16), dict(workspace=0), dict(seq_lengths_out=0), dict(num_caches=1),
               dict(op=_lib.PAGES_EXTEND), dict(max_blocks=1 << 30), dict(slots=1 << 20, max_blocks=1 << 20)):
        assert _call(lib, "dsa_pages", pages_params(**kw)) == 1, kw
    assert _call(lib, "dsa_pages", pages_params(op=_lib.PAGES_COPY, n=0)) == 0


def test_parameter_structs_match_the_header(tmp_path):
    import shutil
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    import test_abi_layout as layout
    keep = dict(layout.STRUCTS)
    layout.STRUCTS.clear()
    layout.STRUCTS.update({"DsaAttnPagedParams": _lib.AttnPagedParams, "DsaRotaryParams": _lib.RotaryParams,
                           "DsaCacheRows": _lib.CacheRows, "DsaCacheAppendParams": _lib.CacheAppendParams,
                           "DsaPageCache": _lib.PageCache, "DsaPagesParams": _lib.PagesParams})
    try:
        layout.test_ctypes_structs_match_the_header(tmp_path)
    finally:
        layout.STRUCTS.clear()
        layout.STRUCTS.update(keep)


def test_rotary_frequencies_in_python():
    f = dsa.rotary_frequencies(64)
    assert f[0] == 1.0 and f[31] == pytest.approx(10000.0 ** (-62 / 64))
    assert dsa.rotary_frequencies(64, scaling="linear", factor=4.0)[5] == pytest.approx(f[5] / 4)
    ntk = dsa.rotary_frequencies(64, scaling="ntk", factor=4.0)
    assert ntk[0] == 1.0 and ntk[31] == pytest.approx(f[31] / 4)   # the slowest pair by the whole factor


def test_error_flag_is_kept(monkeypatch):
    """Every call of every operator asks for its flag: one tensor per device, made once, not a new view
    a call; the report flag stands beside it in the pair that check_device_errors reads."""
    pair = torch.zeros(2, dtype=torch.int32)
    monkeypatch.setattr(_lib, "_err_bufs", {3: pair})
    monkeypatch.setattr(_lib, "_error_views", {}, raising=False)
    dev = torch.device("cuda", 3)
    flag = _lib.error_flag(dev)
    assert _lib.error_flag(dev) is flag and _lib.error_flag("cuda:3") is flag
    flag.fill_(7)
    _lib.report_flag(dev).fill_(9)
    assert pair.tolist() == [7, 9] and flag.shape == (1,)


def test_c_entries_refuse_sizes_that_would_wrap(lib):
    """Offsets and sizes near the end of 64 bits are refused, not added up past it."""
    fake, huge = 1 << 20, (1 << 63) - 8
    p = _lib.RotaryParams()
    p.x = p.out = p.positions = p.table = fake
    p.batch, p.s, p.heads, p.head_dim, p.dim, p.max_positions = 1, 2, 4, 64, 64, 8
    for offset in (huge, huge - 64, 1 << 40):
        p.offset = offset
        assert _call(lib, "dsa_rotary", p) == 1
    p = _lib.CacheAppendParams()
    p.block_table = p.starts = p.table = fake
    p.batch, p.s, p.num_pages, p.page_size, p.max_blocks, p.entries, p.dim, p.max_positions = 1, 2, 4, 8, 2, 1, 64, 8
    e = p.rows[0]
    e.src = e.cache = fake
    e.width_bytes, e.row_stride, e.page_stride, e.rotary = 128, 128, 1024, 1
    for offset in (huge, huge - 64, (1 << 62) - 64, 1 << 62, 1 << 40):
        e.offset = offset
        assert _call(lib, "dsa_cache_append", p) == 1
    size = lib.dsa_attn_paged_workspace_size
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_int64] * 4
    for args in ((1 << 40, 1 << 40, 16, 512), (1 << 31, 1, 16, 512), (1, 1 << 31, 16, 512), (1 << 30, 1 << 10, 16, 512), (1, 1, 16, 1 << 60)):
        assert size(*args) == -1
    size = lib.dsa_pages_workspace_size
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_int32] + [ctypes.c_int64] * 3
    for args in ((1, huge, 4, 4), (1, 4, huge, 4), (1, 4, 4, huge), (1, 1 << 31, 4, 4)):
        assert size(*args) == -1


def test_binding_of_another_torch(tmp_path, monkeypatch):
    """A compiled path that was built for another torch is not used, and is built again."""
    import types
    from dsa_triton_ascend_b200 import build
    calls = []
    other = types.SimpleNamespace(TORCH_VERSION="0.0.1", connect=lambda *a: calls.append(a))
    monkeypatch.setattr(dsa, "_binding", other, raising=False)
    monkeypatch.setitem(__import__("sys").modules, "dsa_triton_ascend_b200._binding", other)
    monkeypatch.setattr(_lib, "_binding", None)
    assert _lib.binding() is None and not calls

    made = []

    def compile_it(cmd, check):
        made.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "wb") as f:
            f.write(b"new")
    monkeypatch.setattr(build.subprocess, "run", compile_it)
    path = tmp_path / "_binding.so"
    monkeypatch.setattr(build, "BINDING", str(path))
    path.write_bytes(b"\0dsa binding for torch 0.0.1\0")      # newer than its source
    build.build_binding()
    assert len(made) == 1 and path.read_bytes() == b"new"
    path.write_bytes(b"\0dsa binding for torch " + torch.__version__.encode() + b"\0")
    build.build_binding()
    assert len(made) == 1


def test_binding_is_of_this_torch():
    from dsa_triton_ascend_b200 import build
    if not os.path.exists(build.BINDING):
        pytest.skip("binding not built")
    from dsa_triton_ascend_b200 import _binding
    assert _binding.TORCH_VERSION == torch.__version__


def test_c_append_of_nothing(lib):
    """Empty tensors have no address: a call without batches or tokens is no error, as in the others."""
    p = _lib.CacheAppendParams()
    p.num_pages, p.page_size, p.max_blocks, p.entries = 4, 8, 2, 1
    for p.batch, p.s in ((0, 1), (3, 0), (0, 0)):
        assert _call(lib, "dsa_cache_append", p) == 0
    p.batch = p.s = 1
    assert _call(lib, "dsa_cache_append", p) == 1


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e39])
def test_scale_that_no_fp32_holds(lib, scale):
    """The kernels keep the scale above 0 by a maximum, which a NaN would pass unseen."""
    with pytest.raises(ValueError, match="scale_value"):
        attn(scale_value=scale)
    p = _lib.AttnPagedParams()
    for f in ("query", "query_rope", "key_cache", "key_rope_cache", "block_table", "act_k", "out", "workspace"):
        setattr(p, f, 1 << 20)
    p.batch, p.s1, p.n1, p.d, p.num_pages, p.page_size, p.max_blocks, p.scale = 2, 1, 16, 512, 4, 16, 2, scale
    p.workspace_bytes = 1 << 40
    assert _call(lib, "dsa_attn_paged", p) == 1
