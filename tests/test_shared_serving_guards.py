"""Refusals of the operators for batches that share a prompt, before any GPU work, and the layout of
their parameters (CPU only)."""
import ctypes
import importlib
import os
import shutil
import subprocess

import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from dsa_triton_ascend_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("kw,msg", [
    (dict(sparse_mode=1), "sparse_mode"),
    (dict(query=t(2, 8, 512)), r"\[B, S1, N1, D\]"),
    (dict(query=t(2, 1, 8, 384)), "share a D"),
    (dict(query=t(2, 1, 129, 512), query_rope=t(2, 1, 129, 64)), "N1"),
    (dict(block_table=i(3, 2)), "block_table"),
    (dict(scale_value=float("nan")), "finite"),
    (dict(query=t(2, 1, 8, 512, dtype=torch.float16)), "dtype"),
    (dict(), "CUDA"),
])
def test_flash_attention_shared_prefix(kw, msg):
    args = dict(query=t(2, 1, 8, 512), query_rope=t(2, 1, 8, 64), key_cache=t(4, 16, 1, 512),
                key_rope_cache=t(4, 16, 1, 64), block_table=i(2, 2), group_starts=i(2), prefix_lengths=i(1))
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        dsa.flash_attention_shared_prefix(**args)


@pytest.mark.parametrize("starts,prefixes,msg", [
    (i(2).long(), i(1), "group_starts"), (i(2, 1), i(1), "group_starts"), ([0, 2], i(1), "group_starts"),
    (i(2), i(1).long(), "prefix_lengths"), (i(2), None, "prefix_lengths"), (i(2), i(1), "CUDA"), (None, None, "group_starts"),
])
def test_groups_of_a_shared_prefix(starts, prefixes, msg, monkeypatch):
    module = importlib.import_module("dsa_triton_ascend_b200.flash_attention_paged")   # (the name is the function's, too)
    monkeypatch.setattr(module, "_plan", lambda *a: (bytes(_lib.AttnPagedParams()), True, True, (2, 1, 1, 8), 16))
    with pytest.raises(ValueError, match=msg):
        module._shared_plan(t(2, 1, 8, 512), t(2, 1, 8, 64), t(4, 16, 1, 512), t(4, 16, 1, 64), i(2, 2), starts, prefixes, 1.0, 0)
    monkeypatch.setattr(module.H, "require_cuda", lambda *a: None)
    with pytest.raises(ValueError, match="must have 2 entries"):
        module._shared_plan(t(2, 1, 8, 512), t(2, 1, 8, 64), t(4, 16, 1, 512), t(4, 16, 1, 64), i(2, 2), i(3), i(1), 1.0, 0)


@pytest.mark.parametrize("kw,msg", [
    (dict(layout="neox"), "layout"), (dict(order="rows"), "order"),
    (dict(x=t(2, 64)), r"\[B, S, N, H\]"),
    (dict(sections=[8, 12, 11]), "add up"), (dict(sections=[16, 16, 0]), "positive"), (dict(sections=[40, -8]), "positive"),
    (dict(sections=[]), "positive"), (dict(sections=[8, 8, 8, 4, 4]), "positive"), (dict(sections=32), "sequence"),
    (dict(sections=[10, 12, 10], order="cycled"), "turns"), (dict(sections=[1, 31], order="cycled"), "turns"),
    (dict(positions=i(2, 3)), "positions"), (dict(positions=i(2, 2, 3)), "positions"),
    (dict(positions=t(3, 2, 3, dtype=torch.float32)), "int32 or int64"),
    (dict(offset=1), "exceed"), (dict(offset=-1), "exceed"),
    (dict(x=t(2, 3, 4, 64, dtype=torch.float64)), "dtype"), (dict(table=t(8, 64)), "table"),
    (dict(table=t(8, dtype=torch.float32)), "table"), (dict(), "CUDA"),
])
def test_rotary_embedding_axes(kw, msg):
    args = dict(x=t(2, 3, 4, 64), table=t(8, 64, dtype=torch.float32), positions=i(3, 2, 3), sections=[8, 12, 12])
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        dsa.rotary_embedding_axes(**args)


def test_rotary_axes():
    assert dsa.rotary_axes([2, 1, 3]) == [0, 0, 1, 2, 2, 2]
    assert dsa.rotary_axes((3, 2, 1), "cycled") == [0, 1, 2, 0, 1, 0]
    assert dsa.rotary_axes([2, 2, 2], "cycled") == [0, 1, 2] * 2
    assert dsa.rotary_axes([5], "cycled") == dsa.rotary_axes([5]) == [0] * 5
    for sections in ([24, 20, 20], [11, 11, 10], [16, 16], [29, 1, 2]):
        axes = dsa.rotary_axes(sections, "cycled")
        assert [axes.count(a) for a in range(len(sections))] == sections


@pytest.mark.parametrize("kw,msg", [
    (dict(tokens=[]), "equal length"), (dict(tokens=[t(5, 1, 64)] * 5, caches=[t(4, 16, 1, 64)] * 5), "equal length"),
    (dict(caches=[t(4, 16, 1, 64)] * 2), "equal length"),
    (dict(slot_map=i(5, 1)), "slot_map"), (dict(slot_map=t(5)), "slot_map"), (dict(slot_map=[1, 2]), "slot_map"),
    (dict(), "CUDA"),
])
def test_paged_cache_store(kw, msg):
    args = dict(tokens=[t(5, 1, 64)], caches=[t(4, 16, 1, 64)], slot_map=i(5))
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        dsa.paged_cache_store(**args)


@pytest.mark.parametrize("kw,msg", [
    (dict(tokens=[t(4, 1, 64)]), "tokens 0 must be"), (dict(tokens=[t(5, 64)]), "tokens 0 must be"),
    (dict(tokens=[t(5, 1, 32)]), "tokens 0 must be"), (dict(tokens=[t(5, 1, 64).half()]), "dtype"),
    (dict(caches=[t(4, 16, 2, 64)]), "tokens 0 must be"), (dict(caches=[t(4, 64)]), "num_pages"),
    (dict(caches=[t(0, 16, 1, 64)]), "empty"),
    (dict(tokens=[t(5, 1, 64)] * 2, caches=[t(4, 16, 1, 64), t(4, 8, 1, 64)]), "pages of"),
    (dict(tokens=[t(5, 1, 4)], caches=[t(4, 16, 1, 4)]), "16-byte"),
    (dict(caches=[t(4, 16, 1, 68)[..., :64]]), "16-byte"),
    (dict(caches=[t(1, 16, 1, 64).expand(4, 16, 1, 64)]), "expanded"),
])
def test_paged_cache_store_shapes(kw, msg, monkeypatch):
    from dsa_triton_ascend_b200 import paged_cache as module
    monkeypatch.setattr(module.H, "require_cuda", lambda *a: None)
    args = dict(tokens=[t(5, 1, 64)], caches=[t(4, 16, 1, 64)], slot_map=i(5))
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        dsa.paged_cache_store(**args)


@pytest.mark.parametrize("kw,msg", [
    (dict(block_table=t(4, 3)), "block_table"), (dict(block_table=i(4)), "block_table"),
    (dict(block_table=i(0, 3), seq_lengths=i(0)), "empty"), (dict(seq_lengths=i(3)), "seq_lengths"),
    (dict(rows=i(2, 1)), "rows"), (dict(rows=[0, 1]), "rows"), (dict(rows=i(2).long()), "rows"), (dict(counts=i(3)), "counts"),
    (dict(page_size=0), "page_size"), (dict(num_tokens=-1), "num_tokens"), (dict(num_tokens=1 << 31), "num_tokens"),
    (dict(max_groups=-1), "max_groups"), (dict(min_prefix=-1), "min_prefix"), (dict(page_size=1 << 30), "32 bits"),
])
def test_paged_batch_plan(kw, msg, monkeypatch):
    from dsa_triton_ascend_b200 import paged_cache as module
    args = dict(block_table=i(4, 3), seq_lengths=i(4), rows=i(2), counts=i(2), page_size=16, num_tokens=5)
    with pytest.raises(ValueError, match="CUDA"):
        dsa.paged_batch_plan(**args)
    monkeypatch.setattr(module.H, "require_cuda", lambda *a: None)
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        dsa.paged_batch_plan(**args)


# ------------------------------------------------------------------------------------------
# the C entries
# ------------------------------------------------------------------------------------------

@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_ctypes_structs_match_the_header(tmp_path):
    structs = {"DsaAttnSharedParams": _lib.AttnSharedParams, "DsaRotaryAxesParams": _lib.RotaryAxesParams,
               "DsaBatchPlanParams": _lib.BatchPlanParams, "DsaCacheStoreParams": _lib.CacheStoreParams}
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "dsa_b200.h"', 'int main(void) {']
    for cname, py in structs.items():
        lines.append(f'  printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {tuple(l.split()[:2]): int(l.split()[2]) for l in out.splitlines()}
    for cname, py in structs.items():
        assert got[(cname, "size")] == ctypes.sizeof(py), cname
        assert all(got[(cname, f)] == getattr(py, f).offset for f, _ in py._fields_), cname


def test_c_entries_refuse_what_the_kernels_cannot_take():
    """Each refusal is on the host: nothing here has a GPU, and no address is looked at."""
    lib, bad = _lib.lib(), _lib.DSA_ERR_INVALID_ARG

    def shared(**kw):
        p = _lib.AttnSharedParams()
        a = p.attn
        for f in ("query", "query_rope", "key_cache", "key_rope_cache", "block_table", "act_k", "out", "workspace"):
            setattr(a, f, 1024)
        p.group_starts = p.prefix_lengths = 1024
        a.batch, a.s1, a.n1, a.d, a.num_pages, a.page_size, a.max_blocks, p.groups = 4, 1, 16, 512, 9, 16, 4, 1
        a.q_batch_stride, a.q_token_stride, a.q_head_stride = 16 * 512, 16 * 512, 512
        a.qr_batch_stride, a.qr_token_stride, a.qr_head_stride = 16 * 64, 16 * 64, 64
        a.k_page_stride, a.k_row_stride, a.kr_page_stride, a.kr_row_stride = 16 * 512, 512, 16 * 64, 64
        a.scale, a.workspace_bytes = 1.0, 1 << 40
        for k, v in kw.items():
            setattr(p if k in ("groups", "group_starts", "prefix_lengths") else a, k, v)
        return lib.dsa_attn_shared(p, None)

    for kw in (dict(groups=-1), dict(groups=1 << 31), dict(groups=(1 << 30) + 1), dict(group_starts=0), dict(prefix_lengths=0), dict(batch=-1), dict(s1=-1),
               dict(page_size=12), dict(n1=0), dict(n1=129), dict(scale=float("inf")), dict(out=1025), dict(workspace=0),
               dict(act_k=0), dict(q_head_stride=4), dict(num_pages=0)):
        assert shared(**kw) == bad, kw
    assert lib.dsa_attn_shared(None, None) == bad and shared(batch=0) == shared(s1=0) == 0

    def axes(**kw):
        p = _lib.RotaryAxesParams()
        r = p.rotary
        r.x = r.out = r.positions = r.table = 1024
        r.batch = r.s = r.heads = 1
        r.head_dim = r.dim = 64
        r.max_positions, p.axes = 8, 3
        for k, v in kw.items():
            if k == "axis":
                p.axis_of[v[0]] = v[1]
            else:
                setattr(p if k == "axes" else r, k, v)
        return lib.dsa_rotary_axes(p, None)

    for kw in (dict(axes=0), dict(axes=5), dict(axis=(31, 3)), dict(axis=(0, 255)), dict(x=0), dict(table=0), dict(dim=63),
               dict(dim=258, head_dim=258), dict(offset=1), dict(offset=-1), dict(max_positions=0), dict(dtype=9), dict(s=-1)):
        assert axes(**kw) == bad, kw
    assert lib.dsa_rotary_axes(None, None) == bad and axes(heads=0) == 0

    def plan(**kw):
        p = _lib.BatchPlanParams()
        for f, kind in p._fields_:
            if kind is ctypes.c_void_p:
                setattr(p, f, 1024)
        p.batch, p.slots, p.max_blocks, p.page_size, p.num_tokens, p.max_groups = 2, 4, 3, 16, 5, 2
        p.workspace_bytes = 1 << 20
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.dsa_batch_plan(p, None)

    for kw in (dict(batch=-1), dict(slots=0), dict(max_blocks=0), dict(page_size=0), dict(page_size=1 << 30), dict(num_tokens=-1),
               dict(max_groups=-1), dict(min_prefix=-1), dict(block_table=0), dict(rows=0), dict(counts=0), dict(slot_map=0),
               dict(group_starts=0), dict(prefix_lengths=0), dict(workspace=0), dict(workspace_bytes=7), dict(key_lengths=0)):
        assert plan(**kw) == bad, kw
    assert lib.dsa_batch_plan(None, None) == bad and lib.dsa_batch_plan_workspace_size(-1) == -1

    def store(row=None, **kw):
        p = _lib.CacheStoreParams()
        e = p.rows[0]
        e.src = e.cache = 1024
        e.src_token_stride = e.row_stride = e.width_bytes = 64
        e.page_stride = 1024
        p.slots, p.tokens, p.num_pages, p.page_size, p.entries = 1024, 3, 4, 16, 1
        for k, v in (row or {}).items():
            setattr(e, k, v)
        for k, v in kw.items():
            setattr(p, k, v)
        return lib.dsa_cache_store(p, None)

    for kw in (dict(entries=0), dict(entries=5), dict(slots=0), dict(tokens=-1), dict(num_pages=0), dict(page_size=0)):
        assert store(**kw) == bad, kw
    for row in (dict(src=0), dict(cache=0), dict(src=1032), dict(width_bytes=8), dict(width_bytes=72), dict(row_stride=8),
                dict(page_stride=8), dict(src_token_stride=8), dict(rotary=1)):
        assert store(row) == bad, row
    assert lib.dsa_cache_store(None, None) == bad and store(tokens=0) == 0
