"""The compiled path of repeated calls gives what the Python path gives (GPU).

A call of a new signature is checked in Python and keeps its parameters; the next call of that
signature takes the compiled path.  Here both paths run on the same inputs, on other inputs of
the same signature, and on what the compiled path has to leave to the Python path.
"""
import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from dsa_triton_ascend_b200 import _lib

pytestmark = pytest.mark.gpu


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.fixture
def paths(monkeypatch):
    """both(call): the results of the Python path and of the compiled one, which has to be taken."""
    assert _lib.binding() is not None
    taken = []

    class Spy:
        def __getattr__(self, name):
            f = getattr(real, name)

            def g(*a):
                r = f(*a)
                if name in ("attn", "rotary", "append", "upkeep"):
                    taken.append(r is not None)
                return r
            return g

    real = _lib.binding()
    spy = Spy()

    def both(call, compiled=True):
        monkeypatch.setattr(_lib, "_binding", False)
        plain = call()
        monkeypatch.setattr(_lib, "_binding", spy)
        call()
        taken.clear()
        fast = call()
        assert taken == [compiled]
        return plain, fast
    return both


def same(a, b):
    a, b = [t if isinstance(t, (tuple, list)) else (t,) for t in (a, b)]
    assert len(a) == len(b) and all(torch.equal(x, y) and x.shape == y.shape and x.dtype == y.dtype
                                    for x, y in zip(a, b))


def test_attention(paths):
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    kc, krc = rnd(9, 16, 1, 256), rnd(9, 16, 1, 64)
    table, lens = i32(0, 1, 2, 3, 4, 5, 6, 7).view(2, 4), i32(50, 64)
    for n1 in (8, 128):
        for _ in range(2):
            q, qr = rnd(2, 3, n1, 256), rnd(2, 3, n1, 64)
            for kw in (dict(), dict(sparse_mode=3), dict(actual_seq_lengths_query=i32(1, 3), sparse_mode=3)):
                for stats in (False, True):
                    call = lambda: dsa.flash_attention_paged(q, qr, kc, krc, table, lens, 0.05,
                                                             return_softmax_lse=stats, **kw)
                    same(*paths(call))
    q, qr = rnd(2, 1, 8, 256), rnd(2, 1, 8, 64)
    a, b = paths(lambda: dsa.flash_attention_paged(q, qr, kc, krc, table, lens, 0.05))
    c, _ = paths(lambda: dsa.flash_attention_paged(q, qr, kc, krc, table, lens, 0.1))
    assert not torch.equal(a[0], c[0])                       # the scale is part of the signature
    same(*paths(lambda: dsa.flash_attention_paged(q, qr, kc, krc, table, [50, 64], 0.05), compiled=False))
    flat = torch.empty(2 * 8 * 256 + 1, device="cuda", dtype=torch.bfloat16)
    off = flat[1:].view(2, 1, 8, 256)
    off.copy_(q)
    x, y = paths(lambda: dsa.flash_attention_paged(off, qr, kc, krc, table, lens, 0.05), compiled=False)
    same(x, a)
    same(y, a)
    dsa.check_device_errors()


def test_rotary(paths):
    table = dsa.rotary_table(64, 64)
    pos = torch.arange(6, device="cuda", dtype=torch.int32).view(2, 3)
    for _ in range(2):
        x = torch.randn(2, 3, 4, 128, device="cuda").bfloat16()
        for layout in ("interleaved", "half"):
            for offset in (0, 32):
                for inverse in (False, True):
                    same(*paths(lambda: dsa.rotary_embedding(x, table, pos, layout, offset, inverse)))
        y = x.clone()
        ref = dsa.rotary_embedding(x, table, pos)

        def in_place():
            y.copy_(x)
            assert dsa.rotary_embedding(y, table, pos, out=y) is y
            return y.clone()
        a, b = paths(in_place)
        same(a, ref)
        same(b, ref)
        z = torch.empty_like(x)
        same(*paths(lambda: dsa.rotary_embedding(x, table, pos, out=z).clone(), compiled=False))
    with pytest.raises(ValueError, match="layout"):
        dsa.rotary_embedding(x, table, pos, "other")
    with pytest.raises(ValueError, match="CUDA"):
        dsa.rotary_embedding(x.cpu(), table.cpu(), pos.cpu())
    dsa.check_device_errors()


def test_append_and_upkeep(paths):
    table, lens, refs = i32(0, 1, 2, -1, -1, -1, 3, -1, -1).view(3, 3), i32(20, 0, 3), i32(1, 1, 1, 1, 0, 0)
    caches = [torch.randn(6, 8, 1, w, device="cuda").bfloat16() for w in (64, 128)]
    keep = [c.clone() for c in caches]
    rot = dsa.rotary_table(32, 64)

    def fresh(call):
        def f():
            for c, k in zip(caches, keep):
                c.copy_(k)
            r = call()
            r = [] if r is None else list(r)
            return [t.clone() for t in r + caches]
        return f

    tokens = [torch.randn(3, 2, 1, w, device="cuda").bfloat16() for w in (64, 128)]
    for kw in (dict(), dict(counts=i32(1, 0, 2)), dict(table=rot, rotary=[("interleaved", 0), ("half", 64)]),
               dict(table=rot, rotary=[None, ("half", 0)])):
        same(*paths(fresh(lambda: dsa.paged_cache_append(tokens, caches, i32(0, 1, 2, 3, 4, 5, 3, 4, 5).view(3, 3),
                                                         i32(5, 7, 9), **kw))))
    same(*paths(fresh(lambda: dsa.paged_cache_extend(table, lens, refs, i32(1, 9, 0), 8))))
    same(*paths(fresh(lambda: dsa.paged_cache_fork(caches, table, lens, refs, i32(0), i32(1)))))
    same(*paths(fresh(lambda: dsa.paged_cache_fork([], table, lens, refs, i32(2), i32(1), page_size=8))))
    same(*paths(fresh(lambda: dsa.paged_cache_free(table, lens, refs, i32(0, 2)))))
    same(*paths(fresh(lambda: dsa.paged_cache_compact(caches, table, i32(0, 1, 0, 1, 0, 1)))))
    same(*paths(fresh(lambda: dsa.paged_cache_copy(caches, i32(0, 1), i32(4, 5)))))
    wide = i32(0, 1, 2, -1, 0, 0, -1, -1, -1, 0, 0, 0, 3, -1, -1, 0, 0, 0).view(3, 6)[:, :3]   # not contiguous
    same(*paths(fresh(lambda: dsa.paged_cache_free(wide, lens, refs, i32(0, 2))), compiled=False))
    dsa.check_device_errors()
    dsa.paged_cache_extend(table, lens, refs, i32(1, 90, 0), 8)     # the compiled path reports as well
    with pytest.raises(RuntimeError, match="bits 0x4"):
        dsa.check_device_errors()


def test_counted_queries_are_read_where_they_are(paths):
    """With counts per sequence no keys are shared, so heads-first queries are not copied, and the
    call is one that the compiled path takes."""
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    kc, krc = rnd(9, 16, 1, 512), rnd(9, 16, 1, 64)
    table, lens = i32(0, 1, 2, 3, 4, 5, 6, 7).view(2, 4), i32(50, 64)
    q, qr = [rnd(2, 8, 3, w).transpose(1, 2) for w in (512, 64)]
    call = lambda a, b: dsa.flash_attention_paged(a, b, kc, krc, table, lens, 0.05, actual_seq_lengths_query=i32(1, 3),
                                                  sparse_mode=3, return_softmax_lse=True)
    plain, fast = paths(lambda: call(q, qr))
    same(plain, fast)
    same(fast, call(q.contiguous(), qr.contiguous()))
    dsa.check_device_errors()


def test_copied_queries(paths):
    """Queries that are copied first (heads-first ones that share their keys, odd strides), one or both."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    kc, krc = rnd(9, 16, 1, 256), rnd(9, 16, 1, 64)
    table, lens = i32(0, 1, 2, 3, 4, 5, 6, 7).view(2, 4), i32(50, 64)
    q, qr = rnd(2, 3, 8, 256), rnd(2, 3, 8, 64)
    call = lambda a, b: dsa.flash_attention_paged(a, b, kc, krc, table, lens, 0.05, sparse_mode=3, return_softmax_lse=True)
    ref = call(q, qr)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    odd = lambda t: torch.cat([t, t[..., :3]], -1)[..., :t.shape[-1]]
    for a, b in ((heads_first(q), heads_first(qr)), (odd(q), qr), (q, odd(qr)), (heads_first(q), odd(qr))):
        plain, fast = paths(lambda: call(a, b))
        same(plain, fast)
        same(ref, fast)
    dsa.check_device_errors()


def test_refused_calls_stay_refused():
    """A call that the checks refuse is refused after a valid call of nearly the same signature too."""
    caches = [torch.randn(6, 8, 1, w, device="cuda").bfloat16() for w in (64, 128)]
    keep = [c.clone() for c in caches]
    tokens = [torch.randn(2, 1, 1, w, device="cuda").bfloat16() for w in (64, 128)]
    table, lens, refs = i32(0, 1, -1, -1).view(2, 2), i32(9, 0), i32(1, 1, 0, 0, 0, 0)
    append = lambda rotary, n=2: dsa.paged_cache_append(tokens[:n], caches[:n], table, i32(3, 0), counts=i32(0, 0), rotary=rotary)
    for n, good, bad in ((2, None, ([None], [], [None] * 3, ())), (2, [None, None], ([None], [None] * 3)),
                         (1, None, ([], [None] * 2)), (1, [None], ([], [None] * 2))):
        for _ in range(3):
            append(good, n)
        for r in bad:
            with pytest.raises(ValueError, match="one entry"):
                append(r, n)
    assert all(torch.equal(a, b) for a, b in zip(caches, keep))
    fork = lambda size: dsa.paged_cache_fork(caches, table, lens, refs, i32(0), i32(1), page_size=size)
    for good in (None, 8):
        for _ in range(3):
            fork(good)
        for size in (-1, 0, 7):
            with pytest.raises(ValueError, match="page_size"):
                fork(size)
    x, rot, pos = torch.randn(1, 2, 4, 64, device="cuda"), dsa.rotary_table(8, 64), i32(0, 1).view(1, 2)
    for _ in range(3):
        dsa.rotary_embedding(x, rot, pos)
    for offset in (-1, 1):
        with pytest.raises(ValueError, match="exceed"):
            dsa.rotary_embedding(x, rot, pos, offset=offset)
    dsa.check_device_errors()


def test_out_of_memory_is_what_torch_raises():
    """The compiled path raises torch's own exceptions, as the Python path does: a caller that makes
    room and tries again asks for this one.  (The allocator's limit is what runs out here, not the
    card.)"""
    x = torch.randn(1, 4096, 64, 64, device="cuda").bfloat16()
    table = dsa.rotary_table(4096, 64)
    pos = torch.arange(4096, device="cuda", dtype=torch.int32)[None]
    ref = [dsa.rotary_embedding(x, table, pos) for _ in range(2)]     # of a known signature from here on
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction(1e-6)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            dsa.rotary_embedding(x, table, pos)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert torch.equal(dsa.rotary_embedding(x, table, pos), ref[0])
