"""The operators for batches that share a prompt, together (GPU): the example's packed steps against
plain attention, and the compiled path of repeated calls against the Python path.

Every sequence's keys are kept beside the session, unpaged, in order and before rotation; the tolerance is
that of test_paged_serving_gpu.py: u + 2^-7 |z_rope| and the fp32 sums' 2^-12 of A, and u of the result,
for keys and queries that are rotated and rounded to bf16 (2^-8 each).
"""
import importlib
import os
import sys

import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from dsa_triton_ascend_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def give_memory_back():
    """Large blocks that stay in torch's cache would serve a later test that counts on its being empty."""
    yield
    torch.cuda.empty_cache()

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _axes(at):
    """Positions on three axes of tokens at `at`, as a film of 6 x 5 places a frame would have them."""
    return torch.stack([at // 30 + 2, at % 30 // 5 + at // 40, at % 5 + 1])


def _rotated(x, at, sections):
    """x [n, 64] at positions at [n], in 64 bits."""
    f = torch.tensor([10000.0 ** (-2.0 * i / 64) for i in range(32)], dtype=torch.float64, device="cuda")
    if sections is None:
        ang = at.double()[:, None] * f
    else:
        axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device="cuda")
        ang = _axes(at)[axis].t().double() * f
    out = x.double().clone()
    a, b = x.double()[..., 0::2], x.double()[..., 1::2]
    out[..., 0::2], out[..., 1::2] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    return out


@pytest.mark.parametrize("heads", [8, 32, 128])
@pytest.mark.parametrize("sections", [None, (8, 12, 12)])
@pytest.mark.parametrize("share", [False, True])
def test_packed_steps_of_forks(heads, sections, share, monkeypatch):
    """A prompt that six forks continue with tokens of their own, beside another one, in several orders."""
    from paged_serving import PagedSession
    if share:   # however little it saves
        module = importlib.import_module("dsa_triton_ascend_b200.flash_attention_paged")
        monkeypatch.setattr(module, "_LEAST_SAVING", 0)
        monkeypatch.setattr(module, "binding", lambda: None)
        monkeypatch.setattr(module, "remember", lambda *a: None)
    g = torch.Generator(device="cuda")
    g.manual_seed(heads)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()
    session, rows = PagedSession(slots=10, num_pages=80, page_size=16, max_blocks=24, heads=heads), {}

    def step(slots, counts, spare=0):
        n, S, T = len(slots), max(counts), sum(counts)
        q, qr = rnd(n, S, heads, 512), rnd(n, S, heads, 64)
        new = [rnd(T + spare, 1, w) for w in (512, 64, 128)]
        out = session.extend_packed(i32(*slots), i32(*counts), q, qr, *new, sections=sections, axes=_axes)
        t = 0
        for i, (s, c) in enumerate(zip(slots, counts)):
            old = rows.get(s)
            mine = [x[t:t + c, 0] for x in new[:2]]
            rows[s] = mine if old is None else [torch.cat(p) for p in zip(old, mine)]
            t += c
            key, rope = rows[s]
            total = key.shape[0]
            kr = _rotated(rope, torch.arange(total, device="cuda"), sections)
            assert not out[i, c:].any()
            for k in sorted({0, c // 2, c - 1} if c else ()):
                at = total - c + k
                seen, seen_r = key[:at + 1].double(), kr[:at + 1]
                qd = q[i, k].double()
                qrd = _rotated(qr[i, k], torch.full((heads,), at, device="cuda"), sections)
                z = (qd @ seen.t() + qrd @ seen_r.t()) * session.scale
                ez = (2.0 ** -7 * (qrd.abs() @ seen_r.abs().t()) * session.scale).amax(-1, keepdim=True)
                p = torch.softmax(z, -1)
                ref, mag = p @ seen, p @ seen.abs()
                bound = (2.0 ** -8 + 2 * ez + 2.0 ** -12) * mag + 2.0 ** -8 * ref.abs()
                assert bool(((out[i, k].double() - ref).abs() <= bound).all()), (s, k)
        dsa.check_device_errors()

    step([3, 5], [150, 40])
    session.fork(i32(3, 3, 3, 3, 3), i32(0, 1, 2, 4, 6))
    for s in (0, 1, 2, 4, 6):
        rows[s] = rows[3]
    step([0, 1, 2, 3, 4, 6, 5], [1] * 7)
    step([5, 6, 4, 3, 2, 1, 0], [2, 1, 5, 0, 17, 1, 3], spare=9)
    step([1, 5, 0], [1, 1, 1])
    session.fork(i32(2), i32(7))         # a fork of a fork shares more
    rows[7] = rows[2]
    step([0, 1, 2, 7, 3], [1, 2, 1, 30, 1])
    assert session.lengths.tolist() == [156, 155, 169, 152, 156, 44, 152, 198, 0, 0]


@pytest.mark.parametrize("old", [0, 60])
def test_a_packed_step_that_the_pool_cannot_serve(old):
    """The refused slot keeps its keys (or none), the others' tokens go where they would without it."""
    from paged_serving import PagedSession

    def run(pages):
        g = torch.Generator(device="cuda")
        g.manual_seed(7)
        rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()
        tokens = lambda n, S, T: (rnd(n, S, 8, 512), rnd(n, S, 8, 64), rnd(T, 1, 512), rnd(T, 1, 64), rnd(T, 1, 128))
        session = PagedSession(slots=4, num_pages=pages, page_size=16, max_blocks=8, heads=8)
        session.extend_packed(i32(0, 1, 2), i32(20, old, 33), *tokens(3, 60, 53 + old))
        dsa.check_device_errors()
        kept = [c[session.block_table[1, :old // 16].long()].clone() for c in session.caches]
        out = session.extend_packed(i32(0, 1, 2), i32(3, 50, 4), *tokens(3, 50, 57))
        return session, kept, out

    full, kept, out = run(7 + old // 16)                # 50 tokens more take three pages or four
    with pytest.raises(RuntimeError, match="bits 0x14"):
        dsa.check_device_errors()
    assert full.lengths.tolist() == [23, old, 37, 0] and not out[1].any()
    assert all(torch.equal(c[full.block_table[1, :old // 16].long()], k) for c, k in zip(full.caches, kept))
    roomy, _, want = run(40)
    dsa.check_device_errors()
    # the same keys, summed in other parts: twice the fp32 sums' 2^-12 of the values, and a rounding each
    most = roomy.caches[0].abs().max().double()
    for b in (0, 2):
        x, y = out[b].double(), want[b].double()
        assert bool(((x - y).abs() <= 2.0 ** -11 * most + 2.0 ** -8 * (x.abs() + y.abs()) * 1.01).all())
        n = full.lengths[b].item()
        for x, y in zip(full.caches, roomy.caches):
            pages = [t[b, :-(-n // 16)].long() for t in (full.block_table, roomy.block_table)]
            assert torch.equal(x[pages[0]].flatten(0, 1)[:n], y[pages[1]].flatten(0, 1)[:n])


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
                if name in ("shared", "axes", "plan", "store"):
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
        plain, fast = [t if isinstance(t, (tuple, list)) else (t,) for t in (plain, fast)]
        assert len(plain) == len(fast) and all(torch.equal(x, y) and x.shape == y.shape and x.dtype == y.dtype
                                               for x, y in zip(plain, fast))
        return plain
    return both


def test_compiled_attention(paths):
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()
    kc, krc = rnd(400, 64, 1, 256), rnd(400, 64, 1, 64)
    table = torch.arange(300, dtype=torch.int32, device="cuda").repeat(40, 1)
    table[:, 299] = torch.arange(40, device="cuda") + 300
    lens, starts, prefixes = i32(*[19137 + i for i in range(40)]), i32(0, 25, 40), i32(19136, 15000)
    for n1, s1 in ((8, 1), (16, 3), (128, 1)):
        q, qr = rnd(40, s1, n1, 256), rnd(40, s1, n1, 64)
        for kw in (dict(), dict(sparse_mode=3), dict(actual_seq_lengths_query=i32(*[i % 2 for i in range(40)]), sparse_mode=3)):
            for stats in (False, True):
                paths(lambda: dsa.flash_attention_shared_prefix(q, qr, kc, krc, table, starts, prefixes, lens, 0.05,
                                                                return_softmax_lse=stats, **kw))
    a = paths(lambda: dsa.flash_attention_shared_prefix(q, qr, kc, krc, table, starts, prefixes, lens, 0.05))
    b = paths(lambda: dsa.flash_attention_shared_prefix(q, qr, kc, krc, table, starts, prefixes, lens, 0.1))
    assert not torch.equal(a[0], b[0])                       # the scale is part of the signature
    paths(lambda: dsa.flash_attention_shared_prefix(q, qr, kc, krc, table, starts, prefixes, lens.tolist(), 0.05), compiled=False)
    wide = rnd(40, 2, 16, 256)[:, :1]                        # heads that are no rows of one matrix: copied
    q, qr = rnd(40, 1, 16, 256), rnd(40, 1, 16, 64)
    wide.copy_(q)
    a = paths(lambda: dsa.flash_attention_shared_prefix(q, qr, kc, krc, table, starts, prefixes, lens, 0.05))
    b = paths(lambda: dsa.flash_attention_shared_prefix(wide, qr, kc, krc, table, starts, prefixes, lens, 0.05))
    assert torch.equal(a[0], b[0])
    dsa.check_device_errors()


def test_compiled_rotary(paths):
    table = dsa.rotary_table(64, 64)
    pos = torch.arange(18, device="cuda", dtype=torch.int32).view(3, 2, 3)
    for _ in range(2):
        x = torch.randn(2, 3, 4, 128, device="cuda").bfloat16()
        seen = []
        for layout in ("interleaved", "half"):
            for order in ("blocks", "cycled"):
                for sections in ((12, 10, 10), [16, 8, 8]):
                    for inverse in (False, True):
                        seen.append(paths(lambda: dsa.rotary_embedding_axes(x, table, pos, sections, layout, order, 32, inverse))[0])
        assert len({t.float().sum().item() for t in seen}) == len(seen)      # each of them another signature
        y, ref = x.clone(), dsa.rotary_embedding_axes(x, table, pos, (12, 10, 10))

        def in_place():
            y.copy_(x)
            assert dsa.rotary_embedding_axes(y, table, pos, (12, 10, 10), out=y) is y
            return y.clone()
        assert torch.equal(paths(in_place)[0], ref)
        z = torch.empty_like(x)
        paths(lambda: dsa.rotary_embedding_axes(x, table, pos, (12, 10, 10), out=z).clone(), compiled=False)
        paths(lambda: dsa.rotary_embedding_axes(x, table, pos.long(), (12, 10, 10)), compiled=False)
    with pytest.raises(ValueError, match="turns"):
        dsa.rotary_embedding_axes(x, table, pos, (10, 12, 10), order="cycled")
    dsa.check_device_errors()


def test_compiled_plan_and_store(paths):
    table, lens = i32(0, 1, 2, -1, -1, -1, 0, 1, 3).view(3, 3), i32(20, 0, 23)
    for tokens in (4, 9, 0, 3):      # the number of places is no part of the signature
        got = paths(lambda: dsa.paged_batch_plan(table, lens, i32(0, 2, 1), i32(1, 2, 0), 8, tokens))
        assert got[5].tolist() == ([19, 29, 30] + [-1] * 6)[:tokens]
        if tokens == 0:
            with pytest.raises(RuntimeError, match="bits 0x4"):
                dsa.check_device_errors()
    for bad in (-1, 1 << 31):
        with pytest.raises(ValueError, match="num_tokens"):
            dsa.paged_batch_plan(table, lens, i32(0, 2, 1), i32(1, 2, 0), 8, bad)
    assert got[6].tolist() == [0, 2, 3, 3] and got[7].tolist() == [16, 0, 0]
    for a in got:                    # parts of one allocation: writing to one leaves the others
        b = [t.clone() for t in got if t is not a]
        a.fill_(-7)
        assert all(torch.equal(x, y) for x, y in zip(b, [t for t in got if t is not a]))
    caches = [torch.zeros(6, 8, 1, w, device="cuda").bfloat16() for w in (64, 128)]
    new = [torch.randn(5, 1, w, device="cuda").bfloat16() for w in (64, 128)]

    def stored(slots):
        for c in caches:
            c.zero_()
        return [c.clone() for c in dsa.paged_cache_store(new, caches, slots)]
    paths(lambda: stored(torch.tensor([3, -1, 47, 0, 9], device="cuda")))
    paths(lambda: stored(i32(3, -1, 47, 0, 9)), compiled=False)
    strided = torch.randn(5, 1, 64, 2, device="cuda").bfloat16()[..., 0]
    new[0] = strided
    paths(lambda: stored(torch.tensor([3, -1, 47, 0, 9], device="cuda")), compiled=False)
    dsa.check_device_errors()
