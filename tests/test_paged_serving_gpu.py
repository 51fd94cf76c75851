"""The serving operators together (GPU): the example's session against plain attention.

Every sequence's keys are kept beside the session, unpaged and in order; after prompts, forks,
steps, frees and compaction a step's output is compared with attention over them in 64 bits.
The tolerance is that of tests/test_attn_paged_gpu.py with one rounding more, of the rotated keys
and queries to bf16 (2^-8 each), which moves a score by at most 2^-7 of its rotary part:
u + 2^-7 |z_rope| + 2^-18 of A, and u of the result.
"""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rotated(x, at, layout="interleaved"):
    """x [n, heads, 64 or more] at positions at [n], in 64 bits."""
    f = torch.tensor([10000.0 ** (-2.0 * i / 64) for i in range(32)], dtype=torch.float64, device="cuda")
    ang = at.double()[:, None, None] * f
    out = x.double().clone()
    i = torch.arange(32, device="cuda")
    ia, ib = (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + 32)
    a, b = x.double()[..., ia], x.double()[..., ib]
    out[..., ia], out[..., ib] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    return out


class Mirror:
    """The sequences in order, as (key, key_rope, key_index) rows before rotation."""

    def __init__(self):
        self.rows = {}

    def add(self, slots, counts, key, key_rope, key_index):
        for n, s in enumerate(slots):
            new = [t[n, :counts[n], 0] for t in (key, key_rope, key_index)]
            old = self.rows.get(s)
            self.rows[s] = new if old is None else [torch.cat(p) for p in zip(old, new)]

    def check(self, session, slots, out, query, query_rope, positions=None, picked=None):
        u = 2.0 ** -8
        for n, s in enumerate(slots):
            key, rope, _ = self.rows[s]
            total = key.shape[0]
            for t in range(query.shape[1]) if positions is None else positions[n]:
                pos = total - 1 if positions is None else t
                see = torch.arange(pos + 1, device="cuda") if picked is None else picked[n]
                k, kr = key.double()[see], _rotated(rope[:, None], torch.arange(total, device="cuda"))[see, 0]
                q, qr = query[n, t].double(), _rotated(query_rope[n, t][None], i32(pos))[0]
                z = (q @ k.t() + qr @ kr.t()) * session.scale
                ez = (2.0 ** -7 * (qr.abs() @ kr.abs().t()) * session.scale).amax(-1, keepdim=True)
                p = torch.softmax(z, -1)
                ref, mag = p @ k, p @ k.abs()
                bound = (u + 2 * ez + 2.0 ** -12) * mag + u * ref.abs()
                assert bool(((out[n, t].double() - ref).abs() <= bound).all())


@pytest.mark.parametrize("heads", [16, 128])
def test_session(heads):
    import dsa_triton_ascend_b200 as dsa
    from paged_serving import PagedSession
    g = torch.Generator(device="cuda")
    g.manual_seed(heads)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()
    session, mirror = PagedSession(slots=8, num_pages=40, page_size=16, heads=heads), Mirror()

    def tokens(n, s):
        return [rnd(n, s, heads, 512), rnd(n, s, heads, 64), rnd(n, s, 1, 512), rnd(n, s, 1, 64), rnd(n, s, 1, 128)]

    def step(slots, **kw):
        t = tokens(len(slots), 1)
        mirror.add(slots, [1] * len(slots), *t[2:])
        out = session.step(i32(*slots), *t, **kw)
        if not kw:
            mirror.check(session, slots, out, t[0], t[1])
        return out, t

    t = tokens(2, 70)
    mirror.add([3, 5], [70, 33], *t[2:])
    out = session.prompt(i32(3, 5), i32(70, 33), *t)
    mirror.check(session, [3, 5], out, t[0], t[1], positions=[[0, 1, 15, 16, 69], [0, 31, 32]])
    assert not out[1, 33:].any()
    session.fork(i32(3, 3, 5), i32(0, 7, 1))
    mirror.rows.update({0: mirror.rows[3], 7: mirror.rows[3], 1: mirror.rows[5]})
    for _ in range(18):
        step([3, 5, 0, 7, 1])
    session.free(i32(3, 1))
    for s in (3, 1):
        mirror.rows.pop(s)
    before = int((session.refs > 0).sum())
    session.compact()
    assert int((session.refs[:before] > 0).sum()) == before and not session.refs[before:].any()
    step([7, 0, 5])
    out, t = step([7, 5], query_index=rnd(2, 1, 64, 128), weights=torch.rand(2, 1, 64, generator=g, device="cuda"),
                  top_k=64)
    assert out.isfinite().all()
    step([0, 5])
    dsa.check_device_errors()
    assert session.lengths.tolist() == [90, 0, 0, 0, 0, 54, 0, 90]


def test_step_in_a_captured_graph():
    """A decode step replays with the state it left: lengths, table and pages grow on the GPU."""
    import dsa_triton_ascend_b200 as dsa
    from paged_serving import PagedSession
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()
    heads = 16
    session, mirror = PagedSession(slots=2, num_pages=12, page_size=16, heads=heads), Mirror()
    tokens = lambda n, s: [rnd(n, s, heads, 512), rnd(n, s, heads, 64), rnd(n, s, 1, 512), rnd(n, s, 1, 64), rnd(n, s, 1, 128)]
    rows = i32(1, 0)
    t = tokens(2, 1)
    state = [session.block_table, session.lengths, session.refs]

    def step():
        session.block_table, session.lengths, session.refs = state
        out = session.step(rows, *t)
        for a, b in zip(state, (session.block_table, session.lengths, session.refs)):
            a.copy_(b)
        return out

    keep = [x.clone() for x in state]
    step()
    torch.cuda.synchronize()
    for a, b in zip(state, keep):
        a.copy_(b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for a, b in zip(state, keep):
        a.copy_(b)
    for _ in range(35):
        for a, b in zip(t, tokens(2, 1)):
            a.copy_(b)
        mirror.add([1, 0], [1, 1], *[x.clone() for x in t[2:]])
        graph.replay()
        mirror.check(session, [1, 0], out, t[0], t[1])
    dsa.check_device_errors()
    assert state[1].tolist() == [35, 35] and int(state[2].sum()) == 6


def test_step_over_the_picked_keys():
    """A step with ``top_k`` after prompts, a fork, a free and a compaction: the indexer's picks are the
    highest of the 64-bit scores, and the output is attention over just those keys.

    An index score is sum_h w_h relu(qi_h . ki) over keys and queries that are rotated and rounded to
    bf16 (2^-8 each), formed in fp32; so it is off by at most 2^-7 + 2^-9 of sum_h |w_h| |qi_h| . |ki|,
    the second part for the products' sum and second-order terms, and two keys may change places only
    where their scores are nearer than twice that."""
    import dsa_triton_ascend_b200 as dsa
    from paged_serving import PagedSession
    heads, top_k = 16, 32
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()
    session, mirror = PagedSession(slots=6, num_pages=40, page_size=16, heads=heads), Mirror()
    tokens = lambda n, s: [rnd(n, s, heads, 512), rnd(n, s, heads, 64), rnd(n, s, 1, 512), rnd(n, s, 1, 64), rnd(n, s, 1, 128)]
    t = tokens(3, 90)
    mirror.add([0, 4, 2], [90, 50, 77], *t[2:])
    session.prompt(i32(0, 4, 2), i32(90, 50, 77), *t)
    session.fork(i32(2), i32(5))
    mirror.rows[5] = mirror.rows[2]
    session.free(i32(0))
    session.compact()
    slots = [5, 4, 2]
    t = tokens(3, 1)
    mirror.add(slots, [1] * 3, *t[2:])
    qi, w = rnd(3, 1, 64, 128), torch.rand(3, 1, 64, generator=g, device="cuda")
    out = session.step(i32(*slots), *t, query_index=qi, weights=w, top_k=top_k)
    at = session.lengths[i32(*slots)][:, None] - 1
    picked, _ = dsa.lightning_indexer_paged(
        dsa.rotary_embedding(qi, session.table, at, layout="half"), session.caches[2], w, session.block_table[i32(*slots)],
        actual_seq_lengths_key=session.lengths[i32(*slots)], sparse_count=top_k)
    dsa.check_device_errors()
    picked = picked.reshape(3, top_k).long()
    for n, s in enumerate(slots):
        total = mirror.rows[s][2].shape[0]
        mine = picked[n].tolist()
        assert len(set(mine)) == top_k and 0 <= min(mine) and max(mine) < total
        k = _rotated(mirror.rows[s][2][:, None], torch.arange(total, device="cuda"), "half")[:, 0]
        q = _rotated(qi[n, 0][None], i32(total - 1), "half")[0]
        score = w[n, 0].double() @ (q @ k.t()).relu()
        slack = (2.0 ** -7 + 2.0 ** -9) * (w[n, 0].double() @ (q.abs() @ k.abs().t()))
        rest = torch.ones(total, dtype=torch.bool, device="cuda")
        rest[picked[n]] = False
        assert bool((score[picked[n]] + slack[picked[n]]).min() >= (score[rest] - slack[rest]).max())
    mirror.check(session, slots, out, t[0], t[1], picked=picked)
