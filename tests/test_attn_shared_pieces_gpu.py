"""flash_attention_shared_prefix where every prefix of a page or more is shared, whatever that costs (GPU).

Whether a call's prefixes went through pieces is seen from the pages: of a shared prefix those of the
group's first row with keys are read, so all other rows of the group name a page of NaN there, and a row
that read its own would give NaN.  The reference and its tolerances are those of test_attn_paged_gpu.py;
the join of a prefix's parts with a row's own is one more fp32 sum of the few that the 2^-18 there allows.
"""
import importlib
import random

import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from dsa_triton_ascend_b200 import _lib
from test_attn_paged_gpu import i32
from test_attn_shared_gpu import Shared

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def give_memory_back():
    """Large blocks that stay in torch's cache would serve a later test that counts on its being empty."""
    yield
    torch.cuda.empty_cache()


@pytest.fixture(autouse=True)
def share_whatever_it_costs(monkeypatch):
    module = importlib.import_module("dsa_triton_ascend_b200.flash_attention_paged")
    monkeypatch.setattr(module, "_LEAST_SAVING", -1)
    if _lib.binding() is not None:   # which keeps what a signature's first call decided
        monkeypatch.setattr(module, "binding", lambda: None)
        monkeypatch.setattr(module, "remember", lambda *a: None)


class Pieces(Shared):
    """As Shared; `run` hands the table over with a page of NaN in place of what no row may read."""

    def first_seen(self, b, mode, act_q):
        """Keys that the first token of row b with any sees."""
        n, s1 = self.lens[b], self.q.shape[1]
        aq = s1 if act_q is None else int(act_q[b])
        for s in range(min(s1, aq)):
            seen = n if mode == 0 else min(n, n - aq + s + 1)
            if n > 0 and seen > 0:
                return seen
        return 0

    def shared(self, mode=0, act_q=None):
        """(the group's rows, those with keys, shared pages) of each group."""
        starts = self.starts.tolist()
        for g, prefix in enumerate(self.prefixes.tolist()):
            rows = range(starts[g], starts[g + 1])
            seen = {b: self.first_seen(b, mode, act_q) for b in rows}
            some = [b for b in rows if seen[b]]
            yield rows, some, max(0, min([prefix] + [seen[b] for b in some])) // self.page if some else 0

    def run(self, mode=0, act_q=None, check=True, lens=None, least=1, **kw):
        groups, kept = list(self.shared(mode, act_q)), self.table
        assert sum(pages > 0 for _, _, pages in groups) >= least      # something is shared at all
        used = {int(p) for p in kept.flatten()}
        poison = next(p for p in range(self.kc.shape[0]) if p not in used and self.kc[p].isnan().all())
        self.table = kept.clone()
        for rows, some, pages in groups:
            for b in rows:
                if some and b != some[0]:
                    self.table[b, :pages] = poison
        try:
            got = super().run(mode, act_q, False, lens, **kw)
        finally:
            self.table = kept
        if check:
            dsa.check_device_errors()
            self.check(got, mode, act_q)
        return got


@pytest.mark.parametrize("heads", [1, 5, 16, 17, 32, 40, 64])
@pytest.mark.parametrize("d", [128, 256, 512])
def test_heads_and_widths(heads, d):
    Pieces([(130, [0, 1, 63]), (64, [5] * 9), (1000, [200, 3])], [0, 70], heads, d, seed=heads).run(least=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 256, 1000])
def test_pages_and_types(dtype, page):
    c = Pieces([(1000, [0, 1, 30, 1025]), (7, [1, 2]), (2100, [9] * 5)], [8], 20, 256, page, dtype=dtype, seed=page)
    c.run(least=2)
    c = Pieces([(1000, [0, 1, 30, 1025]), (2100, [9] * 3)], [8], 20, 512, page, dtype=dtype, seed=page)
    c.run(least=2)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 33, 150])
@pytest.mark.parametrize("heads", [8, 16, 48])
def test_sizes_of_a_group(rows, heads):
    """Pieces that a group fills, begins and overfills; rows that hold nothing but the prefix."""
    rng = random.Random(rows)
    Pieces([(320, [rng.choice([0, rng.randint(0, 100)]) for _ in range(rows)])], (), heads, 512, 32, seed=rows).run()
    Pieces([(320, [rng.randint(0, 100) for _ in range(rows)]), (65, [1, 2])], (3,), heads, 128, 32, seed=rows).run(least=2)


@pytest.mark.parametrize("heads", [1, 16, 60])
@pytest.mark.parametrize("s1,act_q", [(2, None), (7, None), (12, None), (3, [3, 2, 0, 1, 3]), (5, [5, 1, 4, 5, 2])])
@pytest.mark.parametrize("mode", [0, 3])
@pytest.mark.parametrize("d", [256, 512])
def test_several_new_tokens(heads, s1, act_q, mode, d):
    # (packed rows of 120 heads fill a piece by themselves: nothing is shared there, and no row may name another page)
    Kind = Shared if heads == 60 and s1 == 2 and act_q is None else Pieces
    Kind([(128, [130, 64, 2]), (40, [100, 31])], (), heads, d, 16, s1=s1, seed=s1).run(mode, act_q)


@pytest.mark.parametrize("mode", [0, 3])
@pytest.mark.parametrize("s1", [1, 4])
@pytest.mark.parametrize("heads", [16, 24])
def test_idle_rows_and_rows_shorter_than_the_prefix(mode, s1, heads):
    """Idle rows first, between and last in a group (their table rows hold no page); a row that sees
    less than the prefix limits what is shared; a group of idle rows only; one of a single row."""
    c = Pieces([(192, [None, 10, None, 64, None]), (64, [None, None, None]), (130, [9]), (256, [1, 2, 3])], [1, 0],
               heads, 256, 32, s1=s1, seed=s1)
    c.run(mode, least=3)
    c.lens[1], c.lens[9], c.lens[11] = 70, 1, 38      # shorter than the shared 192 and 256
    c.run(mode)
    if s1 > 1:   # tokens before the first key
        c.lens[3] = 2
        c.run(mode)
        c.run(mode, act_q=[s1, s1 - 1, 1, s1 + 3, 0, 0, 1, 2, 3, 1, s1, 2, 0, 2])


@pytest.mark.parametrize("mode", [0, 3])
@pytest.mark.parametrize("heads,d", [(16, 512), (5, 128), (48, 256), (1, 512)])
def test_ragged_counts(mode, heads, d):
    """Rows of one token among long ones, rows without any, tokens before the first key; a padded token's
    query is NaN and reaches nothing."""
    counts = [40, 1, 0, 1, 1, 40, 3, 0, 17, 1, 1, 1, 0, 40, 0]
    c = Pieces([(256, [70, 1, None, 9, 30, 41, 5, None, 18, 1, 2]), (96, [40, None, 50])], [60], heads, d, 32, s1=40, seed=heads)
    for b, n in enumerate(counts):
        c.q[b, n:] = float("nan")
    got = c.run(mode, act_q=counts, least=2)
    assert bool(got[0].isfinite().all())
    counts[5], c.lens[5] = 40, 33                      # seven tokens before the first key (in mode 3)
    c.run(mode, act_q=counts)


@pytest.mark.parametrize("rows,s1,heads,d", [(90, 5, 8, 512), (100, 3, 50, 128), (40, 70, 16, 256), (2100, 2, 4, 128), (700, 1, 9, 128)])
def test_ragged_counts_of_many_rows(rows, s1, heads, d):
    """Windows of several rows, rows of several windows, gaps of whole windows; batches past what the plan
    holds in shared memory."""
    rng = random.Random(rows)
    few = [rng.choice([0, 0, 1, rng.randint(0, s1), s1]) if (b // 19) % 3 else 0 for b in range(rows)]
    own = [None if n == 0 and rng.random() < 0.5 else rng.randint(s1, s1 + 40) for n in few]
    cut = rows // 3
    c = Pieces([(64, own[:cut]), (40, own[cut:])], (), heads, d, 8 if d == 128 else 32, s1=s1, seed=rows)
    c.run(rng.choice([0, 3]), act_q=few)               # (of 40 rows the first group is idle)


def test_prefixes_of_any_length():
    """Longer than the rows, below zero, none, a part of a page, less than is shared."""
    c = Pieces([(200, [20, 30, 40]), (200, [5, 6]), (200, [7, 8]), (200, [9, 1])], (), 16, 128, 32, seed=1)
    for now in ([1 << 30, -1, 0, 31], [192, 33, 100, -(1 << 31)], [0, 0, 0, 0], [1, 2, 3, 191]):
        # (rows of a group have no more in common than the 192 tokens of its whole pages)
        c.prefixes = i32([min(n, 192) if n < 1 << 30 else n for n in now])
        if now[0] == 1 << 30:
            c.lens[0] = 200                            # what its shortest row sees bounds it: 6 pages
        c.run(least=0 if now[0] == 0 else 1)


def test_rows_outside_all_groups_and_empty_groups():
    c = Pieces([(200, [20, 30, 40, 50, 60])], (), 16, 128, 32, seed=2)
    for starts in ([2, 4], [0, 0, 0, 5, 5], [1, 1, 5, 5], [5, 5], [0, 2, 5]):
        c.starts, c.prefixes = i32(starts), i32([200] * (len(starts) - 1))
        c.run(least=starts != [5, 5])


@pytest.mark.parametrize("heads,rows", [(8, 30), (16, 5), (32, 12)])
@pytest.mark.parametrize("d", [256, 512])
def test_long_prefixes_are_split_and_joined(heads, rows, d):
    rng = random.Random(heads)
    Pieces([(30011, [rng.choice([0, 1, 3000]) for _ in range(rows)]), (9000, [17, 5000, 0])], [4000], heads, d, 64,
           seed=heads).run(least=2)


def test_many_groups():
    rng = random.Random(5)
    groups = [(rng.randint(0, 150), [rng.randint(0, 90) for _ in range(rng.randint(1, 6))]) for _ in range(260)]
    Pieces(groups, [rng.randint(0, 90) for _ in range(11)], 16, 128, 16, seed=5).run(least=200)
    Pieces([(64, [1, 2])] * 1100, (), 4, 128, 32, seed=6).run(least=1100)


@pytest.mark.parametrize("heads,d", [(16, 512), (48, 512), (64, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_running_maximum_that_grows(heads, d, dtype):
    c = Pieces([(1280, [1, 200, 64]), (640, [5, 500])], (), heads, d, 64, dtype=dtype, seed=5)
    for grow in (True, False):
        for b, n in enumerate(c.lens):
            for t0 in range(0, n, 64):
                page = int(c.table[b, t0 // 64])
                f = 1.5 ** (t0 // 64 % 9) if grow else 1.5 ** (9 - t0 // 64 % 9)
                c.krc[page] = (c.krc[page].float().clamp(-2, 2) * min(f, 20.0)).to(dtype)
        c.run(least=2)


@pytest.mark.parametrize("d", [128, 512])
def test_negative_scale_and_equal_scores(d):
    c = Pieces([(192, [8, 3, 0])], [5], 16, d, 16, seed=7)
    for scale in (-0.05, 0.0):
        c.scale = scale
        c.run()


@pytest.mark.parametrize("heads,d", [(16, 256), (16, 512), (40, 512)])
def test_blocks_without_a_page_in_the_prefix(heads, d):
    """Some of a prefix's blocks, and all of another's: the rows then have what is their own, or nothing."""
    c = Pieces([(300, [20, 40]), (96, [1, 0, 0])], (), heads, d, 32, seed=10)
    skip = {(b, j) for b in (0, 1) for j in (0, 4, 8)} | {(b, j) for b in (2, 3, 4) for j in (0, 1, 2)} | {(0, 9)}
    for b, j in skip:
        c.table[b, j] = -1
    got = c.run(check=False, least=2)
    dsa.check_device_errors()
    c.check(got, skip=skip)


@pytest.mark.parametrize("heads,d", [(16, 128), (16, 512), (40, 512)])
def test_a_page_past_the_pool_is_left_out_and_reported(heads, d):
    c = Pieces([(100, [20, 40])], (), heads, d, 16, seed=11)
    c.table[:, 2] = c.kc.shape[0]
    got = c.run(check=False)
    with pytest.raises(RuntimeError, match="bits 0x4"):
        dsa.check_device_errors()
    c.check(got, skip={(0, 2), (1, 2)})


@pytest.mark.parametrize("heads,d", [(16, 512), (40, 512), (16, 256), (40, 128)])
def test_nan_stays_with_its_row(heads, d):
    """A NaN in one token's query, or in keys that one row alone holds, reaches no other row; one in a
    shared key reaches every row of the group and no other."""
    c = Pieces([(320, [30, 40, 50, 60, 9]), (64, [3, 4])], [20], heads, d, 32, seed=12)
    ref = c.run(least=2)
    c.q[2, 0, 3] = float("nan")
    c.kc[int(c.table[3, 10]), 1] = float("nan")
    c.krc[int(c.table[0, 10]), 0] = float("inf")
    got = c.run(check=False)
    for b in range(8):
        same = torch.equal(got[0][b], ref[0][b])
        assert same == (b in (1, 4, 5, 6, 7)), b
    assert torch.equal(got[0][2, 0, :3], ref[0][2, 0, :3]) and bool(got[0][2, 0, 3].isnan().all())
    assert torch.equal(got[0][2, 0, 4:], ref[0][2, 0, 4:])
    assert bool(got[0][3].isnan().all()) and bool(got[2][3].isnan().all())
    c.kc[int(c.table[0, 3]), 7, 0, 5] = float("nan")
    got = c.run(check=False)
    for b in range(5):
        assert bool(got[2][b].isnan().all()), b
    assert all(torch.equal(x[5:], y[5:]) for x, y in zip(got, ref))


def test_infinite_scores():
    """Scores of -inf weigh nothing beside others; a shared key whose score is +inf makes the row NaN."""
    c = Pieces([(128, [30, 40, 5])], [20], 16, 512, 32, seed=18)
    ref = c.run()
    page = int(c.table[0, 1])
    c.q[..., 0] = c.q[..., 0].abs() + 0.5
    c.kc[page, 5, 0, 0] = float("-inf")
    got = c.run(check=False)
    dsa.check_device_errors()
    # (its value holds the -inf, too: 0 * inf in that column alone)
    for b in range(3):
        k = torch.cat([torch.cat([c.kc[p, :, 0], c.krc[p, :, 0]], -1) for p in c.table[b].tolist() if p >= 0])[:c.lens[b]].double()
        z = torch.cat([c.q[b, 0], c.qr[b, 0]], -1).double() @ k.t() * c.scale
        p = torch.softmax(z, -1)
        keep = torch.arange(k.shape[0], device="cuda") != 32 + 5
        want = p[:, keep] @ k[keep, 1:512]
        mag = p[:, keep] @ k[keep, 1:512].abs()
        ez = 576 * 2.0 ** -23 * c.scale * (torch.cat([c.q[b, 0], c.qr[b, 0]], -1).double().abs() @ k[keep].abs().t()).amax()
        bound = (2.0 ** -8 + 4 * ez + 2.0 ** -18) * mag + 2.0 ** -8 * want.abs() + 2.0 ** -24
        assert bool(((got[0][b, 0, :, 1:].double() - want).abs() <= bound).all()), b
    c.kc[page, 5, 0, 0] = float("inf")
    got = c.run(check=False)
    assert all(bool(got[2][b].isnan().all()) for b in range(3)) and bool(got[0][3].isfinite().all())
    assert ref[0].shape == got[0].shape


@pytest.mark.parametrize("d", [128, 512])
def test_queries_that_lie_otherwise_are_copied(d):
    c = Pieces([(130, [64, 33, 7])], (), 30, d, 64, s1=2, seed=8)
    out = c.run(3)
    for wide in (torch.empty(3, 2, 30, 640, device="cuda", dtype=torch.bfloat16),
                 torch.empty(3, 30, 2, 640, device="cuda", dtype=torch.bfloat16).transpose(1, 2),
                 torch.empty(3, 3, 30, 640, device="cuda", dtype=torch.bfloat16)[:, :2],
                 torch.empty(3, 2, 30, 643, device="cuda", dtype=torch.bfloat16)):
        q, qr = wide[..., 8:8 + d], wide[..., 521:585]   # the second base is not 16-byte aligned
        q.copy_(c.q)
        qr.copy_(c.qr)
        c.q, c.qr = q, qr
        assert all(torch.equal(x, y) for x, y in zip(out, c.run(3)))
    c.q, c.qr = c.q[:1].expand(3, 2, 30, d), c.qr[:1].expand(3, 2, 30, 64)
    c.run()
    one = Pieces([(130, [64, 33, 7])], (), 1, d, 64, s1=1, seed=8)     # a head, of a wider tensor
    one.q = torch.cat([one.q] * 2, 2)[:, :, 1:]
    one.run()
    step = Pieces([(130, [64, 33, 7])], (), 1, d, 64, s1=3, seed=8)    # tokens of one head, of a longer step
    step.q = torch.cat([step.q] * 2, 1)[:, 1:4]
    step.run(3)


def test_joint_cache():
    c = Pieces([(130, [64, 33, 7])], (), 16, 512, 64, seed=9)
    ref = c.run()
    pool = torch.cat([c.kc, c.krc], -1)
    c.kc, c.krc = pool[..., :512], pool[..., 512:]
    assert all(torch.equal(x, y) for x, y in zip(ref, c.run()))


@pytest.mark.parametrize("d,pages", [(512, 70000), (128, 33000)])
def test_cache_beyond_32_bit_offsets(d, pages):
    page = 64 if d == 512 else 512       # more than 2^31 latent values
    c = Pieces([(page * 2 + 22, [10, 64])], (), 16, d, page, seed=13)
    ref = c.run()
    kc = torch.zeros(pages, page, 1, d, device="cuda", dtype=torch.bfloat16)
    krc = torch.zeros(pages, page, 1, 64, device="cuda", dtype=torch.bfloat16)
    ids = sorted({int(p) for p in c.table.flatten() if p >= 0})
    for i, p in enumerate(ids):
        kc[pages - 1 - i], krc[pages - 1 - i] = c.kc[p], c.krc[p]
    where = {p: pages - 1 - i for i, p in enumerate(ids)}
    kc[0] = krc[0] = float("nan")        # the page that no row may read
    c.table = i32([[where.get(p, -1) for p in row] for row in c.table.tolist()])
    c.kc, c.krc = kc, krc
    assert all(torch.equal(x, y) for x, y in zip(ref, c.run()))


def test_same_bits_every_time_and_on_another_stream():
    c = Pieces([(9000, [100] * 9), (300, [5, 7000])], [40], 16, 512, 64, seed=14)
    ref = c.run(least=2)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(ref, c.run(check=False)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run(check=False)
    again = c.run(check=False)      # at the same time
    side.synchronize()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(ref, got, again))


def test_captured_graph_follows_lengths_counts_and_groups():
    c = Shared([(640, [100, 20, 64]), (128, [5, 70])], [40], 16, 512, 64, s1=3, seed=15)
    lens, counts, before = i32(c.lens), i32([3] * 6), list(c.lens)
    c.run(3, act_q=counts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.run(3, act_q=counts, check=False, lens=lens)
    for now, many, starts, prefixes in (
            (before, [3] * 6, [0, 3, 5], [640, 128]), ([650, 1, 0, 133, 128, 40], [1, 3, 0, 2, 1, 0], [0, 3, 5], [640, 128]),
            (before, [0, 0, 3, 1, 1, 1], [1, 3, 3], [600, 0]), (before, [2, 2, 2, 0, 0, 0], [0, 0, 6], [64, 0])):
        lens.copy_(i32(now))
        counts.copy_(i32(many))
        c.starts.copy_(i32(starts))
        c.prefixes.copy_(i32(prefixes))
        graph.replay()
        dsa.check_device_errors()
        c.lens = list(now)
        c.check(got, 3, many)


def test_without_statistics():
    c = Pieces([(77, [1, 2])], (), 16, 128, 8, seed=16)
    full = c.run()
    out, top, total = dsa.flash_attention_shared_prefix(c.q, c.qr, c.kc, c.krc, c.table, c.starts, c.prefixes,
                                                        actual_seq_lengths_key=c.lens, scale_value=c.scale)
    assert torch.equal(out, full[0]) and not top.any() and not total.any()


def test_a_long_batch_of_prompts():
    """Many tokens a row: each is a row of its own behind the prefix, and the pieces are many."""
    Pieces([(256, [60, 41, 33])], [50], 16, 128, 16, s1=40, seed=17).run(3, act_q=[40, 33, 1, 40])
    Pieces([(256, [900, 41]), (64, [2100])], [50], 16, 128, 16, s1=700, seed=17).run(3, act_q=[700, 1, 650, 3])


def test_too_many_heads_share_nothing():
    """More than 64 heads fill a piece by themselves: each row reads its own table."""
    for heads in (65, 128):
        Shared([(130, [64, 33, 7])], (), heads, 256, 64, seed=8).run()
