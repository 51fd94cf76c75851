"""flash_attention_shared_prefix against attention in 64 bits (GPU).

The reference and its tolerances are those of flash_attention_paged (test_attn_paged_gpu.py): the
join of a prefix's parts with a row's own is one more fp32 sum of the few that the 2^-18 there allows.
"""
import importlib
import math
import random

import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from dsa_triton_ascend_b200 import _lib
from test_attn_paged_gpu import Case, i32

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def give_memory_back():
    """Large blocks that stay in torch's cache would serve a later test that counts on its being empty."""
    yield
    torch.cuda.empty_cache()


@pytest.fixture(autouse=True)
def small_calls_share(monkeypatch):
    """Prefixes are shared however little that saves."""
    module = importlib.import_module("dsa_triton_ascend_b200.flash_attention_paged")
    monkeypatch.setattr(module, "_LEAST_SAVING", 0)
    if _lib.binding() is not None:   # which keeps what a signature's first call decided
        monkeypatch.setattr(module, "binding", lambda: None)
        monkeypatch.setattr(module, "remember", lambda *a: None)


class Shared(Case):
    """Groups (shared tokens, [tokens of each row behind them; None: an idle row]), then rows of their
    own.  Unused rows and pages hold NaN."""

    def __init__(self, groups, alone=(), heads=16, d=512, page=64, s1=1, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(dtype)
        rows = [(i, None if own is None else n + own, n) for i, (n, more) in enumerate(groups) for own in more]
        rows += [(None, n, 0) for n in alone]
        self.lens, self.page, self.scale = [n or 0 for _, n, _ in rows], page, 1.0 / math.sqrt(d + 64)
        B = len(rows)
        self.q, self.qr = rnd(B, s1, heads, d), rnd(B, s1, heads, 64)
        need = sum(n // page for n, _ in groups) + sum(-(-(n or 0) // page) for _, n, _ in rows) + 2
        ids = list(range(need))
        random.Random(seed).shuffle(ids)
        pool = torch.full((need, page, 1, d + 64), float("nan"), device="cuda", dtype=dtype)
        first = [[ids.pop() for _ in range(n // page)] for n, _ in groups]
        for pages in first:
            for p in pages:
                pool[p] = rnd(page, 1, d + 64)
        width = max([1] + [-(-n // page) for n in self.lens])
        table = []
        for i, n, _ in rows:
            row = list(first[i]) if i is not None and n is not None else []
            row = row[:-(-(n or 0) // page)]
            for j in range(len(row), -(-(n or 0) // page)):
                row.append(ids.pop())
                m = min(page, n - j * page)
                pool[row[-1], :m] = rnd(m, 1, d + 64)
            table.append(row + [-1] * (width - len(row)))
        self.table = i32(table)
        starts = [0]
        for _, more in groups:
            starts.append(starts[-1] + len(more))
        self.starts, self.prefixes = i32(starts), i32([n for n, _ in groups])
        self.kc, self.krc = pool[..., :d].contiguous(), pool[..., d:].contiguous()

    def run(self, mode=0, act_q=None, check=True, lens=None, **kw):
        got = dsa.flash_attention_shared_prefix(
            self.q, self.qr, self.kc, self.krc, self.table, self.starts, self.prefixes,
            actual_seq_lengths_key=i32(self.lens) if lens is None else lens, scale_value=self.scale,
            actual_seq_lengths_query=act_q, sparse_mode=mode, return_softmax_lse=True, **kw)
        if check:
            dsa.check_device_errors()
            self.check(got, mode, act_q)
        return got


@pytest.mark.parametrize("heads", [1, 5, 16, 17, 32, 40, 64, 65, 128])
@pytest.mark.parametrize("d", [128, 256, 512])
def test_heads_and_widths(heads, d):
    Shared([(130, [0, 1, 63]), (64, [5] * 9), (1000, [200, 3])], [0, 70], heads, d, seed=heads).run()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 256, 1000])
def test_pages_and_types(dtype, page):
    Shared([(1000, [0, 1, 30, 1025]), (7, [1, 2]), (2100, [9] * 5)], [8], 20, 256, page, dtype=dtype, seed=page).run()


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 33, 150])
@pytest.mark.parametrize("heads", [8, 16, 48])
def test_sizes_of_a_group(rows, heads):
    """Pieces that a group fills, begins and overfills."""
    rng = random.Random(rows)
    Shared([(320, [rng.randint(0, 100) for _ in range(rows)])], (), heads, 512, 32, seed=rows).run()
    Shared([(320, [rng.randint(0, 100) for _ in range(rows)]), (65, [1, 2])], (3,), heads, 128, 32, seed=rows).run()


@pytest.mark.parametrize("heads", [1, 16, 60])
@pytest.mark.parametrize("s1,act_q", [(2, None), (7, None), (12, None), (3, [3, 2, 0, 1, 3]), (5, [5, 1, 4, 5, 2])])
@pytest.mark.parametrize("mode", [0, 3])
def test_several_new_tokens(heads, s1, act_q, mode):
    Shared([(128, [130, 64, 2]), (40, [100, 31])], (), heads, 512, 16, s1=s1, seed=s1).run(mode, act_q)


@pytest.mark.parametrize("mode", [0, 3])
@pytest.mark.parametrize("s1", [1, 4])
def test_idle_rows_and_rows_shorter_than_the_prefix(mode, s1):
    """Idle rows first, between and last in a group (their table rows hold no page); a row that sees
    less than the prefix limits what is shared; a group of idle rows only; one of a single row."""
    c = Shared([(192, [None, 10, None, 64, None]), (64, [None, None, None]), (130, [9]), (256, [1, 2, 3])], [1, 0],
               16, 256, 32, s1=s1, seed=s1)
    c.run(mode)
    c.lens[1], c.lens[9], c.lens[11] = 70, 1, 31      # shorter than the shared 192 and 256
    c.run(mode)
    if s1 > 1:   # tokens before the first key
        c.lens[3] = 2
        c.run(mode)
        c.run(mode, act_q=[s1, s1 - 1, 1, s1 + 3, 0, 0, 1, 2, 3, 1, s1, 2, 0, 2])


def test_prefixes_of_any_length():
    """Longer than the rows, below zero, none, a part of a page, less than is shared."""
    c = Shared([(200, [20, 30, 40]), (200, [5, 6]), (200, [7, 8]), (200, [9, 1])], (), 16, 128, 32, seed=1)
    for now in ([1 << 30, -1, 0, 31], [192, 33, 100, -(1 << 31)], [0, 0, 0, 0], [1, 2, 3, 191]):
        c.prefixes = i32(now)
        c.run()


@pytest.mark.parametrize("page", [8, 32, 1000])
def test_idle_groups_and_empty_ones_with_endless_prefixes(page):
    """Nothing bounds the prefix of a group without a row that sees keys: it shares nothing."""
    c = Shared([(2000, [None, None, None, None]), (2000, [20, 30, None]), (64, [None])], [5], 16, 128, page, seed=4)
    c.starts = i32([0, 4, 4, 7, 8])
    for now in ((1 << 31) - 1, (1 << 31) - 64, (1 << 31) - 65, 1 << 30, 1 << 21):
        c.prefixes = i32([now, now, 2000, now])
        c.run()


def test_rows_outside_all_groups_and_empty_groups():
    c = Shared([(200, [20, 30, 40, 50, 60])], (), 16, 128, 32, seed=2)
    for starts in ([2, 4], [0, 0, 0, 5, 5], [1, 1, 5, 5], [5, 5], [0, 2, 5]):
        c.starts, c.prefixes = i32(starts), i32([200] * (len(starts) - 1))
        c.run()
    c.starts, c.prefixes = i32([0]), i32([])
    c.run()


@pytest.mark.parametrize("starts", [[0, 6], [-1, 3], [3, 1, 5], [0, 1 << 30], [0, 4, 2, 5]])
def test_starts_that_divide_no_batch(starts):
    """Nothing is shared, and it is reported; the result is the same."""
    c = Shared([(200, [20, 30, 40, 50, 60])], (), 16, 128, 32, seed=3)
    c.starts, c.prefixes = i32(starts), i32([200] * (len(starts) - 1))
    got = c.run(check=False)
    with pytest.raises(RuntimeError, match="bits 0x4"):
        dsa.check_device_errors()
    c.check(got)


@pytest.mark.parametrize("heads,rows", [(8, 30), (16, 5), (32, 12)])
@pytest.mark.parametrize("d", [256, 512])
def test_long_prefixes_are_split_and_joined(heads, rows, d):
    rng = random.Random(heads)
    Shared([(30011, [rng.choice([0, 1, 3000]) for _ in range(rows)]), (9000, [17, 5000, 0])], [4000], heads, d, 64,
           seed=heads).run()


def test_many_groups():
    rng = random.Random(5)
    groups = [(rng.randint(0, 150), [rng.randint(0, 90) for _ in range(rng.randint(1, 6))]) for _ in range(260)]
    Shared(groups, [rng.randint(0, 90) for _ in range(11)], 16, 128, 16, seed=5).run()
    Shared([(64, [1, 2])] * 1100, (), 4, 128, 32, seed=6).run()


@pytest.mark.parametrize("heads,d", [(16, 512), (48, 512), (64, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_running_maximum_that_grows(heads, d, dtype):
    c = Shared([(1280, [1, 200, 64]), (640, [5, 500])], (), heads, d, 64, dtype=dtype, seed=5)
    for grow in (True, False):
        for b, n in enumerate(c.lens):
            for t0 in range(0, n, 64):
                page = int(c.table[b, t0 // 64])
                f = 1.5 ** (t0 // 64 % 9) if grow else 1.5 ** (9 - t0 // 64 % 9)
                c.krc[page] = (c.krc[page].float().clamp(-2, 2) * min(f, 20.0)).to(dtype)
        c.run()


def test_negative_scale_and_equal_scores():
    c = Shared([(192, [8, 3, 0])], [5], 16, 128, 16, seed=7)
    for scale in (-0.05, 0.0):
        c.scale = scale
        c.run()


def test_blocks_without_a_page_in_the_prefix():
    c = Shared([(300, [20, 40]), (96, [1, 0, 0])], (), 16, 256, 32, seed=10)
    skip = {(b, j) for b in (0, 1) for j in (0, 4, 8)} | {(b, j) for b in (2, 3, 4) for j in (0, 1, 2)} | {(0, 9)}
    for b, j in skip:
        c.table[b, j] = -1
    got = c.run(check=False)
    dsa.check_device_errors()
    c.check(got, skip=skip)


def test_a_page_past_the_pool_is_left_out_and_reported():
    c = Shared([(100, [20, 40])], (), 16, 128, 16, seed=11)
    c.table[:, 2] = c.kc.shape[0]
    got = c.run(check=False)
    with pytest.raises(RuntimeError, match="bits 0x4"):
        dsa.check_device_errors()
    c.check(got, skip={(0, 2), (1, 2)})


@pytest.mark.parametrize("heads", [16, 40])
def test_nan_stays_with_its_row(heads):
    """A NaN in one token's query, or in keys that one row alone holds, reaches no other row."""
    c = Shared([(320, [30, 40, 50, 60, 9])], [20], heads, 512, 32, seed=12)
    ref = c.run()
    c.q[2, 0, 3] = float("nan")
    c.kc[int(c.table[3, 10]), 1] = float("nan")
    c.krc[int(c.table[0, 10]), 0] = float("inf")
    got = c.run(check=False)
    for b in range(6):
        same = torch.equal(got[0][b], ref[0][b])
        assert same == (b in (1, 4, 5)), b
    assert torch.equal(got[0][2, 0, :3], ref[0][2, 0, :3]) and bool(got[0][2, 0, 3].isnan().all())
    assert bool(got[0][3].isnan().all()) and bool(got[2][3].isnan().all())


def test_queries_that_lie_otherwise_are_copied():
    c = Shared([(130, [64, 33, 7])], (), 40, 512, 64, s1=2, seed=8)
    out = c.run(3)
    for wide in (torch.empty(3, 2, 40, 640, device="cuda", dtype=torch.bfloat16),
                 torch.empty(3, 40, 2, 640, device="cuda", dtype=torch.bfloat16).transpose(1, 2),
                 torch.empty(3, 3, 40, 640, device="cuda", dtype=torch.bfloat16)[:, :2],
                 torch.empty(3, 2, 40, 643, device="cuda", dtype=torch.bfloat16)):
        q, qr = wide[..., 8:520], wide[..., 521:585]   # the second base is not 16-byte aligned
        q.copy_(c.q)
        qr.copy_(c.qr)
        c.q, c.qr = q, qr
        assert all(torch.equal(x, y) for x, y in zip(out, c.run(3)))
    c.q, c.qr = c.q[:1].expand(3, 2, 40, 512), c.qr[:1].expand(3, 2, 40, 64)
    c.run()
    one = Shared([(130, [64, 33, 7])], (), 1, 128, 64, s1=1, seed=8)     # a head, of a wider tensor
    one.q = torch.cat([one.q] * 2, 2)[:, :, 1:]
    one.run()


def test_joint_cache():
    c = Shared([(130, [64, 33, 7])], (), 16, 512, 64, seed=9)
    ref = c.run()
    pool = torch.cat([c.kc, c.krc], -1)
    c.kc, c.krc = pool[..., :512], pool[..., 512:]
    assert all(torch.equal(x, y) for x, y in zip(ref, c.run()))


def test_cache_beyond_32_bit_offsets():
    page, d = 64, 512
    c = Shared([(150, [10, 64])], (), 16, d, page, seed=13)
    ref = c.run()
    kc = torch.zeros(34000, page, 1, d, device="cuda", dtype=torch.bfloat16)
    krc = torch.zeros(34000, page, 1, 64, device="cuda", dtype=torch.bfloat16)
    ids = sorted({int(p) for p in c.table.flatten() if p >= 0})
    for i, p in enumerate(ids):
        kc[33999 - i], krc[33999 - i] = c.kc[p], c.krc[p]
    where = {p: 33999 - i for i, p in enumerate(ids)}
    c.table = i32([[where.get(p, -1) for p in row] for row in c.table.tolist()])
    c.kc, c.krc = kc, krc
    assert all(torch.equal(x, y) for x, y in zip(ref, c.run()))


def test_same_bits_every_time_and_on_another_stream():
    c = Shared([(9000, [100] * 9), (300, [5, 7000])], [40], 16, 512, 64, seed=14)
    ref = c.run()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(ref, c.run(check=False)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run(check=False)
    again = c.run(check=False)      # at the same time
    side.synchronize()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(ref, got, again))


def test_captured_graph_follows_lengths_groups_and_prefixes():
    c = Shared([(640, [100, 20, 64]), (128, [5, 70])], [40], 16, 512, 64, seed=15)
    lens, before = i32(c.lens), list(c.lens)
    c.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = c.run(check=False, lens=lens)
    for now, starts, prefixes in ((before, [0, 3, 5], [640, 128]), ([650, 1, 0, 133, 128, 40], [0, 3, 5], [640, 128]),
                                  (before, [1, 3, 3], [600, 0]), (before, [0, 0, 6], [64, 0])):
        lens.copy_(i32(now))
        c.starts.copy_(i32(starts))
        c.prefixes.copy_(i32(prefixes))
        graph.replay()
        dsa.check_device_errors()
        c.lens = list(now)
        c.check(got)


def test_without_statistics_and_without_rows():
    c = Shared([(77, [1, 2])], (), 16, 128, 8, seed=16)
    full = c.run()
    out, top, total = dsa.flash_attention_shared_prefix(c.q, c.qr, c.kc, c.krc, c.table, c.starts, c.prefixes,
                                                        actual_seq_lengths_key=c.lens, scale_value=c.scale)
    assert torch.equal(out, full[0]) and not top.any() and not total.any()
    out, _, _ = dsa.flash_attention_shared_prefix(c.q[:0], c.qr[:0], c.kc, c.krc, c.table[:0], c.starts[:1] * 0,
                                                  c.prefixes[:0])
    assert out.shape == (0, 1, 16, 128)
    c.starts = torch.stack([c.starts, c.starts], 1)[:, 0]          # strided lists are read as they are
    c.prefixes = torch.stack([c.prefixes, c.prefixes], 1)[:, 0]
    assert all(torch.equal(x, y) for x, y in zip(full, c.run()))


def test_a_long_batch_of_prompts():
    """Many tokens a row: each is a row of its own behind the prefix, and the pieces are many."""
    Shared([(256, [60, 41, 33])], [50], 16, 128, 16, s1=40, seed=17).run(3, act_q=[40, 33, 1, 40])
