"""paged_batch_plan and paged_cache_store against plain Python (GPU): whole numbers and copies, exact."""
import random

import pytest
import torch

import dsa_triton_ascend_b200 as dsa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def give_memory_back():
    """Large blocks that stay in torch's cache would serve a later test that counts on its being empty."""
    yield
    torch.cuda.empty_cache()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def errors():
    try:
        dsa.check_device_errors("cuda")
    except RuntimeError as e:
        return int(str(e).split("bits ")[1].split(" ")[0], 16)
    return 0


def _expect(table, lens, rows, counts, page, T, most, least):
    """The plan as lists, and the error bits."""
    B, width, err = len(rows), len(table[0]), 0
    req = []
    for r, c in zip(rows, counts):
        n = lens[r] if 0 <= r < len(lens) else 0
        if not 0 <= r < len(lens) or c < 0 or c > n or n > width * page:
            err, r, n, c = 4, 0, 0, max(c, 0)
        req.append((r, n, c))
    out = [[table[r][j] if j * page < n else -1 for j in range(width)] for r, n, _ in req]
    ends, where, pos, slots = [], [], [], []
    for b, (r, n, c) in enumerate(req):
        for p in range(n - c, n):
            if p < 0:   # of a request that cannot be: its place is kept
                where.append(-1)
                pos.append(0)
                slots.append(-1)
                continue
            where.append(b)
            pos.append(p)
            slots.append(-1 if table[r][p // page] < 0 else table[r][p // page] * page + p % page)
            err |= 4 if slots[-1] < 0 and len(slots) <= T else 0
        ends.append(len(where))
    err |= 4 if len(where) > T else 0
    pad = T - len(where)
    lists = [(x + [v] * pad)[:T] for x, v in ((where, -1), (pos, 0), (slots, -1))]
    groups = []
    for b, (r, n, c) in enumerate(req):
        same = 0
        if b:
            o, m, d = req[b - 1]
            whole = min(n - c, m - d) // page
            while same < whole and table[r][same] >= 0 and table[r][same] == table[o][same]:
                same += 1
        if b == 0 or same * page < max(least, page):
            groups.append([b, None])
        else:
            groups[-1][1] = same * page if groups[-1][1] is None else min(groups[-1][1], same * page)
    starts = ([g[0] for g in groups] + [B] * (most + 1))[:most + 1]
    prefixes = ([g[1] or 0 for g in groups] + [0] * most)[:most]
    return (out, [n for _, n, _ in req], ends, *lists, starts, prefixes), err


def _pool(rng, slots, width, page, share):
    """A table in which many slots continue another one's first pages."""
    table, lens, fresh = [], [], 0
    for s in range(slots):
        n = rng.choice([0, 1, page, rng.randint(0, width * page), rng.randint(0, width * page)])
        row = []
        if s and rng.random() < share:
            o = rng.choice([s - 1, rng.randrange(s)])
            row = table[o][:rng.randint(0, min(n, lens[o]) // page)]
        while len(row) * page < n:
            row.append(fresh)
            fresh += 1
        table.append(row + [-1] * (width - len(row)))
        lens.append(n)
    ids = list(range(max(fresh, 1)))
    rng.shuffle(ids)
    return [[ids[p] if p >= 0 else -1 for p in row] for row in table], lens


def _check(table, lens, rows, counts, page, T, most=None, least=1):
    want, err = _expect(table, lens, rows, counts, page, T, len(rows) if most is None else most, least)
    for _ in range(2):   # a new signature, and the same again
        got = dsa.paged_batch_plan(i32(table), i32(lens), i32(rows), i32(counts), page, T, max_groups=most, min_prefix=least)
        assert errors() == err
        for g, w, name in zip(got, want, got._fields):
            assert g.tolist() == w, name
        assert got.slot_map.dtype == torch.int64 and all(g.dtype == torch.int32 for g in got if g is not got.slot_map)
    return got


@pytest.mark.parametrize("slots,width,page,batch", [(1, 1, 1, 1), (6, 5, 8, 4), (40, 33, 16, 40), (70, 300, 1, 64),
                                                    (300, 9, 64, 257), (1500, 20, 8, 1300), (5000, 2, 16, 4100)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_plan(slots, width, page, batch, seed):
    rng = random.Random(seed)
    table, lens = _pool(rng, slots, width, page, 0.3 * seed + 0.2)
    rows = sorted(rng.sample(range(slots), batch)) if seed else [rng.randrange(slots) for _ in range(batch)]
    counts = [rng.choice([min(1, lens[r]), 0, rng.randint(0, lens[r])]) for r in rows]
    T = sum(counts)
    for T, most, least in ((T, None, 1), (T + 70, batch // 2, 3 * page), (T + 1, 1, 0), (T, 0, page + 1)):
        _check(table, lens, rows, counts, page, T, most, least)


def test_long_prompts_and_tables():
    """Requests of many thousands of tokens; rows of several spans, alike up to the last page or to a gap."""
    rng = random.Random(9)
    width, page = 2100, 16
    base = list(range(width))
    rng.shuffle(base)
    table = [list(base) for _ in range(7)]
    for s, j in ((1, 2099), (2, 256), (3, 255), (4, 31), (5, 1024)):
        table[s][j] = width + s
    table[6][700] = -1
    lens = [width * page, width * page, width * page - 3, 9000, width * page, width * page - 1, width * page]
    _check(table, lens, list(range(7)), [20000, 0, 1, 9000, 17, 2, 3], page, 30000)
    _check(table, lens, [0, 6, 6, 0, 1, 1], [0, 1, 1, 0, 0, 0], page, 3)


@pytest.mark.parametrize("batch", [1, 2, 8, 16, 24, 48, 56, 57])
@pytest.mark.parametrize("T", [0, 1, 1023, 1024, 1025, 5000, 6144, 6145, 9000])
def test_small_steps_of_any_number_of_tokens(batch, T):
    """One launch or two, by requests and blocks of tokens; the last tokens behind the requests' or left out."""
    rng = random.Random(batch * T)
    table, lens = _pool(rng, 60, 40, 16, 0.7)
    rows = rng.sample(range(60), batch)
    counts = [rng.randint(0, lens[r]) for r in rows]
    _check(table, lens, rows, counts, 16, T)


def test_requests_that_cannot_be():
    table, lens = [[0, 1, 2], [3, 4, -1], [5, -1, -1]], [20, 16, 99]
    _check(table, lens, [0, 1, -1, 3, 1, 0, 2], [1, 2, 1, 1, -1, 21, 1], 8, 4)
    _check(table, [20, 24, 8], [0, 1, 2], [1, 9, 8], 8, 18)            # tokens without a page
    _check(table, [20, 16, 8], [0, 1, 2], [5, 6, 7], 8, 9)             # more than there is room for
    _check(table, [-5, 16, 8], [0, 1, 2], [0, 0, 0], 8, 5)


def test_without_requests_tokens_or_groups():
    table, lens = [[0, 1], [2, 3]], [5, 16]
    got = _check(table, lens, [], [], 8, 3)
    assert got.group_starts.tolist() == [0]
    _check(table, lens, [], [], 8, 0, 4)
    _check(table, lens, [1, 0], [0, 0], 8, 0)


def test_state_is_left_as_it_was_and_captured():
    rng = random.Random(3)
    table, lens = _pool(rng, 30, 12, 16, 0.6)
    rows = list(range(20))
    state = [i32(table), i32(lens), i32(rows), i32([min(2, lens[r]) for r in rows])]
    keep = [t.clone() for t in state]
    call = lambda: dsa.paged_batch_plan(*state, 16, 41)
    ref = call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for now in (rows, rows[::-1], [5] * 20):
        state[2].copy_(i32(now))
        state[3].copy_(i32([min(1, lens[r]) for r in now]))
        graph.replay()
        want, err = _expect(table, lens, now, [min(1, lens[r]) for r in now], 16, 41, 20, 1)
        assert errors() == err and all(g.tolist() == w for g, w in zip(got, want))
    side = torch.cuda.Stream()
    for t, k in zip(state, keep):
        t.copy_(k)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = call()
    here = call()
    side.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(ref, there, here))
    assert all(torch.equal(a, b) for a, b in zip(state, keep))


def test_strided_state():
    rng = random.Random(4)
    table, lens = _pool(rng, 9, 6, 8, 0.5)
    counts = [min(3, n) for n in lens]
    ref = dsa.paged_batch_plan(i32(table), i32(lens), i32(list(range(9))), i32(counts), 8, 30)
    wide = lambda t: torch.stack([t, t * 0 - 7], -1)[..., 0]
    got = dsa.paged_batch_plan(wide(i32(table)), wide(i32(lens)), wide(i32(list(range(9)))), wide(i32(counts)), 8, 30)
    assert all(torch.equal(a, b) for a, b in zip(ref, got)) and errors() == 0


# ------------------------------------------------------------------------------------------

def _stored(tokens, caches, slots):
    caches = [c.clone() for c in caches]
    for i, s in enumerate(slots):
        if 0 <= s < caches[0].shape[0] * caches[0].shape[1]:
            for t, c in zip(tokens, caches):
                c[s // c.shape[1], s % c.shape[1]] = t[i]
    return caches


@pytest.mark.parametrize("page,pages,T", [(8, 5, 1), (8, 5, 40), (24, 50, 333), (128, 90, 3000), (1, 100, 7)])
@pytest.mark.parametrize("widths,dtype", [((512, 64, 128), torch.bfloat16), ((8,), torch.float16), ((4, 1024), torch.float32),
                                          ((16, 144, 32, 16), torch.uint8), ((4096, 64), torch.bfloat16)])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_store(page, pages, T, widths, dtype, index):
    rng = random.Random(T)
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    rnd = lambda *shape: torch.randint(0, 255, shape, generator=g, device="cuda").to(dtype)
    slots = rng.sample(range(page * pages), min(T, page * pages))
    slots = [-1 if rng.random() < 0.1 else s for s in slots] + [-1 << 31] * (T - len(slots))
    tokens, caches = [rnd(T, 1, w) for w in widths], [rnd(pages, page, 1, w) for w in widths]
    want = _stored(tokens, caches, slots)
    got = dsa.paged_cache_store(tokens, caches, torch.tensor(slots, device="cuda", dtype=index))
    assert errors() == 0
    assert all(a is b and torch.equal(a, c) for a, b, c in zip(got, caches, want))


def test_store_leaves_out_slots_past_the_pool_and_reports():
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    tokens, cache = torch.randn(5, 1, 64, generator=g, device="cuda").half(), torch.zeros(3, 8, 1, 64, device="cuda").half()
    slots = [23, 24, 1 << 40, -5, 0]
    want = _stored([tokens], [cache], slots)
    dsa.paged_cache_store([tokens], [cache], torch.tensor(slots, device="cuda"))
    assert errors() == 4 and torch.equal(cache, want[0])


def test_store_of_strided_tokens_into_parts_of_a_joint_cache():
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    pool = torch.randn(6, 16, 1, 704, generator=g, device="cuda").bfloat16()
    wide = torch.randn(40, 3, 700, generator=g, device="cuda").bfloat16()
    caches = [pool[..., :512], pool[..., 512:576], pool[..., 576:]]
    keep = pool.clone()
    slots = random.Random(1).sample(range(96), 40)
    # in place, at an address that is not aligned, and with a stride between values
    for tokens in ([wide[:, 1:2, :512], wide[:, :1, 520:584], wide[:, 2:, 0:128]],
                   [wide[:, 1:2, 1:513], wide[:, :1, 3:67], wide[:, :1, 0:256:2]],
                   [wide[:1, :1, :512].expand(40, 1, 512), wide[:, :1, :64], wide[:, 1:2, :128]]):
        want = _stored(tokens, caches, slots)
        dsa.paged_cache_store(tokens, caches, torch.tensor(slots, device="cuda"))
        assert errors() == 0 and all(torch.equal(a, b) for a, b in zip(caches, want))
        pool.copy_(keep)


def test_store_past_32_bits_captured_and_without_tokens():
    cache = torch.zeros(70000, 64, 1, 512, device="cuda", dtype=torch.bfloat16)      # 4.6 GB
    tokens = torch.randn(3, 1, 512, device="cuda").bfloat16()
    slots = torch.tensor([70000 * 64 - 1, 0, 3333333], device="cuda")
    graph = torch.cuda.CUDAGraph()
    dsa.paged_cache_store([tokens], [cache], slots)
    with torch.cuda.graph(graph):
        dsa.paged_cache_store([tokens], [cache], slots)
    slots.copy_(torch.tensor([5, -1, 70000 * 64 - 2], device="cuda"))
    graph.replay()
    flat = cache.view(-1, 512)
    for s, t in ((70000 * 64 - 1, 0), (0, 1), (3333333, 2), (5, 0), (70000 * 64 - 2, 2)):
        assert torch.equal(flat[s], tokens[t, 0])
        flat[s] = 0
    assert errors() == 0 and not cache.any()
    assert dsa.paged_cache_store([tokens[:0]], [cache], slots[:0])[0] is cache
