"""paged_cache_append and the upkeep of pages against plain Python (GPU).

Whole numbers and copied bytes have to be equal; rotated rows equal rotary_embedding's.
"""
import random

import pytest
import torch

import dsa_triton_ascend_b200 as dsa

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def errors():
    """The device error bits of the calls before, cleared."""
    try:
        dsa.check_device_errors()
        return 0
    except RuntimeError as e:
        return int(str(e).split("bits 0x")[1].split()[0], 16)


def _pool(num_pages, page, widths=(512, 64), dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return [torch.randn(num_pages, page, 1, w, generator=g, device="cuda").to(dtype) for w in widths]


def _state(rng, slots, width, pages, page, fill):
    """A consistent random pool: table, lengths, reference counts."""
    free = list(range(pages))
    rng.shuffle(free)
    table, lens, refs = [[-1] * width for _ in range(slots)], [0] * slots, [0] * pages
    for s in range(slots):
        if rng.random() > fill:
            continue
        n = rng.randint(1, width * page)
        need = -(-n // page)
        if need > len(free):
            continue
        share = 0
        donors = [d for d in range(s) if lens[d]]
        if donors and rng.random() < 0.4:
            d = rng.choice(donors)
            share = rng.randint(0, min(lens[d], n) // page)
            table[s][:share] = table[d][:share]
        for j in range(share, need):
            table[s][j] = free.pop()
        for j in range(need):
            refs[table[s][j]] += 1
        lens[s] = n
    return table, lens, refs


# ---------------------------------------------------------------------------- append

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,S,page", [(1, 1, 16), (32, 1, 128), (3, 77, 16), (2, 130, 24)])
def test_append(dtype, B, S, page):
    rng = random.Random(B + S)
    g = torch.Generator(device="cuda")
    g.manual_seed(S)
    starts = [rng.randint(0, 200) for _ in range(B)]
    counts = [S if S == 1 else rng.randint(0, S) for _ in range(B)]
    width = -(-(200 + S) // page)
    ids = list(range(B * width + 2))
    rng.shuffle(ids)
    table = [ids[b * width:(b + 1) * width] for b in range(B)]
    caches = _pool(len(ids), page, (512, 64, 128), dtype)
    tokens = [torch.randn(B, S, 1, w, generator=g, device="cuda").to(dtype) for w in (512, 64, 128)]
    rot = dsa.rotary_table(512, 64)
    pos = i32(starts)[:, None] + torch.arange(S, device="cuda", dtype=torch.int32)
    turned = [tokens[0], dsa.rotary_embedding(tokens[1], rot, pos),
              dsa.rotary_embedding(tokens[2], rot, pos, layout="half", offset=32)]
    ref = [c.clone() for c in caches]
    for c, t in zip(ref, turned):
        for b in range(B):
            for s in range(counts[b]):
                at = starts[b] + s
                c[table[b][at // page], at % page] = t[b, s]
    back = dsa.paged_cache_append(tokens, caches, i32(table), i32(starts), counts=i32(counts), table=rot,
                                  rotary=[None, ("interleaved", 0), ("half", 32)])
    assert errors() == 0
    assert all(x is y for x, y in zip(back, caches))
    assert all(torch.equal(x, y) for x, y in zip(caches, ref))


def test_append_into_a_joint_cache_from_a_joint_projection():
    """Latent and rotary keys as views of 576-wide rows, on both sides."""
    page, B, S = 64, 2, 5
    joint = torch.zeros(9, page, 1, 576, device="cuda", dtype=torch.bfloat16)
    rows = torch.randn(B, S, 1, 576, device="cuda").bfloat16()
    table = i32([[3, 1], [7, 0]])
    dsa.paged_cache_append([rows[..., :512], rows[..., 512:]], [joint[..., :512], joint[..., 512:]], table, i32([62, 0]))
    assert errors() == 0
    assert torch.equal(joint[3, 62:], rows[0, :2]) and torch.equal(joint[1, :3], rows[0, 2:])
    assert torch.equal(joint[7, :5], rows[1]) and int((joint != 0).any(-1).sum()) == 10


def test_append_unaligned_and_expanded_tokens():
    cache = torch.zeros(2, 16, 1, 64, device="cuda", dtype=torch.bfloat16)
    flat = torch.randn(4 * 67 + 1, device="cuda").bfloat16()
    rows = flat[1:].view(1, 4, 1, 67)[..., :64]
    dsa.paged_cache_append([rows], [cache], i32([[1]]), i32([2]))
    assert errors() == 0 and torch.equal(cache[1, 2:6], rows[0])
    one = torch.randn(1, 1, 1, 64, device="cuda").bfloat16().expand(1, 3, 1, 64)
    dsa.paged_cache_append([one], [cache], i32([[0]]), i32([13]))
    assert errors() == 0 and torch.equal(cache[0, 13:], one[0])


def test_append_leaves_out_what_has_no_place():
    """Positions past the block table, before 0 or past the rotary table; pages that are not."""
    page = 8
    caches = _pool(4, page, (64,))
    ref = caches[0].clone()
    tokens = torch.randn(5, 1, 1, 64, device="cuda").bfloat16()
    rot = dsa.rotary_table(12, 64)
    table = i32([[0, 1], [1, -1], [2, 4], [3, 3], [2, 2]])
    dsa.paged_cache_append([tokens], caches, table, i32([16, 8, 9, -1, 13]), table=rot, rotary=[("half", 0)])
    assert errors() == 1 << 2 and torch.equal(caches[0], ref)
    dsa.paged_cache_append([tokens], caches, table, i32([16, 8, 9, -1, 13]), counts=i32([0, 0, -3, 0, 0]))
    assert errors() == 0 and torch.equal(caches[0], ref)


# ---------------------------------------------------------------------------- bookkeeping

def _apply_extend(table, lens, refs, counts, page):
    free = [p for p, r in enumerate(refs) if r == 0]
    taken, wrong, full = 0, False, False
    for s, n in enumerate(counts):
        if n < 0 or lens[s] + n > len(table[0]) * page:
            wrong = True
            continue
        had, has = -(-lens[s] // page), -(-(lens[s] + n) // page)
        if has > had and taken + has - had > len(free):
            full, taken = True, taken + has - had
            continue
        for j in range(had, has):
            table[s][j] = free[taken]
            refs[free[taken]] = 1
            taken += 1
        lens[s] += n
    return (4 if wrong else 0) | (16 if full else 0)


def _apply_fork(table, lens, refs, parents, children, page, caches):
    free = [p for p, r in enumerate(refs) if r == 0]
    old, taken, err, made = list(lens), 0, 0, set()
    rows = [list(r) for r in table]
    for p, c in zip(parents, children):
        if not (0 <= p < len(lens) and 0 <= c < len(lens)) or old[c] or c in made:
            err |= 4
            continue
        made.add(c)
        full, rest = divmod(old[p], page)
        if rest and taken >= len(free):
            err, taken = err | 16, taken + 1
            continue
        table[c] = rows[p][:full] + [-1] * (len(rows[p]) - full)
        for j in range(full):
            refs[rows[p][j]] += 1
        if rest:
            new = free[taken]
            taken += 1
            table[c][full], refs[new] = new, 1
            for x in caches:
                x[new, :rest] = x[rows[p][full], :rest]
        lens[c] = old[p]
    return err


def _equal(got, ref):
    return all(g.tolist() == r for g, r in zip(got, ref))


@pytest.mark.parametrize("slots,width,pages,page", [(4, 3, 7, 8), (40, 9, 150, 16), (70, 33, 3000, 1), (2100, 4, 5000, 8)])
@pytest.mark.parametrize("seed", [0, 1])
def test_extend(slots, width, pages, page, seed):
    rng = random.Random(seed)
    table, lens, refs = _state(rng, slots, width, pages, page, 0.5)
    counts = [rng.choice([0, 1, page, rng.randint(0, 2 * page)]) for _ in range(slots)]
    if seed:
        counts[0], counts[-1] = -1, width * page + 1
    inputs = [i32(table), i32(lens), i32(refs)]
    keep = [t.clone() for t in inputs]
    got = dsa.paged_cache_extend(*inputs, i32(counts), page)
    err = _apply_extend(table, lens, refs, counts, page)
    assert errors() == err
    assert _equal(got, (table, lens, refs))
    assert all(torch.equal(a, b) for a, b in zip(inputs, keep))


def test_extend_when_the_pool_runs_out():
    table, lens, refs = [[0, -1], [-1, -1], [-1, -1], [-1, -1]], [5, 0, 0, 0], [1, 0, 0]
    counts = [3, 8, 16, 8]      # within its page; one page; two of one left; none left
    got = dsa.paged_cache_extend(i32(table), i32(lens), i32(refs), i32(counts), 8)
    assert errors() == 1 << 4
    assert _equal(got, ([[0, -1], [1, -1], [-1, -1], [-1, -1]], [8, 8, 0, 0], [1, 1, 0]))
    assert _apply_extend(table, lens, refs, counts, 8) == 1 << 4 and _equal(got, (table, lens, refs))


@pytest.mark.parametrize("slots,width,pages,page,n", [(4, 3, 7, 8, 2), (40, 9, 200, 16, 15), (64, 5, 5000, 24, 30), (2100, 3, 6000, 8, 1040)])
@pytest.mark.parametrize("seed", [0, 1])
def test_fork(slots, width, pages, page, n, seed):
    rng = random.Random(seed)
    table, lens, refs = _state(rng, slots, width, pages, page, 0.5)
    used, idle = [s for s in range(slots) if lens[s]] or [0], [s for s in range(slots) if not lens[s]] or [0]
    rng.shuffle(idle)
    children = idle[:n]
    parents = [rng.choice(used + idle[:1]) for _ in children]
    if seed:   # out of range, in use, twice
        parents += [-1, slots, used[0], used[0], parents[0]]
        children += [idle[-1], idle[-1], slots + 5, used[-1], children[0]]
    caches = _pool(pages, page, (64, 24), seed=seed)
    ref = [c.clone() for c in caches]
    got = dsa.paged_cache_fork(caches, i32(table), i32(lens), i32(refs), i32(parents), i32(children))
    err = _apply_fork(table, lens, refs, parents, children, page, ref)
    assert errors() == err
    assert _equal(got, (table, lens, refs))
    assert all(torch.equal(a, b) for a, b in zip(caches, ref))


def test_fork_when_the_pool_runs_out():
    table, lens, refs = [[0, 1], [-1, -1], [-1, -1], [2, -1], [-1, -1]], [12, 0, 0, 8, 0], [1, 1, 1, 0]
    parents, children = [0, 0, 3], [1, 2, 4]     # the last shares full pages only
    got = dsa.paged_cache_fork([], i32(table), i32(lens), i32(refs), i32(parents), i32(children), page_size=8)
    assert errors() == 1 << 4
    assert _apply_fork(table, lens, refs, parents, children, 8, []) == 1 << 4
    assert _equal(got, (table, lens, refs))
    assert got[0].tolist()[1] == [0, 3] and got[0].tolist()[2] == [-1, -1] and got[0].tolist()[4] == [2, -1]


@pytest.mark.parametrize("slots,width,pages", [(4, 3, 9), (60, 20, 700), (1100, 3, 4000)])
def test_free(slots, width, pages):
    rng = random.Random(slots)
    table, lens, refs = _state(rng, slots, width, pages, 8, 0.7)
    rows = [rng.randrange(slots) for _ in range(slots // 2)]     # repeats free once
    got = dsa.paged_cache_free(i32(table), i32(lens), i32(refs), i32(rows + [-1, slots]))
    assert errors() == 1 << 2
    for r in set(rows):
        for p in table[r]:
            if p >= 0:
                refs[p] -= 1
        table[r], lens[r] = [-1] * width, 0
    assert _equal(got, (table, lens, refs))


def test_free_of_a_page_that_nobody_holds():
    got = dsa.paged_cache_free(i32([[0, 1, 99], [0, -1, -1]]), i32([17, 3]), i32([1, 1]), i32([0, 1]))
    assert errors() == 1 << 2
    assert _equal(got, ([[-1] * 3] * 2, [0, 0], [0, 0]))


@pytest.mark.parametrize("slots,width,pages,page", [(3, 2, 5, 8), (50, 9, 300, 16), (30, 40, 9000, 8)])
@pytest.mark.parametrize("fill", [0.0, 0.3, 0.9])
def test_compact(slots, width, pages, page, fill):
    rng = random.Random(pages)
    table, lens, refs = _state(rng, slots, width, pages, page, fill)
    caches = _pool(pages, page, (64, 24), seed=1)
    ref = [c.clone() for c in caches]
    got = dsa.paged_cache_compact(caches, i32(table), i32(refs))
    assert errors() == 0
    live = sum(r > 0 for r in refs)
    movers = [p for p in range(live, pages) if refs[p]]
    holes = [p for p in range(live) if not refs[p]]
    where = dict(zip(movers, holes))
    for m, h in where.items():
        refs[h], refs[m] = refs[m], 0
        for x in ref:
            x[h] = x[m]
    table = [[where.get(p, p) for p in row] for row in table]
    assert _equal(got, (table, refs))
    assert all(torch.equal(a, b) for a, b in zip(caches, ref))
    assert got[1][:live].min() > 0 if live else True


def test_copy_strided_many_caches():
    """More caches than one launch takes; views of joint rows; pages of odd sizes."""
    caches = []
    for i in range(35):
        joint = torch.randint(-100, 100, (6, 5, 1, 80), device="cuda", dtype=torch.int16)
        caches.append(joint[..., 8:8 + 8 * (1 + i % 4)])
    ref = [c.clone() for c in caches]
    dsa.paged_cache_copy(caches, i32([4, -1, 0]), i32([1, 2, 5]))
    assert errors() == 0
    for c, r in zip(caches, ref):
        r[1], r[5] = r[4], r[0]
        assert torch.equal(c, r)
    dsa.paged_cache_copy(caches, i32([6, 0]), i32([0, 6]))
    assert errors() == 1 << 2
    assert all(torch.equal(c, r) for c, r in zip(caches, ref))
    dsa.paged_cache_copy(caches, i32([]), i32([]))
    assert errors() == 0


def test_copy_beyond_32_bit_offsets():
    pages, page, width = 40000, 64, 1024          # 2.6 GB
    cache = torch.empty(pages, page, 1, width, dtype=torch.uint8, device="cuda").view(torch.float16)
    cache = cache.view(pages, page, 1, width // 2)
    cache[39999] = 7.0
    cache[1] = 0.0
    dsa.paged_cache_copy([cache], i32([39999]), i32([1]))
    dsa.paged_cache_append([cache[1:2, :1] * 2], [cache], i32([[39998]]), i32([63]))
    assert errors() == 0
    assert bool((cache[1] == 7.0).all()) and bool((cache[39998, 63] == 14.0).all())


def test_upkeep_in_a_captured_graph():
    table, lens, refs = i32([[0, -1], [-1, -1]]), i32([5, 0]), i32([1, 0, 0])
    caches = _pool(3, 8, (64,))
    ref = caches[0].clone()
    step = lambda: dsa.paged_cache_fork(caches, table, lens, refs, i0, i1)
    i0, i1 = i32([0]), i32([1])
    step()
    torch.cuda.synchronize()
    caches[0].copy_(ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    assert errors() == 0
    assert _equal(out, ([[0, -1], [1, -1]], [5, 5], [1, 1, 0]))
    ref[1, :5] = ref[0, :5]
    assert torch.equal(caches[0], ref)


def test_a_report_stops_no_other_operator():
    """A pool that ran out is an answer, not a failure: attention goes on, and the report stays
    until it is asked for, by whichever name of the device."""
    q, k = torch.randn(1, 1, 4, 512, device="cuda").bfloat16(), torch.randn(1, 8, 1, 512, device="cuda").bfloat16()
    idx = torch.arange(8, device="cuda", dtype=torch.int32).reshape(1, 1, 1, 8)
    sparse = lambda: dsa.sparse_flash_attention_triton(q, k, k, idx, 0.04, query_rope=q[..., :64], key_rope=k[..., :64])[0]
    ref = sparse()
    dsa.paged_cache_extend(i32([[-1]]), i32([0]), i32([1]), i32([3]), 8)
    assert torch.equal(sparse(), ref)
    with pytest.raises(RuntimeError, match="no free page"):
        dsa.check_device_errors(torch.device("cuda", torch.cuda.current_device()))
    dsa.check_device_errors()
    dsa.paged_cache_extend(i32([[-1]]), i32([0]), i32([1]), i32([3]), 8)
    with pytest.raises(RuntimeError, match="bits 0x10"):
        dsa.check_device_errors("cuda")


def _grow_in_order(table, lens, refs, counts, page):
    """Rows in order, each taking the lowest free pages; one that what is left cannot serve takes none."""
    free = [p for p, r in enumerate(refs) if r == 0]
    err = 0
    for s, n in enumerate(counts):
        if n < 0 or lens[s] + n > len(table[0]) * page:
            err |= 1 << 2
            continue
        had, has = -(-lens[s] // page), -(-(lens[s] + n) // page)
        if has - had > len(free):
            err |= 1 << 4
            continue
        for j in range(had, has):
            table[s][j] = free.pop(0)
            refs[table[s][j]] = 1
        lens[s] += n
    return err


def test_extend_past_a_row_that_does_not_fit():
    """A row that the pool cannot serve leaves its pages to the rows after it."""
    table, lens, refs = [[0, -1, -1], [-1] * 3, [-1] * 3, [-1] * 3], [5, 0, 0, 0], [1, 0, 0]
    got = dsa.paged_cache_extend(i32(table), i32(lens), i32(refs), i32([3, 8, 16, 8]), 8)
    assert errors() == 1 << 4
    assert _equal(got, ([[0, -1, -1], [1, -1, -1], [-1] * 3, [2, -1, -1]], [8, 8, 0, 8], [1, 1, 1]))
    # a prompt that is too long, before decode steps of one page each
    table, lens, refs = [[-1] * 6 for _ in range(5)], [0] * 5, [0] * 4
    got = dsa.paged_cache_extend(i32(table), i32(lens), i32(refs), i32([48, 1, 2, 3, 8]), 8)
    assert errors() == 1 << 4
    assert got[1].tolist() == [0, 1, 2, 3, 8] and [r[0] for r in got[0].tolist()] == [-1, 0, 1, 2, 3]


@pytest.mark.parametrize("slots,width,pages,page", [(6, 5, 9, 8), (300, 20, 700, 16), (1024, 9, 1500, 8),
                                                    (3000, 7, 4000, 4), (3000, 7, 140000, 4)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_extend_of_more_than_the_pool_holds(slots, width, pages, page, seed):
    """Requests of every size against a pool that runs out early, late, or within a block of rows."""
    rng = random.Random(seed)
    refs = [int(rng.random() < 0.3 + 0.3 * seed) for _ in range(pages)]
    if pages > 8 * slots:
        refs[2 * slots * seed + 40:] = [1] * (pages - 2 * slots * seed - 40)
    lens = [rng.choice([0, 0, 1, page, page + 1]) for _ in range(slots)]
    table = [[rng.randrange(pages) if j * page < n else -1 for j in range(width)] for n in lens]
    counts = [rng.choice([0, 1, page, rng.randint(0, width * page), rng.randint(0, (width - 2) * page)]) for _ in range(slots)]
    got = dsa.paged_cache_extend(i32(table), i32(lens), i32(refs), i32(counts), page)
    assert errors() == _grow_in_order(table, lens, refs, counts, page)
    assert _equal(got, (table, lens, refs))


def test_append_rotates_rows_of_several_types():
    """Rotated rows of two and three types, with and without copied ones beside them."""
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    types = [torch.bfloat16, torch.float16, torch.float32, torch.bfloat16]
    B, S, page = 3, 21, 16
    starts, counts = [5, 0, 40], [21, 0, 13]
    table = [[4, 1, 9, 7], [2, 3, 0, 5], [6, 8, 10, 11]]
    rot = dsa.rotary_table(64, 64)
    pos = i32(starts)[:, None] + torch.arange(S, device="cuda", dtype=torch.int32)
    for rotary in ([("interleaved", 0), ("half", 64), None, None], [("half", 0), ("half", 32), ("interleaved", 4), None],
                   [None, ("interleaved", 8), ("half", 64), ("interleaved", 0)]):
        caches = [torch.randn(12, page, 1, 128, generator=g, device="cuda").to(t) for t in types]
        tokens = [torch.randn(B, S, 1, 128, generator=g, device="cuda").to(t) for t in types]
        ref = [c.clone() for c in caches]
        for c, t, r in zip(ref, tokens, rotary):
            if r is not None:
                t = dsa.rotary_embedding(t, rot, pos, layout=r[0], offset=r[1])
            for b in range(B):
                for s in range(counts[b]):
                    at = starts[b] + s
                    c[table[b][at // page], at % page] = t[b, s]
        dsa.paged_cache_append(tokens, caches, i32(table), i32(starts), counts=i32(counts), table=rot, rotary=rotary)
        assert errors() == 0
        assert all(torch.equal(x, y) for x, y in zip(caches, ref))


@pytest.mark.parametrize("B,S", [(0, 1), (0, 5), (3, 0), (0, 0)])
def test_nothing_to_append(B, S):
    """A step without sequences or without tokens writes nothing, as the other operators take it."""
    caches = _pool(4, 8, (64, 128))
    ref = [c.clone() for c in caches]
    tokens = [torch.empty(B, S, 1, w, device="cuda", dtype=torch.bfloat16) for w in (64, 128)]
    table, starts = torch.zeros(B, 2, device="cuda", dtype=torch.int32), torch.zeros(B, device="cuda", dtype=torch.int32)
    rot = dsa.rotary_table(16, 64)
    for _ in range(2):
        for kw in (dict(), dict(counts=starts), dict(table=rot, rotary=[("half", 0), None])):
            back = dsa.paged_cache_append(tokens, caches, table, starts, **kw)
            assert all(x is y for x, y in zip(back, caches))
    assert errors() == 0 and all(torch.equal(a, b) for a, b in zip(caches, ref))


def test_upkeep_of_no_rows():
    table, lens, refs, none = i32([[0, -1], [-1, -1]]), i32([5, 0]), i32([1, 0]), i32([])
    caches = _pool(2, 8, (64,))
    keep = caches[0].clone()
    for _ in range(2):
        assert _equal(dsa.paged_cache_fork(caches, table, lens, refs, none, none), ([[0, -1], [-1, -1]], [5, 0], [1, 0]))
        assert _equal(dsa.paged_cache_free(table, lens, refs, none), ([[0, -1], [-1, -1]], [5, 0], [1, 0]))
        assert _equal(dsa.paged_cache_extend(table, lens, refs, i32([0, 0]), 8), ([[0, -1], [-1, -1]], [5, 0], [1, 0]))
    assert errors() == 0 and torch.equal(caches[0], keep)
