"""Operators for batches that share a prompt: what a pass of each costs and gives.

Four operators, as a step over a paged cache calls them: the step's plan from its requests'
lengths (block table, slot map, positions, groups of rows with common pages), rotary positions
with several axes on queries and keys, the store of packed tokens by their slots, and attention
that computes a shared prefix once for the rows that share it.  ``run`` computes a pass with
elementary torch operations, or, where ``own`` is true, through the package's operators.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_ROPE = 64          # rotary part of a latent key
_INDEX = 128        # an index key's width


def _dsa():
    import dsa_triton_ascend_b200 as dsa
    return dsa


# ------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------

def listed():
    return [
        # four samples of one short prompt, few heads left on this GPU by head sharding: latency
        {"name": "shared_samples", "op": "attention", "dtype": "bf16", "batch": 4, "s1": 1, "heads": 16, "d": 512,
         "page": 64, "groups": 1, "alone": 0, "empty": 0, "prefix_lo": 1021, "prefix_hi": 1021, "own_lo": 1,
         "own_hi": 130, "mode": 0},
        # 64 answers to questions about one long document, in whole pages and a rest of its own
        {"name": "shared_document", "op": "attention", "dtype": "bf16", "batch": 64, "s1": 1, "heads": 16, "d": 512,
         "page": 64, "groups": 1, "alone": 0, "empty": 0, "prefix_lo": 32811, "prefix_hi": 32811, "own_lo": 17,
         "own_hi": 2048, "mode": 0},
        # a mixed batch: groups of several sizes over system prompts, rows of their own, idle slots, small pages
        {"name": "shared_groups", "op": "attention", "dtype": "fp16", "batch": 93, "s1": 1, "heads": 20, "d": 512,
         "page": 16, "groups": 5, "alone": 9, "empty": 3, "prefix_lo": 700, "prefix_hi": 16384, "own_lo": 1,
         "own_hi": 1500, "mode": 0},
        # two tokens a step (one drafted ahead), causal between them, more heads, a narrower latent
        {"name": "shared_drafted", "op": "attention", "dtype": "bf16", "batch": 24, "s1": 2, "heads": 32, "d": 256,
         "page": 128, "groups": 2, "alone": 0, "empty": 0, "prefix_lo": 9000, "prefix_hi": 20000, "own_lo": 2,
         "own_hi": 777, "mode": 3},
        # the rotary part of a decode step's queries, positions of three axes, a view of the projection's heads
        {"name": "axes_step", "op": "axes", "dtype": "bf16", "batch": 32, "s": 1, "heads": 128, "head": 64,
         "wide": 192, "offset": 0, "sections": "8 12 12", "order": "blocks", "layout": "interleaved",
         "inverse": False, "max_positions": 65536},
        # a prompt with pictures or a film in it, S1 = 8192, 128 heads
        {"name": "axes_prompt", "op": "axes", "dtype": "bf16", "batch": 1, "s": 8192, "heads": 128, "head": 64,
         "wide": 64, "offset": 0, "sections": "8 12 12", "order": "blocks", "layout": "interleaved",
         "inverse": False, "max_positions": 16384},
        # the gradient of index queries, half of each head rotated, axes taken in turn
        {"name": "axes_index_backward", "op": "axes", "dtype": "fp16", "batch": 2, "s": 4093, "heads": 64,
         "head": 128, "wide": 128, "offset": 0, "sections": "12 10 10", "order": "cycled", "layout": "half",
         "inverse": True, "max_positions": 8192},
        # one new token for each of 32 requests: latent, rotary and index keys
        {"name": "store_step", "op": "store", "dtype": "bf16", "batch": 32, "count_lo": 1, "count_hi": 1, "d": 512,
         "page": 128, "past": 4000, "spare": 0, "index": True},
        # the packed prompts of 24 requests, the buffer a little longer than they are
        {"name": "store_prompts", "op": "store", "dtype": "bf16", "batch": 24, "count_lo": 5, "count_hi": 1200,
         "d": 512, "page": 64, "past": 777, "spare": 61, "index": True},
        # a decode step of 32 requests that share prompts
        {"name": "plan_step", "op": "plan", "batch": 32, "slots": 64, "max_blocks": 64, "page": 64, "count_lo": 1,
         "count_hi": 1, "past_lo": 200, "past_hi": 4000, "share": 0.7, "max_groups": 32, "min_prefix": 1, "spare": 0},
        # a step of many requests, prompts among them, long tables
        {"name": "plan_many", "op": "plan", "batch": 509, "slots": 1024, "max_blocks": 512, "page": 64,
         "count_lo": 1, "count_hi": 150, "past_lo": 0, "past_hi": 32000, "share": 0.8, "max_groups": 128,
         "min_prefix": 256, "spare": 100},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng: random.Random):
    op = rng.choice(["attention", "attention", "attention", "axes", "axes", "store", "plan"])
    if op == "attention":
        heads = rng.choice([1, 5, 8, 16, 16, 20, 32, 48, 64, 128])
        s1 = min(rng.choice([1, 1, 1, 2, 3]), 128 // heads)
        hi = _spread(rng, 40, 32768)
        own_hi = _spread(rng, s1, 2048)
        batch = max(2, min(_spread(rng, 2, 128), 32768000 // ((hi + own_hi) * heads * s1)))
        groups = rng.choice([1, 1, 2, 3, 5]) if batch >= 12 else 1
        alone = rng.choice([0, 0, 1, batch // 4]) if batch >= 6 else 0
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "batch": batch, "s1": s1, "heads": heads,
                "d": rng.choice([128, 256, 512, 512]), "page": rng.choice([8, 16, 32, 64, 128, 256]),
                "groups": groups, "alone": alone, "empty": rng.choice([0, 0, 1]) if batch >= 8 else 0,
                "prefix_lo": _spread(rng, 20, hi), "prefix_hi": hi, "own_lo": _spread(rng, s1, own_hi),
                "own_hi": own_hi, "mode": 3 if s1 > 1 else rng.choice([0, 3])}
    if op == "axes":
        half = rng.choice([16, 32, 32, 64])
        axes = rng.choice([2, 3, 3, 4])
        order = rng.choice(["blocks", "cycled"])
        if order == "blocks":
            cuts = sorted(rng.sample(range(1, half), axes - 1))
            sections = [b - a for a, b in zip([0] + cuts, cuts + [half])]
        else:   # an equal turn for each axis, or fewer for the later ones: the first takes what is left
            turns = [rng.randint(1, half // axes) for _ in range(axes - 1)]
            sections = [half - sum(turns)] + turns
        head = 2 * half + rng.choice([0, 0, 64, 128])
        heads = _spread(rng, 1, 128)
        batch = _spread(rng, 1, 16)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        s = max(1, min(_spread(rng, 1, 8192), (30000000 if dtype == "fp32" else 60000000) // (batch * heads * head)))
        return {"op": op, "dtype": dtype, "batch": batch, "s": s,
                "heads": heads, "head": head, "wide": head + rng.choice([0, 0, 128]),
                "offset": rng.choice([0, head - 2 * half]), "sections": " ".join(map(str, sections)), "order": order,
                "layout": rng.choice(["interleaved", "half"]), "inverse": rng.random() < 0.4,
                "max_positions": rng.choice([16384, 32768, 131072])}
    if op == "store":
        hi = _spread(rng, 1, 4096)
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "batch": max(1, min(_spread(rng, 1, 64), 16384 // hi)),
                "count_lo": _spread(rng, 1, hi), "count_hi": hi, "d": rng.choice([128, 256, 512]),
                "page": rng.choice([8, 16, 64, 128]), "past": _spread(rng, 1, 4096), "spare": rng.choice([0, 7, 100]),
                "index": rng.random() < 0.5}
    max_blocks = _spread(rng, 8, 512)
    page = rng.choice([16, 32, 64, 128])
    batch = _spread(rng, 1, 509)
    count_hi = min(_spread(rng, 1, 200), max_blocks * page // 2)
    past_hi = _spread(rng, 1, max_blocks * page - count_hi)
    return {"op": "plan", "batch": batch, "slots": batch + _spread(rng, 1, 512), "max_blocks": max_blocks,
            "page": page, "count_lo": rng.choice([1, _spread(rng, 1, count_hi)]), "count_hi": count_hi,
            "past_lo": rng.randint(0, past_hi), "past_hi": past_hi, "share": rng.choice([0.3, 0.8, 1.0]),
            "max_groups": rng.choice([batch, _spread(rng, 1, batch)]), "min_prefix": rng.choice([1, page, 5 * page]),
            "spare": rng.choice([0, 1, 64])}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _even(lo, hi, n):
    """n whole numbers evenly from hi down to lo."""
    return [hi - ((hi - lo) * i) // max(1, n - 1) for i in range(n)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows_of(case):
    """Per row of the batch: (group, or -1 for a row of its own; tokens; tokens shared), in the batch's
    order.  Groups lie one after another, of sizes 1 : 2 : 3 ..., then the rows of their own."""
    grouped, n = case["batch"] - case["alone"], case["groups"]
    weight = n * (n + 1) // 2
    sizes = [max(1, grouped * (i + 1) // weight) for i in range(n)]
    sizes[-1] += grouped - sum(sizes)
    prefixes = _even(case["prefix_lo"], case["prefix_hi"], n)
    extra = _even(case["own_lo"], case["own_hi"], case["batch"])
    extra = extra[::2] + extra[1::2]     # long and short ones in every group
    rows = []
    for i, size in enumerate(sizes):
        for j in range(size):
            idle = i < case["empty"] and j == size - 1 and size > 1
            rows.append((i, 0 if idle else prefixes[i] + extra[len(rows)], prefixes[i]))
    while len(rows) < case["batch"]:
        rows.append((-1, extra[len(rows)], 0))
    return rows, sizes, prefixes


def _shared_state(case, g, rng):
    rows, sizes, prefixes = _rows_of(case)
    page, dtype = case["page"], _TYPES[case["dtype"]]
    own_pages = [max(0, -(-n // page) - shared // page) for _, n, shared in rows]
    ids = list(range(sum(p // page for p in prefixes) + sum(own_pages) + 3))
    rng.shuffle(ids)
    total, width = len(ids), max(1, max(-(-n // page) for _, n, _ in rows))
    shared_ids = [[ids.pop() for _ in range(p // page)] for p in prefixes]
    table = []
    for (group, n, _), count in zip(rows, own_pages):
        row = list(shared_ids[group]) if n and group >= 0 else []
        row += [ids.pop() for _ in range(count)]
        table.append(row + [-1] * (width - len(row)))
    starts = [0]
    for size in sizes:
        starts.append(starts[-1] + size)
    shape = (case["batch"], case["s1"], case["heads"])
    return dict(
        query=_randn(shape + (case["d"],), dtype, g), query_rope=_randn(shape + (_ROPE,), dtype, g),
        key_cache=_randn((total, page, 1, case["d"]), dtype, g),
        key_rope_cache=_randn((total, page, 1, _ROPE), dtype, g), block_table=_i32(table),
        group_starts=_i32(starts), prefix_lengths=_i32(prefixes), lens=_i32([n for _, n, _ in rows]),
        scale=1.0 / math.sqrt(case["d"] + _ROPE))


def _sections(case):
    return [int(n) for n in case["sections"].split()]


def _frequencies(half):
    return [10000.0 ** (-i / half) for i in range(half)]


def _axis_of(sections, order):
    """The axis of each pair."""
    half, axes = sum(sections), len(sections)
    if order == "blocks":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [i % axes if i < axes * sections[i % axes] else 0 for i in range(half)]


def _media_positions(axes, s, hi, rng):
    """Positions of one sequence of s tokens on each axis: text, where all axes go on together, and
    frames of h x w places, a step of the first axis each; an axis past the third goes with the first."""
    out, at = [], rng.randrange(0, hi - s + 1)
    while len(out) < s:
        out += [(at + i,) * axes for i in range(rng.randint(1, max(1, s // 8)))]
        at = out[-1][0] + 1
        t, h, w = rng.randint(1, 4), rng.randint(2, 24), rng.randint(2, 24)
        spot = [((at + i,) + (at + j, at + k, at + i))[:axes] for i in range(t) for j in range(h) for k in range(w)]
        out += spot
        at += max(t, h, w)
    return [list(axis) for axis in zip(*out[:s])]


def _slots_for(lens, page, total, rng):
    """Pages in random order, of `total`, for sequences of `lens` tokens."""
    ids = list(range(total))
    rng.shuffle(ids)
    return [[ids.pop() for _ in range(-(-n // page))] for n in lens]


def _store_counts(case):
    return _even(case["count_lo"], case["count_hi"], case["batch"])


def _plan_state(case, rng):
    """A pool's table in which requests continue one another's first pages, and a step's requests."""
    slots, width, page, batch = case["slots"], case["max_blocks"], case["page"], case["batch"]
    rows = rng.sample(range(slots), batch)
    counts = _even(case["count_lo"], case["count_hi"], batch)
    rng.shuffle(counts)
    table, lens = [[-1] * width for _ in range(slots)], [0] * slots
    fresh, last = 0, None
    for slot, count in zip(rows, counts):
        past = rng.randint(case["past_lo"], case["past_hi"])
        n = past + count
        blocks = []
        if last is not None and rng.random() < case["share"]:
            blocks = table[last][:min(past, lens[last]) // page]
            if rng.random() < 0.3:
                blocks = blocks[:rng.randint(0, len(blocks))]
        more = -(-n // page) - len(blocks)
        blocks = blocks + list(range(fresh, fresh + more))
        fresh += more
        table[slot][:len(blocks)] = blocks
        lens[slot], last = n, slot
    shuffled = list(range(fresh))
    rng.shuffle(shuffled)
    table = [[shuffled[p] if p >= 0 else -1 for p in row] for row in table]
    return dict(block_table=_i32(table), seq_lengths=_i32(lens), rows=_i32(rows), counts=_i32(counts),
                num_tokens=sum(counts) + case["spare"])


def prepare(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    op = case["op"]
    state = {"op": op, "case": dict(case)}
    if op == "attention":
        state.update(_shared_state(case, g, rng))
    elif op == "axes":
        wide = _randn((case["batch"], case["s"], case["heads"], case["wide"]), _TYPES[case["dtype"]], g)
        axes = len(_sections(case))
        at = [_media_positions(axes, case["s"], case["max_positions"] - 4096, rng) for _ in range(case["batch"])]
        state.update(x=wide[..., case["wide"] - case["head"]:], positions=_i32(at).transpose(0, 1).contiguous(),
                     table=_axes_table(case["max_positions"], sum(_sections(case))))
    elif op == "store":
        counts = _store_counts(case)
        rng.shuffle(counts)
        past = [rng.randint(0, case["past"]) for _ in counts]
        pages = sum(-(-(case["past"] + n) // case["page"]) for n in counts)
        tables = _slots_for([a + n for a, n in zip(past, counts)], case["page"], pages, rng)
        slots = [row[p // case["page"]] * case["page"] + p % case["page"]
                 for row, a, n in zip(tables, past, counts) for p in range(a, a + n)] + [-1] * case["spare"]
        widths = [case["d"], _ROPE] + ([_INDEX] if case["index"] else [])
        dtype = _TYPES[case["dtype"]]
        state.update(tokens=[_randn((len(slots), 1, w), dtype, g) for w in widths],
                     caches=[_randn((pages, case["page"], 1, w), dtype, g) for w in widths],
                     slot_map=torch.tensor(slots, dtype=torch.int64, device="cuda"))
    else:
        state.update(_plan_state(case, rng))
    return state


def _axes_table(max_positions, half):
    if own:
        return _dsa().rotary_table(max_positions, 2 * half)
    freq = torch.tensor(_frequencies(half), dtype=torch.float64, device="cuda")
    angle = torch.arange(max_positions, device="cuda").double()[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], dim=1).float()


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    dsa, op, case = _dsa(), state["op"], state["case"]
    if op == "attention":
        return dsa.flash_attention_shared_prefix(
            state["query"], state["query_rope"], state["key_cache"], state["key_rope_cache"], state["block_table"],
            state["group_starts"], state["prefix_lengths"], actual_seq_lengths_key=state["lens"],
            scale_value=state["scale"], sparse_mode=case["mode"], return_softmax_lse=True)
    if op == "axes":
        return dsa.rotary_embedding_axes(state["x"], state["table"], state["positions"], _sections(case),
                                         layout=case["layout"], order=case["order"], offset=case["offset"],
                                         inverse=case["inverse"])
    if op == "store":
        return dsa.paged_cache_store(state["tokens"], state["caches"], state["slot_map"])
    return tuple(dsa.paged_batch_plan(state["block_table"], state["seq_lengths"], state["rows"], state["counts"],
                                      case["page"], state["num_tokens"], max_groups=case["max_groups"],
                                      min_prefix=case["min_prefix"]))


def _run_plain(state):
    return {"attention": _plain_attention, "axes": _plain_axes, "store": _plain_store,
            "plan": _plain_plan}[state["op"]](state)


def _plain_attention(state):
    q, qr, kc, krc = state["query"], state["query_rope"], state["key_cache"], state["key_rope_cache"]
    B, S1, N1, D = q.shape
    page = kc.shape[1]
    out = torch.zeros_like(q)
    top = torch.zeros((B, 1, S1, N1), dtype=torch.float32, device=q.device)
    total = torch.zeros_like(top)
    for b, n in enumerate(state["lens"].tolist()):
        if n == 0:
            continue
        ids = state["block_table"][b, :-(-n // page)].long()
        k = kc[ids].reshape(-1, D)[:n].float()
        kr = krc[ids].reshape(-1, _ROPE)[:n].float()
        for s in range(S1):
            seen = n if state["case"]["mode"] == 0 else n - S1 + s + 1
            if seen <= 0:
                continue
            score = (q[b, s].float() @ k[:seen].t() + qr[b, s].float() @ kr[:seen].t()) * state["scale"]
            m = score.max(dim=1, keepdim=True).values
            p = (score - m).exp()
            l = p.sum(dim=1, keepdim=True)
            out[b, s] = ((p @ k[:seen]) / l).to(q.dtype)
            top[b, 0, s], total[b, 0, s] = m[:, 0], l[:, 0]
    return out, top, total


def _plain_axes(state):
    case, table, x = state["case"], state["table"], state["x"]
    half = table.shape[1] // 2
    axis = torch.tensor(_axis_of(_sections(case), case["order"]), device=x.device)
    at = state["positions"].long()[axis].permute(1, 2, 0)            # [B, S, half]
    pair = torch.arange(half, device=x.device)
    cos, sin = table[at, pair][:, :, None], table[at, half + pair][:, :, None]
    if case["inverse"]:
        sin = -sin
    out = x.float().clone()
    part = out[..., case["offset"]:case["offset"] + 2 * half]
    if case["layout"] == "interleaved":
        a, b = part[..., 0::2].clone(), part[..., 1::2].clone()
        part[..., 0::2], part[..., 1::2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = part[..., :half].clone(), part[..., half:].clone()
        part[..., :half], part[..., half:] = a * cos - b * sin, a * sin + b * cos
    return out.to(x.dtype)


def _plain_store(state):
    slots = state["slot_map"]
    valid = slots >= 0
    for tokens, cache in zip(state["tokens"], state["caches"]):
        cache.view(-1, cache.shape[-1])[slots[valid]] = tokens[valid][:, 0]
    return state["caches"]


def _plain_plan(state):
    case = state["case"]
    page, T, most = case["page"], state["num_tokens"], case["max_groups"]
    dev = state["rows"].device
    lens = state["seq_lengths"][state["rows"].long()]
    counts = state["counts"]
    table = state["block_table"][state["rows"].long()].clone()
    B, width = table.shape
    block = torch.arange(width, device=dev)
    table[block * page >= lens[:, None]] = -1
    ends = counts.cumsum(0)
    token = torch.arange(T, device=dev)
    row = torch.searchsorted(ends, token, right=True)
    there = row < B
    r = row.clamp(max=B - 1)
    pos = (lens - ends)[r] + token
    pos = torch.where(there, pos, torch.zeros_like(pos))
    slot = table[r, pos // page].long() * page + pos % page
    slot = torch.where(there, slot, torch.full_like(slot, -1))
    row = torch.where(there, row, torch.full_like(row, -1))
    # pages that a row has in common with the row before it, from the first on, all of whose tokens
    # both had before this step
    starts, prefixes = torch.full((most + 1,), B, dtype=torch.int32, device=dev), torch.zeros(most, dtype=torch.int32, device=dev)
    whole = (lens - counts) // page
    same = (table[1:] == table[:-1]) & (table[1:] >= 0) & (block < torch.minimum(whole[1:], whole[:-1])[:, None])
    common = same.int().cumprod(1).sum(1) * page
    first = torch.ones(B, dtype=torch.bool, device=dev)
    first[1:] = common < max(case["min_prefix"], page)
    begin = first.nonzero()[:, 0].tolist()
    shared = common.tolist()
    for i, b in enumerate(begin[:most]):
        e = begin[i + 1] if i + 1 < len(begin) else B
        starts[i] = b
        prefixes[i] = min(shared[b:e - 1]) if e - b > 1 else 0
    if len(begin) > most:
        starts[most] = begin[most]
    return (table, lens, ends.int(), row.int(), pos.int(), slot, starts, prefixes)


# ------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op not in ("attention", "axes"):
        return None   # whole numbers and copies: no computed values
    state = prepare(case, seed)
    if op == "attention":
        return _exact_attention(case, state)
    # each pair (a, b) as a + ib, times exp(+- i angle) of its axis' position
    half, x = sum(_sections(case)), state["x"]
    freq = torch.tensor(_frequencies(half), dtype=torch.float64, device="cuda")
    at = torch.stack([state["positions"][a] for a in _axis_of(_sections(case), case["order"])], dim=-1)
    angle = at[:, :, None].double() * freq
    turn = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle)
    out = x.double().clone()
    first = torch.arange(half, device="cuda") * (2 if case["layout"] == "interleaved" else 1) + case["offset"]
    second = first + (1 if case["layout"] == "interleaved" else half)
    z = torch.complex(out[..., first], out[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_attention(case, state):
    B, S1, N1, D = state["query"].shape
    page = case["page"]
    q = torch.cat([state["query"], state["query_rope"]], dim=-1).double()
    out = torch.zeros((B, S1, N1, D), dtype=torch.float64, device="cuda")
    top = torch.zeros((B, 1, S1, N1), dtype=torch.float64, device="cuda")
    total = torch.zeros_like(top)
    for b in range(B):
        n = int(state["lens"][b])
        if n == 0:
            continue
        t = torch.arange(n, device="cuda")
        row = state["block_table"][b].long()[t // page]
        k = torch.cat([state["key_cache"][row, t % page, 0], state["key_rope_cache"][row, t % page, 0]], dim=-1).double()
        z = torch.einsum("shc,tc->sht", q[b], k) * state["scale"]
        if case["mode"] == 3:
            s = torch.arange(S1, device="cuda")
            z.masked_fill_((t[None, :] > n - S1 + s[:, None])[:, None, :], -math.inf)
        m = z.amax(dim=-1)
        some = torch.isfinite(m)
        w = (z - torch.where(some, m, torch.zeros_like(m))[..., None]).exp()
        l = w.sum(dim=-1)
        out[b] = torch.einsum("sht,tc->shc", w, k[:, :D]) / torch.where(some, l, torch.ones_like(l))[..., None]
        top[b, 0] = torch.where(some, m, torch.zeros_like(m))
        total[b, 0] = l
    return out, top, total


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    size = 4 if case.get("dtype") == "fp32" else 2
    if op == "attention":
        rows, _, prefixes = _rows_of(case)
        d, page, s1 = case["d"], case["page"], case["s1"]
        # keys of shared pages once, every row's others
        keys = sum(p // page * page for p in prefixes) + sum(max(0, n - p // page * page) for _, n, p in rows)
        pairs = sum(max(0, n if case["mode"] == 0 else n - s1 + s + 1) for _, n, _ in rows for s in range(s1))
        blocks = sum(-(-n // page) - p // page for _, n, p in rows if n) + sum(p // page for p in prefixes)
        return {"bytes": keys * (d + _ROPE) * size + len(rows) * s1 * case["heads"] * ((2 * d + _ROPE) * size + 8) + blocks * 4,
                "flops": pairs * case["heads"] * (2 * (d + _ROPE) + 2 * d)}
    if op == "axes":
        tokens, half = case["batch"] * case["s"], sum(_sections(case))
        values = tokens * case["heads"] * case["head"]
        return {"bytes": 2 * values * size + tokens * (2 * half * 4 + len(_sections(case)) * 4),
                "flops": 6 * tokens * case["heads"] * half}
    if op == "store":
        tokens = sum(_store_counts(case))
        width = case["d"] + _ROPE + (_INDEX if case["index"] else 0)
        return {"bytes": tokens * 2 * width * size + (tokens + case["spare"]) * 8, "flops": 0}
    # the requests' rows of the table are read as far as they hold pages and written whole; 16 bytes a token
    batch, mean = case["batch"], (case["past_lo"] + case["past_hi"]) // 2
    tokens = sum(_even(case["count_lo"], case["count_hi"], batch)) + case["spare"]
    return {"bytes": batch * (min(case["max_blocks"], -(-mean // case["page"])) + case["max_blocks"] + 5) * 4
            + tokens * 16 + case["max_groups"] * 8, "flops": 0}
