"""Serving operators around a paged latent cache: what a pass of each costs and gives.

Four operators, as a decode or prefill step calls them: attention of new tokens over a paged
key cache, rotary positions on queries and keys, the append of new tokens to the cache's
pages, and the upkeep of those pages (fork, compact, free).  ``run`` computes a pass with
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
        # one sequence of a chat, few heads left on this GPU by head sharding: latency
        {"name": "attention_single", "op": "attention", "dtype": "bf16", "batch": 1, "s1": 1, "heads": 16,
         "d": 512, "page": 64, "len_lo": 1021, "len_hi": 1021, "empty": 0, "mode": 0},
        # a batch of long sequences with every head: 32 x (8192 .. 65536) keys, pages of 128
        {"name": "attention_long", "op": "attention", "dtype": "bf16", "batch": 32, "s1": 1, "heads": 128,
         "d": 512, "page": 128, "len_lo": 8192, "len_hi": 65536, "empty": 0, "mode": 0},
        # a ragged batch with few heads, idle slots among the rows, small pages
        {"name": "attention_ragged", "op": "attention", "dtype": "fp16", "batch": 67, "s1": 1, "heads": 16,
         "d": 512, "page": 16, "len_lo": 1, "len_hi": 16411, "empty": 3, "mode": 0},
        # two tokens a step (one drafted ahead), causal between them, a narrower latent
        {"name": "attention_drafted", "op": "attention", "dtype": "bf16", "batch": 8, "s1": 2, "heads": 64,
         "d": 256, "page": 64, "len_lo": 4000, "len_hi": 32768, "empty": 0, "mode": 3},
        # the rotary part of a decode step's queries, a view of the projection's heads
        {"name": "rotary_step", "op": "rotary", "dtype": "bf16", "batch": 32, "s": 1, "heads": 128, "head": 64,
         "wide": 192, "offset": 0, "dim": 64, "layout": "interleaved", "inverse": False, "max_positions": 65536,
         "scaling": "yarn"},
        # the rotary part of a prefill's queries, S1 = 8192, 128 heads
        {"name": "rotary_prefill", "op": "rotary", "dtype": "bf16", "batch": 1, "s": 8192, "heads": 128, "head": 64,
         "wide": 64, "offset": 0, "dim": 64, "layout": "interleaved", "inverse": False, "max_positions": 16384,
         "scaling": "none"},
        # the gradient of the index queries: 64 heads of 128, of which the first half is rotated
        {"name": "rotary_index_backward", "op": "rotary", "dtype": "bf16", "batch": 2, "s": 4093, "heads": 64,
         "head": 128, "wide": 128, "offset": 0, "dim": 64, "layout": "half", "inverse": True,
         "max_positions": 8192, "scaling": "linear"},
        # one new token for each of 32 sequences: latent, rotary and index keys
        {"name": "append_step", "op": "append", "dtype": "bf16", "batch": 32, "s": 1, "d": 512, "page": 128,
         "start_lo": 100, "start_hi": 4000, "index": True},
        # two prompts of up to 4096 tokens, the second shorter
        {"name": "append_prompt", "op": "append", "dtype": "bf16", "batch": 2, "s": 4096, "d": 512, "page": 64,
         "start_lo": 0, "start_hi": 777, "index": True},
        # 16 sequences forked for sampling: shared full pages, a copy of each last page in 4 layers
        {"name": "pages_fork", "op": "fork", "dtype": "bf16", "slots": 256, "max_blocks": 128, "pages": 2048,
         "page": 64, "layers": 4, "n": 16, "len_lo": 65, "len_hi": 4000, "live": 0.5},
        # a pool of which most is free, closed up: several hundred pages move
        {"name": "pages_compact", "op": "compact", "dtype": "bf16", "slots": 256, "max_blocks": 128, "pages": 4096,
         "page": 128, "layers": 1, "n": 0, "len_lo": 1, "len_hi": 2048, "live": 0.5},
        # 100 finished sequences give their pages back, some of them shared
        {"name": "pages_free", "op": "free", "dtype": "bf16", "slots": 512, "max_blocks": 512, "pages": 65536,
         "page": 64, "layers": 0, "n": 100, "len_lo": 1, "len_hi": 16384, "live": 0.9},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], evenly in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng: random.Random):
    op = rng.choice(["attention", "attention", "attention", "rotary", "append", "fork", "compact", "free"])
    if op == "attention":
        hi = _spread(rng, 1, 65536)
        batch = max(1, min(_spread(rng, 1, 96), 1000000 // hi))
        heads = rng.choice([1, 5, 8, 16, 20, 32, 48, 64, 96, 128])
        s1 = min(rng.choice([1, 1, 1, 2, 3]), 128 // heads)
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "batch": batch, "s1": s1, "heads": heads,
                "d": rng.choice([128, 256, 512, 512]), "page": rng.choice([8, 16, 32, 64, 128, 256]),
                "len_lo": _spread(rng, 1, hi), "len_hi": hi, "empty": rng.choice([0, 0, 1, 2]) if batch > 2 else 0,
                "mode": 3 if s1 > 1 else rng.choice([0, 3])}
    if op == "rotary":
        dim = rng.choice([32, 64, 64, 128])
        head = dim + rng.choice([0, 0, 64, 128])
        heads = _spread(rng, 1, 128)
        batch = _spread(rng, 1, 16)
        s = max(1, min(_spread(rng, 1, 8192), 67108864 // (batch * heads * head)))
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "batch": batch, "s": s,
                "heads": heads, "head": head, "wide": head + rng.choice([0, 0, 128]),
                "offset": rng.choice([0, head - dim]), "dim": dim, "layout": rng.choice(["interleaved", "half"]),
                "inverse": rng.random() < 0.4, "max_positions": rng.choice([8192, 32768, 131072]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"])}
    if op == "append":
        s = _spread(rng, 1, 4096)
        batch = max(1, min(_spread(rng, 1, 64), 8192 // s))
        hi = _spread(rng, 1, 4096)
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "batch": batch, "s": s,
                "d": rng.choice([128, 256, 512]), "page": rng.choice([8, 16, 64, 128]),
                "start_lo": rng.randrange(0, hi + 1), "start_hi": hi, "index": rng.random() < 0.5}
    slots = _spread(rng, 8, 512)
    page = rng.choice([16, 32, 64, 128])
    max_blocks = _spread(rng, 8, 256)
    hi = _spread(rng, 1, max_blocks * page)
    return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "slots": slots, "max_blocks": max_blocks,
            "pages": _spread(rng, 512, 4096), "page": page,
            "layers": 0 if op == "free" else 1 if page * 4 > 256 else rng.choice([1, 2, 3]),
            "n": 0 if op == "compact" else _spread(rng, 1, slots // 2), "len_lo": _spread(rng, 1, hi), "len_hi": hi,
            "live": rng.choice([0.2, 0.5, 0.8])}


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------

def _even(lo, hi, n):
    """n whole numbers evenly from hi down to lo."""
    return [hi - ((hi - lo) * i) // max(1, n - 1) for i in range(n)]


def _lengths(case):
    n = case["batch"] - case["empty"]
    return _even(case["len_lo"], case["len_hi"], n) + [0] * case["empty"]


def _starts(case):
    return _even(case["start_lo"], case["start_hi"], case["batch"])


def _counts(case):
    """New tokens of each sequence: all of them for a step, ragged for prompts."""
    s = case["s"]
    return [s if s < 4 else s - (s * 3 // 8) * b // case["batch"] for b in range(case["batch"])]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(shape, dtype, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _table_of(lens, page, blocks, rng):
    """Pages in random order for sequences of `lens` tokens: (table [n, max_blocks], pages in all)."""
    need = [-(-n // page) for n in lens]
    total = max(1, sum(need)) + blocks
    ids = list(range(total))
    rng.shuffle(ids)
    width = max(1, max(need))
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return _i32(table), total


_YARN = {"factor": 16.0, "original": 4096, "beta_fast": 32.0, "beta_slow": 1.0}


def _scaling(case):
    """The long-context scaling of a case, as keyword arguments of ``rotary_table``."""
    kind = case["scaling"]
    if kind == "none":
        return {}
    if kind == "yarn":
        return {"scaling": "yarn", "factor": _YARN["factor"], "original_positions": _YARN["original"],
                "beta_fast": _YARN["beta_fast"], "beta_slow": _YARN["beta_slow"],
                "amplitude": 0.1 * math.log(_YARN["factor"]) + 1.0}
    return {"scaling": kind, "factor": 8.0}


def _frequencies(dim, kind, base=10000.0):
    """Angle per position of each rotated pair, and the amplitude, in Python numbers."""
    half = dim // 2
    if kind == "ntk":
        base = base * 8.0 ** (dim / (dim - 2))
    freq = [base ** (-2.0 * i / dim) for i in range(half)]
    if kind == "linear":
        freq = [f / 8.0 for f in freq]
    if kind != "yarn":
        return freq, 1.0
    turn = lambda beta: dim * math.log(_YARN["original"] / (beta * 2.0 * math.pi)) / (2.0 * math.log(base))
    low = max(0, math.floor(turn(_YARN["beta_fast"])))
    high = min(dim - 1, math.ceil(turn(_YARN["beta_slow"])))
    out = []
    for i, f in enumerate(freq):
        ramp = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
        out.append(f / _YARN["factor"] * ramp + f * (1.0 - ramp))
    return out, 0.1 * math.log(_YARN["factor"]) + 1.0


def _cos_sin(positions, dim, kind):
    """Cosines and sines of `positions` in 64 bits: two [n, dim / 2] tensors."""
    freq, amplitude = _frequencies(dim, kind)
    angle = positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=positions.device)
    return angle.cos() * amplitude, angle.sin() * amplitude


def _rotary_table(max_positions, dim, case):
    if own:
        return _dsa().rotary_table(max_positions, dim, **_scaling(case))
    cos, sin = _cos_sin(torch.arange(max_positions, device="cuda"), dim, case["scaling"])
    return torch.cat([cos, sin], dim=1).float()


def _pool_state(case, seed, g):
    """A pool in use: sequences in some of the slots, some sharing their first pages."""
    rng = random.Random(seed)
    page, pages, slots, width = case["page"], case["pages"], case["slots"], case["max_blocks"]
    budget = int(pages * case["live"])
    ids = list(range(pages))
    rng.shuffle(ids)
    table = [[-1] * width for _ in range(slots)]
    lens, refs, used = [0] * slots, [0] * pages, []
    order = list(range(slots))
    rng.shuffle(order)
    # half of the slots at most are in use, so that forks find empty ones
    for slot in order[:max(1, slots // 2)]:
        n = rng.randint(case["len_lo"], case["len_hi"])
        need = -(-n // page)
        shared = []
        if used and rng.random() < 0.3:   # the full pages at the front of an older sequence
            other = rng.choice(used)
            shared = table[other][:min(lens[other], n) // page]
            shared = shared[:rng.randint(0, len(shared))]
        if need - len(shared) > budget:
            continue
        fresh = [ids.pop() for _ in range(need - len(shared))]
        budget -= len(fresh)
        row = shared + fresh
        for p in row:
            refs[p] += 1
        table[slot][:need] = row
        lens[slot] = n
        used.append(slot)
    if not used:   # a pool too small for one such sequence holds one page of it
        p = ids.pop()
        table[order[0]][0], lens[order[0]], refs[p] = p, min(page, case["len_lo"]), 1
        used.append(order[0])
    idle = [s for s in order if lens[s] == 0]
    dtype = _TYPES[case["dtype"]]
    caches = []
    for _ in range(case["layers"]):
        caches.append(_randn((pages, page, 1, 512), dtype, g))
        caches.append(_randn((pages, page, 1, _ROPE), dtype, g))
    state = {"block_table": _i32(table), "seq_lengths": _i32(lens), "ref_counts": _i32(refs), "caches": caches,
             "page": page}
    if case["op"] == "fork":
        n = min(case["n"], len(idle), sum(1 for r in refs if r == 0))
        state["parents"] = _i32([rng.choice(used) for _ in range(n)])
        state["children"] = _i32(idle[:n])
    if case["op"] == "free":
        state["rows"] = _i32(rng.sample(used, min(case["n"], len(used))))
    return state


def prepare(case, seed):
    g = _gen(seed)
    rng = random.Random(seed)
    dtype = _TYPES[case["dtype"]]
    op = case["op"]
    state = {"op": op, "case": dict(case)}
    if op == "attention":
        lens = _lengths(case)
        rng.shuffle(lens)
        table, pages = _table_of(lens, case["page"], 3, rng)
        shape = (case["batch"], case["s1"], case["heads"])
        state.update(
            query=_randn(shape + (case["d"],), dtype, g), query_rope=_randn(shape + (_ROPE,), dtype, g),
            key_cache=_randn((pages, case["page"], 1, case["d"]), dtype, g),
            key_rope_cache=_randn((pages, case["page"], 1, _ROPE), dtype, g),
            block_table=table, lens=_i32(lens), scale=1.0 / math.sqrt(case["d"] + _ROPE))
    elif op == "rotary":
        shape = (case["batch"], case["s"], case["heads"], case["wide"])
        wide = _randn(shape, dtype, g)
        first = case["wide"] - case["head"]
        if case["s"] == 1:   # a decode step: each sequence at its own place
            at = torch.randint(0, case["max_positions"], (case["batch"], 1), generator=g, device="cuda")
        else:
            at = torch.randint(0, case["max_positions"] - case["s"] + 1, (case["batch"], 1), generator=g, device="cuda") \
                + torch.arange(case["s"], device="cuda")
        state.update(x=wide[..., first:], positions=at.to(torch.int32),
                     table=_rotary_table(case["max_positions"], case["dim"], case))
    elif op == "append":
        starts, counts = _starts(case), _counts(case)
        rng.shuffle(starts)
        table, pages = _table_of([a + n for a, n in zip(starts, counts)], case["page"], 3, rng)
        widths = [case["d"], _ROPE] + ([_INDEX] if case["index"] else [])
        shape = (case["batch"], case["s"], 1)
        state.update(
            tokens=[_randn(shape + (w,), dtype, g) for w in widths],
            caches=[_randn((pages, case["page"], 1, w), dtype, g) for w in widths],
            rotary=[None, ("interleaved", 0)] + ([("half", 0)] if case["index"] else []),
            block_table=table, starts=_i32(starts), counts=_i32(counts),
            table=_rotary_table(16384, _ROPE, {"scaling": "none"}))
    else:
        state.update(_pool_state(case, seed, g))
    return state


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    dsa, op = _dsa(), state["op"]
    if op == "attention":
        return dsa.flash_attention_paged(
            state["query"], state["query_rope"], state["key_cache"], state["key_rope_cache"], state["block_table"],
            actual_seq_lengths_key=state["lens"], scale_value=state["scale"], sparse_mode=state["case"]["mode"],
            return_softmax_lse=True)
    if op == "rotary":
        case = state["case"]
        return dsa.rotary_embedding(state["x"], state["table"], state["positions"], layout=case["layout"],
                                    offset=case["offset"], inverse=case["inverse"])
    if op == "append":
        return dsa.paged_cache_append(state["tokens"], state["caches"], state["block_table"], state["starts"],
                                      counts=state["counts"], table=state["table"], rotary=state["rotary"])
    if op == "fork":
        table, lens, refs = dsa.paged_cache_fork(state["caches"], state["block_table"], state["seq_lengths"],
                                                 state["ref_counts"], state["parents"], state["children"],
                                                 page_size=state["page"])
        return [table, lens, refs] + state["caches"]
    if op == "compact":
        table, refs = dsa.paged_cache_compact(state["caches"], state["block_table"], state["ref_counts"])
        return [table, refs] + state["caches"]
    return dsa.paged_cache_free(state["block_table"], state["seq_lengths"], state["ref_counts"], state["rows"])


def _run_plain(state):
    return {"attention": _plain_attention, "rotary": _plain_rotary, "append": _plain_append, "fork": _plain_fork,
            "compact": _plain_compact, "free": _plain_free}[state["op"]](state)


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


def _rotate(x, cos, sin, layout, offset, inverse):
    """x [..., heads, head]; cos, sin [..., 1, dim / 2]."""
    dim = 2 * cos.shape[-1]
    out = x.float().clone()
    part = out[..., offset:offset + dim]
    if layout == "interleaved":
        a, b = part[..., 0::2].clone(), part[..., 1::2].clone()
    else:
        a, b = part[..., :dim // 2].clone(), part[..., dim // 2:].clone()
    if inverse:
        sin = -sin
    ra, rb = a * cos - b * sin, a * sin + b * cos
    if layout == "interleaved":
        part[..., 0::2], part[..., 1::2] = ra, rb
    else:
        part[..., :dim // 2], part[..., dim // 2:] = ra, rb
    return out.to(x.dtype)


def _plain_rotary(state):
    case, table = state["case"], state["table"]
    row = table[state["positions"].long()][:, :, None, :]
    half = table.shape[1] // 2
    return _rotate(state["x"], row[..., :half], row[..., half:], case["layout"], case["offset"], case["inverse"])


def _plain_append(state):
    table, page = state["block_table"], state["caches"][0].shape[1]
    S = state["tokens"][0].shape[1]
    step = torch.arange(S, device=table.device)
    at = state["starts"].long()[:, None] + step
    valid = step < state["counts"].long()[:, None]
    block = table.long().gather(1, (at // page).clamp(max=table.shape[1] - 1))
    where = (block * page + at % page)[valid]
    angle = state["table"][at.clamp(max=state["table"].shape[0] - 1)][:, :, None, :]
    half = angle.shape[-1] // 2
    for tokens, cache, how in zip(state["tokens"], state["caches"], state["rotary"]):
        if how is not None:
            tokens = _rotate(tokens, angle[..., :half], angle[..., half:], how[0], how[1], False)
        cache.view(-1, cache.shape[-1])[where] = tokens[valid][:, 0]
    return state["caches"]


def _plain_fork(state):
    page = state["page"]
    table, lens, refs = state["block_table"].clone(), state["seq_lengths"].clone(), state["ref_counts"].clone()
    free = (state["ref_counts"] == 0).nonzero()[:, 0].tolist()
    taken = 0
    old = lens.tolist()
    for parent, child in zip(state["parents"].tolist(), state["children"].tolist()):
        n = old[parent]
        full, rest = n // page, n % page
        table[child] = -1
        table[child, :full] = table[parent, :full]
        refs.index_add_(0, table[parent, :full].long(), torch.ones(full, dtype=torch.int32, device=refs.device))
        if rest:
            p = free[taken]
            taken += 1
            src = int(table[parent, full])
            for cache in state["caches"]:
                cache[p, :rest] = cache[src, :rest]
            table[child, full] = p
            refs[p] = 1
        lens[child] = n
    return [table, lens, refs] + state["caches"]


def _plain_compact(state):
    refs, table = state["ref_counts"], state["block_table"]
    live = refs > 0
    n = int(live.sum())
    ids = torch.arange(refs.numel(), device=refs.device)
    movers, holes = ids[live & (ids >= n)], ids[~live & (ids < n)]
    where = ids.clone()
    where[movers] = holes
    out = refs.clone()
    out[holes] = refs[movers]
    out[movers] = 0
    new = torch.where(table >= 0, where[table.clamp(min=0).long()].to(torch.int32), table)
    for cache in state["caches"]:
        cache[holes] = cache[movers]
    return [new, out] + state["caches"]


def _plain_free(state):
    table, lens, refs = state["block_table"].clone(), state["seq_lengths"].clone(), state["ref_counts"].clone()
    rows = state["rows"].long()
    held = table[rows]
    held = held[held >= 0].long()
    refs.index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    table[rows] = -1
    lens[rows] = 0
    return table, lens, refs


# ------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------

def exact(case, seed):
    op = case["op"]
    if op not in ("attention", "rotary", "append"):
        return None   # whole numbers and copies: no computed values
    state = prepare(case, seed)
    if op == "attention":
        return _exact_attention(case, state)
    if op == "rotary":
        return _exact_rotated(state["x"], state["positions"].long(), case["dim"], case["scaling"], case["layout"],
                              case["offset"], case["inverse"])
    caches = [c.double() for c in state["caches"]]
    page = case["page"]
    starts, counts = state["starts"].tolist(), state["counts"].tolist()
    for i, how in enumerate(state["rotary"]):
        for b, (start, count) in enumerate(zip(starts, counts)):
            at = torch.arange(start, start + count, device="cuda")
            rows = state["tokens"][i][b:b + 1, :count]
            rows = rows.double() if how is None else _exact_rotated(rows, at[None], _ROPE, "none", how[0], how[1], False)
            caches[i][state["block_table"][b].long()[at // page], at % page] = rows[0]
    return caches


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


def _exact_rotated(x, at, dim, scaling, layout, offset, inverse):
    """Each pair (a, b) as a + ib, times the amplitude and exp(+- i angle)."""
    freq, amplitude = _frequencies(dim, scaling)
    angle = at.double()[..., None, None] * torch.tensor(freq, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, amplitude), -angle if inverse else angle)
    out = x.double().clone()
    first = torch.arange(dim // 2, device="cuda") * (2 if layout == "interleaved" else 1) + offset
    second = first + (1 if layout == "interleaved" else dim // 2)
    z = torch.complex(out[..., first], out[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "attention":
        d, rows = case["d"], case["batch"] * case["s1"] * case["heads"]
        keys = sum(_lengths(case))
        pairs = sum(max(0, n if case["mode"] == 0 else n - case["s1"] + s + 1)
                    for n in _lengths(case) for s in range(case["s1"]))
        blocks = sum(-(-n // case["page"]) for n in _lengths(case))
        return {"bytes": keys * (d + _ROPE) * size + rows * ((2 * d + _ROPE) * size + 8) + blocks * 4,
                "flops": pairs * case["heads"] * (2 * (d + _ROPE) + 2 * d)}
    if op == "rotary":
        tokens = case["batch"] * case["s"]
        values = tokens * case["heads"] * case["head"]
        return {"bytes": 2 * values * size + tokens * (case["dim"] * 4 + 4),
                "flops": 3 * tokens * case["heads"] * case["dim"]}
    if op == "append":
        tokens = sum(_counts(case))
        width = case["d"] + _ROPE + (_INDEX if case["index"] else 0)
        return {"bytes": tokens * (2 * width * size + _ROPE * 4 + 4),
                "flops": tokens * 3 * _ROPE * (2 if case["index"] else 1)}
    # the pool's bookkeeping is read and written once; the pages that move, by the sizes that
    # the case draws its sequences from
    keep = 2 * 4 * (case["slots"] * case["max_blocks"] + case["pages"])
    row = (512 + _ROPE) * size * case["layers"]
    if op == "free":
        return {"bytes": keep + 8 * case["slots"], "flops": 0}
    if op == "fork":
        return {"bytes": keep + 8 * case["slots"] + 2 * case["n"] * (case["page"] // 2) * row, "flops": 0}
    mean = -(-(case["len_lo"] + case["len_hi"]) // (2 * case["page"]))
    live = min(case["pages"] * case["live"], mean * max(1, case["slots"] // 2))
    return {"bytes": keep + 2 * int(live * (1.0 - live / case["pages"])) * case["page"] * row, "flops": 0}
