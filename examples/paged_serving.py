"""Serving one DSA layer from a paged cache: prompts, forks, decode steps, upkeep of the pages.

    python examples/paged_serving.py            # on a B200

A session owns a pool of pages (latent, rotary and index keys) and the device-resident state of
its slots.  ``prompt`` grows empty slots, appends the prompts' keys (rotated on the way) and
attends causally; ``fork`` makes further slots continue a sequence; ``step`` decodes one token
per slot, over every key of the cache, or, with ``top_k``, over the keys that the lightning
indexer picks; ``extend_packed`` takes any number of new tokens per slot, packed, with positions on
one axis or several (pictures and films), and attends with the keys that neighbouring slots share
computed once; ``free`` and ``compact`` give pages back and close up the pool.  Nothing here waits for
the GPU, so a step can be captured into a CUDA graph.

The layer's projections are left out: a caller passes what they would produce (absorbed queries,
the latent key, index queries and weights), before rotary positions.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import dsa_triton_ascend_b200 as dsa   # noqa: E402


class PagedSession:
    """Slots of sequences over a pool of pages."""

    def __init__(self, slots, num_pages, page_size=64, max_blocks=64, heads=128, d=512, max_positions=8192,
                 dtype=torch.bfloat16, device="cuda", **scaling):
        i32 = dict(dtype=torch.int32, device=device)
        pool = lambda width: torch.zeros(num_pages, page_size, 1, width, dtype=dtype, device=device)
        self.page_size, self.heads, self.d = page_size, heads, d
        self.scale = (d + 64) ** -0.5
        self.caches = [pool(d), pool(64), pool(128)]          # latent, rotary and index keys
        self.block_table = torch.full((slots, max_blocks), -1, **i32)
        self.lengths = torch.zeros(slots, **i32)
        self.refs = torch.zeros(num_pages, **i32)
        self.table = dsa.rotary_table(max_positions, 64, device=device, **scaling)

    def _append(self, rows, counts, key, key_rope, key_index):
        """Grow the slots `rows` by `counts` tokens and write their keys; returns the positions
        they start at and the slots' tables."""
        starts = self.lengths[rows]
        grow = torch.zeros_like(self.lengths).index_copy_(0, rows.long(), counts)
        self.block_table, self.lengths, self.refs = dsa.paged_cache_extend(
            self.block_table, self.lengths, self.refs, grow, self.page_size)
        table = self.block_table[rows]
        dsa.paged_cache_append([key, key_rope, key_index], self.caches, table, starts, counts=counts,
                               table=self.table, rotary=[None, ("interleaved", 0), ("half", 0)])
        return starts, table

    def prompt(self, rows, counts, query, query_rope, key, key_rope, key_index):
        """Attention of prompts [n, S, ...] (the first counts[i] tokens of each) in empty slots."""
        starts, table = self._append(rows, counts, key, key_rope, key_index)
        at = starts[:, None] + torch.arange(query.shape[1], dtype=torch.int32, device=query.device)
        query_rope = dsa.rotary_embedding(query_rope, self.table, at)
        return dsa.flash_attention_paged(query, query_rope, self.caches[0], self.caches[1], table,
                                         actual_seq_lengths_key=self.lengths[rows], scale_value=self.scale,
                                         actual_seq_lengths_query=counts, sparse_mode=3)[0]

    def step(self, rows, query, query_rope, key, key_rope, key_index, query_index=None, weights=None, top_k=None):
        """One token [n, 1, ...] for each of the slots `rows`."""
        starts, table = self._append(rows, torch.ones_like(rows, dtype=torch.int32), key, key_rope, key_index)
        at, lengths = starts[:, None], self.lengths[rows]
        query_rope = dsa.rotary_embedding(query_rope, self.table, at)
        if top_k is None:
            return dsa.flash_attention_paged(query, query_rope, self.caches[0], self.caches[1], table,
                                             actual_seq_lengths_key=lengths, scale_value=self.scale)[0]
        query_index = dsa.rotary_embedding(query_index, self.table, at, layout="half")
        picked, _ = dsa.lightning_indexer_paged(query_index, self.caches[2], weights, table,
                                                actual_seq_lengths_key=lengths, sparse_count=top_k)
        return dsa.sparse_flash_attention_triton(
            query, self.caches[0], self.caches[0], picked, self.scale, block_table=table,
            actual_seq_lengths_kv=lengths, query_rope=query_rope, key_rope=self.caches[1], layout_kv="PA_BSND")[0]

    def extend_packed(self, rows, counts, query, query_rope, key, key_rope, key_index, sections=None, axes=None):
        """``counts[i]`` [n] new tokens for slot ``rows[i]``, one slot's behind another's in
        ``key`` [T, 1, ...], ``key_rope`` and ``key_index`` (T at least their sum), with ``query`` [n, S, ...] and
        ``query_rope`` padded to S tokens a slot.  Neighbouring slots that are forks of a sequence share its
        keys.  With ``sections``, ``axes(positions)`` [A, ...] are the positions on A axes.  A slot that the pool cannot
        serve stays as it was, gives zeros and is reported."""
        before = self.lengths[rows]
        grow = torch.zeros_like(self.lengths).index_copy_(0, rows.long(), counts)
        self.block_table, self.lengths, self.refs = dsa.paged_cache_extend(
            self.block_table, self.lengths, self.refs, grow, self.page_size)
        served = torch.where(self.lengths[rows] - before == counts, rows, -1)
        plan = dsa.paged_batch_plan(self.block_table, self.lengths, served, counts, self.page_size, key.shape[0])
        turn = lambda x, at: dsa.rotary_embedding(x, self.table, at) if sections is None else \
            dsa.rotary_embedding_axes(x, self.table, axes(at), sections)
        key_index = dsa.rotary_embedding(key_index, self.table, plan.positions, layout="half")
        dsa.paged_cache_store([key, turn(key_rope, plan.positions), key_index], self.caches, plan.slot_map)
        start = plan.key_lengths - counts
        at = start[:, None] + torch.arange(query.shape[1], dtype=torch.int32, device=query.device).clamp(max=counts[:, None] - 1)
        return dsa.flash_attention_shared_prefix(
            query, turn(query_rope, at.clamp(min=0)), self.caches[0], self.caches[1], plan.block_table, plan.group_starts,
            plan.prefix_lengths, actual_seq_lengths_key=plan.key_lengths, scale_value=self.scale,
            actual_seq_lengths_query=counts, sparse_mode=3)[0]

    def fork(self, parents, children):
        self.block_table, self.lengths, self.refs = dsa.paged_cache_fork(
            self.caches, self.block_table, self.lengths, self.refs, parents, children)

    def free(self, rows):
        self.block_table, self.lengths, self.refs = dsa.paged_cache_free(
            self.block_table, self.lengths, self.refs, rows)

    def compact(self):
        self.block_table, self.refs = dsa.paged_cache_compact(self.caches, self.block_table, self.refs)


def main():
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").bfloat16()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    session = PagedSession(slots=8, num_pages=64)

    def tokens(n, s):   # query, query_rope, key, key_rope, key_index
        return [rnd(n, s, session.heads, session.d), rnd(n, s, session.heads, 64), rnd(n, s, 1, session.d),
                rnd(n, s, 1, 64), rnd(n, s, 1, 128)]

    session.prompt(i32(0, 1), i32(300, 177), *tokens(2, 300))
    session.fork(i32(0, 0, 1), i32(2, 3, 4))              # three samples more
    for _ in range(40):
        session.step(i32(0, 1, 2, 3, 4), *tokens(5, 1))
    session.step(i32(0, 2), *tokens(2, 1), query_index=rnd(2, 1, 64, 128),
                 weights=torch.rand(2, 1, 64, generator=g, device="cuda"), top_k=128)
    counts = [1, 3, 2, 1, 5]                              # rows 0, 2 and 3 share a prompt, 1 and 4 another
    packed = sum(counts)
    session.extend_packed(i32(0, 2, 3, 1, 4), i32(*counts), *tokens(5, max(counts))[:2], *[t[0] for t in tokens(1, packed)[2:]],
                          sections=(8, 12, 12), axes=lambda at: at.expand(3, *at.shape))
    session.free(i32(0, 3))
    session.compact()
    out = session.step(i32(1, 2, 4), *tokens(3, 1))
    dsa.check_device_errors()
    print("lengths", session.lengths.tolist(), "pages in use", int((session.refs > 0).sum()),
          "output", tuple(out.shape), "finite", bool(out.isfinite().all()))


if __name__ == "__main__":
    main()
