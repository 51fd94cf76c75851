"""Serving one DSA layer from a paged cache: prompts, forks, decode steps, upkeep of the pages.

    python examples/paged_serving.py            # on a B200

A session owns a pool of pages (latent, rotary and index keys) and the device-resident state of
its slots.  ``prompt`` grows empty slots, appends the prompts' keys (rotated on the way) and
attends causally; ``fork`` makes further slots continue a sequence; ``step`` decodes one token
per slot, over every key of the cache, or, with ``top_k``, over the keys that the lightning
indexer picks; ``free`` and ``compact`` give pages back and close up the pool.  Nothing here waits
for the GPU, so a step can be captured into a CUDA graph.

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
    session.free(i32(0, 3))
    session.compact()
    out = session.step(i32(1, 2, 4), *tokens(3, 1))
    dsa.check_device_errors()
    print("lengths", session.lengths.tolist(), "pages in use", int((session.refs > 0).sum()),
          "output", tuple(out.shape), "finite", bool(out.isfinite().all()))


if __name__ == "__main__":
    main()
