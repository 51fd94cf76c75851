"""Which prefixes flash_attention_shared_prefix shares, at its own choice (GPU).

As in test_attn_shared_pieces_gpu.py, all rows of a group but the first with keys name a page of NaN in
the prefix: a call that shares it gives the group's result, one that does not gives NaN in those rows.
"""
import random

import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from test_attn_shared_pieces_gpu import Pieces

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def give_memory_back():
    """Large blocks that stay in torch's cache would serve a later test that counts on its being empty."""
    yield
    torch.cuda.empty_cache()


def shares(c, mode=0, act_q=None):
    got = c.run(mode, act_q, check=False)
    dsa.check_device_errors()
    last = c.q.shape[0] - 1                            # (the last row is one of a group, with keys)
    if bool(got[0][last].isnan().any()):
        return False
    assert bool(got[0].isfinite().all())
    c.check(got, mode, act_q)
    return True


@pytest.mark.parametrize("rows,s1,heads,gain", [(64, 5, 16, True), (64, 3, 32, True), (48, 4, 20, True), (32, 7, 16, False)])
def test_packed_tokens_that_take_two_multiprocessors(rows, s1, heads, gain):
    """65 to 112 heads of packed tokens, D = 512, are taken by pairs of CTAs, and so are pieces: of
    64 x 5 tokens 40 pieces cost 23.6 M cycles over 8192 keys, the rows 35.6 M; of 32 x 7 tokens 28 pieces
    16.5 M, the rows 17.8 M, which is less of a difference than a launch more takes."""
    c = Pieces([(8192, [random.Random(b).randint(s1, 90) for b in range(rows)])], (), heads, 512, 64, s1=s1, seed=s1)
    assert shares(c, 3) == gain
