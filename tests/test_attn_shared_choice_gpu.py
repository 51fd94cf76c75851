"""Which prefixes flash_attention_shared_prefix shares, at its own choice (GPU).

As in test_attn_shared_pieces_gpu.py, all rows of a group but the first with keys name a page of NaN in
the prefix: a call that shares it gives the group's result, one that does not gives NaN in those rows.
"""
import importlib
import random

import pytest
import torch

import dsa_triton_ascend_b200 as dsa
from test_attn_shared_gpu import Shared
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


@pytest.mark.parametrize("rows,s1,heads,shared,gain", [
    (64, 5, 16, 8192, True), (64, 3, 32, 16384, True), (48, 4, 20, 16384, True),
    (64, 3, 32, 8192, False), (48, 4, 20, 8192, False), (32, 7, 16, 8192, False)])
def test_packed_tokens_that_take_two_multiprocessors(rows, s1, heads, shared, gain):
    """65 to 112 heads of packed tokens, D = 512, are taken by pairs of CTAs, and so are pieces: of
    64 x 5 tokens 40 pieces cost 25.2 M cycles over 8192 keys, the rows 35.6 M.  The last three lose: 162 us shared
    against 155, 124 against 122, 125 against 97."""
    c = Pieces([(shared, [random.Random(b).randint(s1, 90) for b in range(rows)])], (), heads, 512, 64, s1=s1, seed=s1)
    assert shares(c, 3) == gain


@pytest.mark.parametrize("mode", [0, 3])
def test_padding_is_no_work(mode):
    """Rows of one token each, padded to 64: eight pieces for eight tokens cost 4.7 M cycles over 8192 keys, the
    tokens by themselves 2.5 M.  Beside a row of 64 tokens (71 of them 21.8 M, 15 pieces 8.9 M) they share."""
    c = Pieces([(8192, [70, 64, 90, 66, 64, 80, 75, 64])], (), 16, 512, 64, s1=64, seed=1)
    assert not shares(c, mode, [1] * 8)
    assert shares(c, mode, [1, 1, 64, 1, 1, 1, 1, 1])
    assert shares(c, mode, [64] * 8)


def test_tokens_before_the_first_key_are_no_work():
    """As above, of rows with fewer keys than tokens: in mode 3 the last of each alone sees the prefix."""
    c = Pieces([(8192, [1] * 8)], (), 16, 512, 64, s1=64, seed=2)
    c.lens = [1] * 8                                   # (one key: less than a page, nothing to share)
    got = dsa.flash_attention_shared_prefix(c.q, c.qr, c.kc, c.krc, c.table, c.starts, c.prefixes,
                                            actual_seq_lengths_key=c.lens, scale_value=c.scale, actual_seq_lengths_query=[64] * 8,
                                            sparse_mode=3, return_softmax_lse=True)
    c.check(got, 3, [64] * 8)


@pytest.mark.parametrize("rows,heads,d,shared,gain", [
    (8, 16, 512, 8192, False), (12, 16, 512, 8192, False), (16, 16, 512, 8192, False), (16, 16, 512, 16384, True),
    (64, 16, 512, 4096, True), (64, 64, 512, 4096, False), (16, 64, 512, 32768, True), (16, 16, 256, 8192, False),
    (16, 32, 256, 32768, True), (8, 32, 128, 16384, False), (64, 32, 128, 8192, True)])
def test_wide_tables_share_where_that_gains(rows, heads, d, shared, gain):
    """Tables of 65536 tokens, so that it is the plan that decides.  Measured, shared against not: 36.4 / 24.4, 38.4 /
    36.3 (16 rows), 43 / 54, 44.5 / 54.8, 86 / 71, 101 / 115; 33 / 26, 49 / 59; 30.4 / 26, 41 / 58 us."""
    c = Pieces([(shared, [random.Random(b).randint(1, 400) for b in range(rows)])], (), heads, d, 64, seed=rows)
    c.table = torch.cat([c.table, c.table.new_full((rows, 1024 - c.table.shape[1]), -1)], 1)
    assert shares(c) == gain


@pytest.mark.parametrize("s1,heads,act_q", [(1, 16, None), (3, 16, [3, 1, 2]), (1, 128, None), (12, 8, None)])
def test_queries_of_a_call_that_shares_nothing_are_not_copied(s1, heads, act_q, monkeypatch):
    """Small tables, or more heads than a piece takes: flash_attention_paged's call, whose queries may lie as TMA
    reads them."""
    module = importlib.import_module("dsa_triton_ascend_b200.flash_attention_paged")
    c = Shared([(130, [64, 33, 7])], (), heads, 512, 64, s1=s1, seed=8)
    wide = torch.zeros(3, s1 + 2, heads + 1, 640, device="cuda", dtype=torch.bfloat16)
    q, qr = wide[:, 1:s1 + 1, 1:, :512], wide[:, 1:s1 + 1, 1:, 512:576]
    q.copy_(c.q)
    qr.copy_(c.qr)
    c.q, c.qr = q, qr
    monkeypatch.setattr(module, "_copied", lambda t: pytest.fail("copied"))
    got = c.run(3, act_q=act_q)
    same = dsa.flash_attention_paged(q, qr, c.kc, c.krc, c.table, c.lens, c.scale, act_q, 3, True)
    assert all(torch.equal(x, y) for x, y in zip(got, same))
