"""flash_attention_paged against attention in 64 bits (GPU).

Tolerances follow the kernel's arithmetic.  A score is a sum of D + 64 exact products held in
fp32: with ez = (D + 64) 2^-23 scale max_t |q| . |k_t| it is off by at most ez, and so is the
maximum.  A probability is then off by the factor 1 + ez (of its own score) and 1 + ez (of the
reference), 2^-20 for exp2, and u for its rounding to the key type (2^-8 bf16, 2^-11 fp16); the
sum of probabilities is not rounded to it.  So, with A = sum_t p_t |k_t| / l,
  |out - ref| <= (u + 4 ez + 2^-18) A + u |ref|,   |sum - ref| <= (2 ez + 2^-18) ref.
The sums over t themselves run in fp32 over at most 2^16 keys split into parts: another
2^-23 sqrt(2^16) of A, within the 2^-18 allowed.
"""
import math
import random

import pytest
import torch

import dsa_triton_ascend_b200 as dsa

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """A random paged cache; unused rows and pages hold NaN."""

    def __init__(self, lens, heads=16, d=512, page=64, s1=1, dtype=torch.bfloat16, seed=0, spare=2, joint=False):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rnd = lambda *shape: torch.randn(*shape, generator=g, device="cuda").to(dtype)
        B = len(lens)
        self.lens, self.page, self.scale = lens, page, 1.0 / math.sqrt(d + 64)
        self.q, self.qr = rnd(B, s1, heads, d), rnd(B, s1, heads, 64)
        need = [-(-n // page) for n in lens]
        ids = list(range(sum(need) + spare))
        random.Random(seed).shuffle(ids)
        pool = torch.full((len(ids), page, 1, d + 64), float("nan"), device="cuda", dtype=dtype)
        rows, at = [], 0
        for n, k in zip(lens, need):
            mine = ids[at:at + k]
            at += k
            for j, p in enumerate(mine):
                m = min(page, n - j * page)
                pool[p, :m] = rnd(m, 1, d + 64)
            rows.append(mine + [-1] * (max(need + [1]) - k))
        self.table = i32(rows)
        self.kc, self.krc = (pool[..., :d], pool[..., d:]) if joint else \
            (pool[..., :d].contiguous(), pool[..., d:].contiguous())

    def run(self, mode=0, act_q=None, check=True, **kw):
        got = dsa.flash_attention_paged(self.q, self.qr, self.kc, self.krc, self.table,
                                        actual_seq_lengths_key=i32(self.lens), scale_value=self.scale,
                                        actual_seq_lengths_query=act_q, sparse_mode=mode, return_softmax_lse=True, **kw)
        dsa.check_device_errors()
        if check:
            self.check(got, mode, act_q)
        return got

    def check(self, got, mode=0, act_q=None, skip=()):
        out, top, total = (t.double() for t in got)
        B, S1, N1, D = self.q.shape
        u = UNIT[self.q.dtype]
        assert got[0].dtype == self.q.dtype and top.shape == total.shape == (B, 1, S1, N1)
        for b, n in enumerate(self.lens):
            t = torch.tensor([x for x in range(n) if (b, x // self.page) not in skip], device="cuda", dtype=torch.long)
            aq = S1 if act_q is None else int(act_q[b])
            for s in range(S1):
                seen = 0 if s >= aq else n if mode == 0 else min(n, n - aq + s + 1)
                at = t[t < seen]
                if at.numel() == 0:
                    assert not out[b, s].any() and not top[b, 0, s].any() and not total[b, 0, s].any()
                    continue
                page = self.table[b].long()[at // self.page]
                k = torch.cat([self.kc[page, at % self.page, 0], self.krc[page, at % self.page, 0]], -1).double()
                q = torch.cat([self.q[b, s], self.qr[b, s]], -1).double()
                z = q @ k.t() * self.scale
                ez = (D + 64) * 2.0 ** -23 * abs(self.scale) * (q.abs() @ k.abs().t()).amax(-1, keepdim=True)
                m = z.amax(-1, keepdim=True)
                p = (z - m).exp()
                l = p.sum(-1, keepdim=True)
                ref, mag = p @ k[:, :D] / l, p @ k[:, :D].abs() / l
                bound = (u + 4 * ez + 2.0 ** -18) * mag + u * ref.abs() + 2.0 ** -24
                assert bool(((out[b, s] - ref).abs() <= bound).all()), (b, s, float(((out[b, s] - ref).abs() / bound).max()))
                assert bool(((top[b, 0, s] - m[:, 0]).abs() <= ez[:, 0] + 2.0 ** -22 * m[:, 0].abs()).all())
                assert bool(((total[b, 0, s] - l[:, 0]).abs() <= (2 * ez[:, 0] + 2.0 ** -18) * l[:, 0]).all())


@pytest.mark.parametrize("heads", [1, 5, 16, 17, 32, 40, 64, 65, 100, 128])
@pytest.mark.parametrize("d", [128, 256, 512])
def test_heads_and_widths(heads, d):
    Case([0, 1, 63, 64, 65, 127, 128, 129, 1000], heads, d, seed=heads).run()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [8, 16, 24, 40, 64, 128, 256, 1000])
def test_pages_and_types(dtype, page):
    Case([300, 7, 0, 8, 9, 1025], 20, 256, page, dtype=dtype, seed=page).run()


@pytest.mark.parametrize("heads", [16, 128])
@pytest.mark.parametrize("s1,act_q", [(2, None), (3, [3, 2, 0, 1, 3]), (5, [5, 1, 4, 5, 2])])
@pytest.mark.parametrize("mode", [0, 3])
def test_several_new_tokens(heads, s1, act_q, mode):
    Case([130, 64, 200, 1, 2], heads, 512, 16, s1=s1, seed=s1).run(mode, act_q)


@pytest.mark.parametrize("heads", [8, 32, 128])
def test_long_rows_are_split_and_joined(heads):
    Case([40001, 9000, 33], heads, 512, 128, seed=1).run()
    Case([65536], heads, 128, 64, seed=2).run()


def test_many_short_rows():
    rng = random.Random(0)
    Case([rng.randint(0, 130) for _ in range(700)], 16, 128, 16, seed=3).run()
    Case([64] * 149, 3, 256, 64, seed=4).run()


@pytest.mark.parametrize("heads,d", [(16, 512), (128, 512), (64, 128)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_running_maximum_that_grows(heads, d, dtype):
    """Later keys outweigh the earlier ones by far, so that the accumulated product is rescaled,
    at every tile and more than once; then the other way round, where it never is."""
    c = Case([1500, 700], heads, d, 64, dtype=dtype, seed=5)
    for grow in (True, False):
        for b, n in enumerate(c.lens):
            for t0 in range(0, n, 64):
                page = int(c.table[b, t0 // 64])
                f = 1.5 ** (t0 // 64 % 9) if grow else 1.5 ** (9 - t0 // 64 % 9)
                c.krc[page] = (c.krc[page].float().clamp(-2, 2) * min(f, 20.0)).to(dtype)
        c.run()


def test_few_probabilities_above_the_smallest_half():
    """65536 keys of one weight each 2^-20 of the first key's: half's smallest values."""
    c = Case([40000], 4, 128, 64, dtype=torch.float16, seed=6)
    c.q.zero_()
    c.qr.zero_()
    c.krc.zero_()
    c.qr[..., 0] = 12.0
    c.krc[int(c.table[0, 0]), 0, 0, 0] = 1.1875
    c.scale = 1.0
    c.run()


def test_negative_scale_and_equal_scores():
    c = Case([100, 3], 16, 128, 16, seed=7)
    c.scale = -0.05
    c.run()
    c.scale = 0.0
    c.run()


def test_joint_cache_and_strided_queries():
    a = Case([333, 65], 40, 512, 64, s1=2, seed=8, joint=True)
    out = a.run(3)
    b = Case([333, 65], 40, 512, 64, s1=2, seed=8)
    assert all(torch.equal(x, y) for x, y in zip(out, b.run(3)))
    for wide in (torch.empty(2, 2, 40, 640, device="cuda", dtype=torch.bfloat16),
                 torch.empty(2, 40, 2, 640, device="cuda", dtype=torch.bfloat16).transpose(1, 2),
                 torch.empty(2, 2, 40, 643, device="cuda", dtype=torch.bfloat16)):
        q, qr = wide[..., 8:520], wide[..., 521:585]   # the second base is not 16-byte aligned
        q.copy_(b.q)
        qr.copy_(b.qr)
        b.q, b.qr = q, qr
        assert all(torch.equal(x, y) for x, y in zip(out, b.run(3)))
    one = Case([70, 70, 70], 16, 256, 16, seed=9)
    one.q, one.qr = one.q[:1].expand(3, 1, 16, 256), one.qr[:1].expand(3, 1, 16, 64)   # a broadcast query
    one.run()


def test_blocks_without_a_page():
    """Negative entries inside the length hold no keys, in the middle, at the ends, everywhere."""
    c = Case([500, 300, 64, 200], 16, 256, 32, seed=10)
    skip = {(0, 3), (0, 4), (0, 15), (1, 0), (1, 1), (2, 0), (2, 1), (3, 2)}
    for b, j in skip:
        c.table[b, j] = -1
    c.check(c.run(check=False), skip=skip)


def test_a_page_past_the_pool_is_left_out_and_reported():
    c = Case([100, 100], 16, 128, 16, seed=11)
    c.table[0, 2] = c.kc.shape[0]
    got = dsa.flash_attention_paged(c.q, c.qr, c.kc, c.krc, c.table, actual_seq_lengths_key=i32(c.lens),
                                    scale_value=c.scale, return_softmax_lse=True)
    with pytest.raises(RuntimeError, match="bits 0x4"):
        dsa.check_device_errors()
    c.check(got, skip={(0, 2)})


def test_lengths_past_the_table_and_below_zero():
    c = Case([64, 40, 10], 16, 128, 16, seed=12)
    c.kc.nan_to_num_(0.5)
    c.krc.nan_to_num_(0.5)
    c.table[c.table < 0] = 0
    ask = [1 << 30, -5, 10]
    got = dsa.flash_attention_paged(c.q, c.qr, c.kc, c.krc, c.table, actual_seq_lengths_key=ask,
                                    scale_value=c.scale, return_softmax_lse=True)
    dsa.check_device_errors()
    c.lens = [64, 0, 10]
    c.check(got)
    c.lens = [64, 64, 64]
    c.check(dsa.flash_attention_paged(c.q, c.qr, c.kc, c.krc, c.table, scale_value=c.scale,
                                      return_softmax_lse=True))


def test_cache_beyond_32_bit_offsets():
    page, d = 64, 512
    pages = 34000                                   # 2.2 GB of keys, 1.1 G elements
    kc = torch.zeros(pages, page, 1, d, device="cuda", dtype=torch.bfloat16)
    krc = torch.zeros(pages, page, 1, 64, device="cuda", dtype=torch.bfloat16)
    c = Case([150], 16, d, page, seed=13)
    far = [33999, 33998, 0]
    for j, p in enumerate(far):
        kc[p], krc[p] = c.kc[int(c.table[0, j])], c.krc[int(c.table[0, j])]
    ref = c.run()
    c.kc, c.krc, c.table = kc, krc, i32([far])
    assert all(torch.equal(x, y) for x, y in zip(ref, c.run()))


def test_same_bits_every_time_and_on_another_stream():
    c = Case([5000, 12000, 1], 128, 512, 64, seed=14)
    ref = c.run()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(ref, c.run(check=False)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run(check=False)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(ref, got))


def test_captured_graph_follows_the_lengths():
    """One capture serves every step: lengths and table are read on the GPU."""
    c = Case([900, 40], 16, 512, 64, seed=15)
    lens = i32([900, 40])
    call = lambda: dsa.flash_attention_paged(c.q, c.qr, c.kc, c.krc, c.table, actual_seq_lengths_key=lens,
                                             scale_value=c.scale, return_softmax_lse=True)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for now in ([900, 40], [1, 0], [333, 39]):
        lens.copy_(i32(now))
        graph.replay()
        dsa.check_device_errors()
        c.lens = now
        c.check(got)


def test_without_statistics_and_without_rows():
    c = Case([77], 16, 128, 8, seed=16)
    out, top, total = dsa.flash_attention_paged(c.q, c.qr, c.kc, c.krc, c.table, actual_seq_lengths_key=c.lens,
                                                scale_value=c.scale)
    assert torch.equal(out, c.run()[0]) and not top.any() and not total.any()
    for q, qr, table in ((c.q[:0], c.qr[:0], c.table[:0]), (c.q[:, :0], c.qr[:, :0], c.table)):
        assert dsa.flash_attention_paged(q, qr, c.kc, c.krc, table)[0].shape == q.shape
    dsa.check_device_errors()


def test_agrees_with_the_sparse_operator_over_every_key():
    """Attention over all keys is sparse attention whose indices name every key; both round
    their probabilities to bf16 (2^-8) and their results once more."""
    c = Case([2048, 700], 128, 512, 128, seed=17)
    out, top, total = c.run()
    idx = torch.arange(2048, device="cuda", dtype=torch.int32).expand(2, 1, 1, 2048)
    ref, rt, rl = dsa.sparse_flash_attention_triton(
        c.q, c.kc, c.kc, idx, c.scale, block_table=c.table, actual_seq_lengths_kv=i32(c.lens), query_rope=c.qr,
        key_rope=c.krc, layout_kv="PA_BSND", return_softmax_lse=True)
    dsa.check_device_errors()
    assert torch.allclose(out.float(), ref.float(), rtol=2e-2, atol=2e-3)
    assert torch.allclose(top, rt, rtol=1e-4, atol=1e-5) and torch.allclose(total, rl, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("heads,s1", [(16, 2), (1, 8), (17, 3), (64, 2), (5, 7), (32, 4), (16, 9), (100, 2)])
@pytest.mark.parametrize("d", [128, 512])
@pytest.mark.parametrize("mode", [0, 3])
def test_new_tokens_that_share_their_keys(heads, s1, d, mode):
    """Tokens of a batch are taken together where their heads fit; lengths below, at and above the
    number of tokens, and long ones that are split."""
    Case([0, 1, 2, s1 - 1, s1, s1 + 1, 63, 64, 65, 129, 700, 5000], heads, d, 16, s1=s1, seed=heads + s1).run(mode)
    Case([64] * 40 + [3], heads, d, 64, s1=s1, seed=s1).run(mode)


def test_a_later_token_leaves_the_earlier_ones_alone():
    """NaN and infinite keys that only the last token sees."""
    for s1, heads in ((3, 16), (2, 128), (4, 32)):
        c = Case([200, 64, 65, s1], heads, 256, 16, s1=s1, seed=18)
        for b, n in enumerate(c.lens):
            c.kc[int(c.table[b, (n - 1) // 16]), (n - 1) % 16] = float("nan") if b % 2 else float("inf")
        got = c.run(3, check=False)
        q, qr, lens = c.q, c.qr, c.lens
        assert not got[0][:, -1].isfinite().all()
        # the tokens before it, against the same cache without that key
        c.q, c.qr, c.lens = q[:, :-1].contiguous(), qr[:, :-1].contiguous(), [n - 1 for n in lens]
        c.check([got[0][:, :-1], got[1][:, :, :-1], got[2][:, :, :-1]], 3)


def test_shared_keys_of_a_page_that_is_not_there():
    c = Case([35, 18], 16, 128, 8, s1=3, seed=19)
    c.table[0, 4], c.table[1, 2] = -1, c.kc.shape[0]      # pages of the last keys
    got = dsa.flash_attention_paged(c.q, c.qr, c.kc, c.krc, c.table, actual_seq_lengths_key=i32(c.lens),
                                    scale_value=c.scale, sparse_mode=3, return_softmax_lse=True)
    with pytest.raises(RuntimeError, match="bits 0x4"):
        dsa.check_device_errors()
    c.check(got, 3, skip={(0, 4), (1, 2)})


def test_tokens_of_strided_queries_share_their_keys():
    c = Case([333, 65], 20, 512, 64, s1=3, seed=20)
    ref = c.run(3)
    for wide in (torch.empty(2, 3, 20, 640, device="cuda", dtype=torch.bfloat16),
                 torch.empty(3, 2, 20, 640, device="cuda", dtype=torch.bfloat16).transpose(0, 1)):
        q, qr = wide[..., :512], wide[..., 576:]
        q.copy_(c.q)
        qr.copy_(c.qr)
        c.q, c.qr = q, qr
        assert all(torch.equal(x, y) for x, y in zip(ref, c.run(3)))


@pytest.mark.parametrize("heads,d", [(16, 512), (128, 512), (100, 256)])
@pytest.mark.parametrize("lens", [[100, 40], [9000, 3000]])    # whole rows, split rows
def test_nan_where_it_is_seen(heads, d, lens):
    """A NaN query makes its own head's row NaN, a NaN key its sequence's; nothing else."""
    c = Case(lens, heads, d, 64, seed=21)
    ref = c.run()
    c.q[0, 0, 3] = float("nan")
    got = c.run(check=False)
    rest = [h for h in range(heads) if h != 3]
    assert got[0][0, 0, 3].isnan().all() and got[1][0, 0, 0, 3].isnan() and got[2][0, 0, 0, 3].isnan()
    assert torch.equal(got[0][:, :, rest], ref[0][:, :, rest]) and torch.equal(got[0][1], ref[0][1])
    c.q[0, 0, 3] = 0.0
    c.krc[int(c.table[1, 0]), 5, 0, 7] = float("nan")
    got = c.run(check=False)
    assert got[0][1].isnan().all() and got[1][1].isnan().all() and got[2][1].isnan().all()
    assert torch.equal(got[0][0][:, rest], ref[0][0][:, rest]) and got[0][0].isfinite().all()


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_heads_of_a_narrow_latent(d, dtype):
    """More than 64 heads at D <= 256: lengths around tile and page ends, rows that are split, pages
    that are missing inside a row, keys that raise the running maximum, several new tokens."""
    c = Case([0, 1, 63, 64, 65, 130, 700, 20001], 100, d, 24, dtype=dtype, seed=31)
    c.run()
    c.table[6, 3] = c.table[7, 40] = -1   # the keys of those pages are not seen
    for b, n in enumerate(c.lens):
        for t0 in range(0, n, 96):
            page = int(c.table[b, t0 // 24])
            if page >= 0:
                c.krc[page] = (c.krc[page].float().clamp(-2, 2) * min(1.5 ** (t0 // 96 % 9), 20.0)).to(dtype)
    c.check(c.run(check=False), skip={(6, 3), (7, 40)})
    for s1, heads in ((2, 64), (8, 16), (3, 128)):
        Case([0, 1, s1, 64, 5000, 200], heads, d, 16, s1=s1, dtype=dtype, seed=s1).run(3)


@pytest.mark.parametrize("d,s1,heads", [(256, 2, 64), (128, 2, 64), (256, 5, 20), (128, 8, 16), (512, 4, 32)])
def test_heads_first_queries_share_their_keys(d, s1, heads):
    """Queries laid out heads-first, or as a slice of more heads, take the path that contiguous ones
    take: the same bits, where reading the keys token by token would split and round differently."""
    c = Case([3333, 900, s1, 1], heads, d, 64, s1=s1, seed=s1 + d)
    ref = c.run(3)
    q, qr = c.q, c.qr
    for view in (lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda t: torch.cat([t, t, t], 2)[:, :, heads:2 * heads]):
        c.q, c.qr = view(q), view(qr)
        assert not c.q.is_contiguous()
        assert all(torch.equal(x, y) for x, y in zip(ref, c.run(3)))


@pytest.mark.parametrize("heads", [4, 16, 64])
def test_a_score_of_minus_infinity_alone(heads):
    """A row whose only score is -inf has no weight to give and is left at zeros, whether its token
    is taken by itself or with others (whose last keys the join takes in)."""
    c = Case([1, 2], heads, 128, 16, s1=2, seed=41)
    c.qr[..., 0] = c.qr[..., 0].abs() + 1
    for b in range(2):
        c.krc[int(c.table[b, 0]), :2, 0, 0] = float("-inf")
    both = c.run(3, check=False)
    assert not any(t.any() for t in both)               # (NaN counts as any)
    q, qr = c.q, c.qr
    for s in range(2):
        c.q, c.qr, c.lens = q[:, s:s + 1].contiguous(), qr[:, s:s + 1].contiguous(), [s, 1 + s]
        assert all(torch.equal(a.flatten(), b.flatten()) for a, b in
                   zip(c.run(check=False), (both[0][:, s:s + 1], both[1][:, :, s:s + 1], both[2][:, :, s:s + 1])))
    # beside a finite score it weighs nothing
    c = Case([200, 2], heads, 128, 16, s1=2, seed=42)
    c.qr[..., 0] = c.qr[..., 0].abs() + 1
    for b, n in enumerate(c.lens):
        c.krc[int(c.table[b, (n - 1) // 16]), (n - 1) % 16, 0, 0] = float("-inf")
    got = c.run(3, check=False)
    q, qr = c.q, c.qr
    c.q, c.qr, c.lens = q[:, 1:].contiguous(), qr[:, 1:].contiguous(), [199, 1]
    c.check([got[0][:, 1:], got[1][:, :, 1:], got[2][:, :, 1:]])
