"""rotary_embedding_axes against the rotation in 64 bits, and its gradient (GPU).

The tolerance is that of rotary_embedding (test_rotary_gpu.py): two fp32 products of table entries rounded
once, 2^-22 (|a| + |b|), and one rounding of the result, u of it; copied values are exact.
"""
import pytest
import torch

import dsa_triton_ascend_b200 as dsa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, scope="module")
def give_memory_back():
    """Large blocks that stay in torch's cache would serve a later test that counts on its being empty."""
    yield
    torch.cuda.empty_cache()

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _axes(sections, order):
    """Axis of each pair, by hand."""
    if order == "blocks":
        return sum(([a] * n for a, n in enumerate(sections)), [])
    left, out = list(sections), []
    for i in range(sum(sections)):
        a = i % len(sections)
        if a and not left[a]:
            a = 0
        left[a] -= 1
        out.append(a)
    assert not any(left[1:])
    return out


def _expect(x, positions, axis_of, layout, offset, inverse, freq=None):
    half = len(axis_of)
    freq = torch.tensor(freq or dsa.rotary_frequencies(2 * half), dtype=torch.float64, device="cuda")
    ang = positions.double()[axis_of].movedim(0, -1).unsqueeze(-2) * freq
    c, s = ang.cos(), ang.sin() * (-1 if inverse else 1)
    i = torch.arange(half, device="cuda")
    ia = offset + (2 * i if layout == "interleaved" else i)
    ib = ia + (1 if layout == "interleaved" else half)
    ref = x.double().clone()
    a, b = x.double()[..., ia], x.double()[..., ib]
    ref[..., ia], ref[..., ib] = a * c - b * s, a * s + b * c
    bound = torch.zeros_like(ref)
    for at in (ia, ib):
        bound[..., at] = 2.0 ** -22 * (a.abs() + b.abs()) + UNIT[x.dtype] * ref[..., at].abs()
        if x.dtype == torch.float16:
            bound[..., at] += 2.0 ** -25   # half a step among the subnormal values
    return ref, bound


def _check(x, positions, sections, layout="interleaved", order="blocks", offset=0, inverse=False, out=None):
    table = dsa.rotary_table(max(1, int(positions.max()) + 1 if positions.numel() else 1), 2 * sum(sections))
    ref, bound = _expect(x, positions, _axes(sections, order), layout, offset, inverse)
    for _ in range(2):   # a new signature, and the same again
        got = dsa.rotary_embedding_axes(x, table, positions, sections, layout=layout, order=order, offset=offset,
                                        inverse=inverse, out=out)
        dsa.check_device_errors()
        assert got.shape == x.shape and got.dtype == x.dtype
        assert bool(((got.double() - ref).abs() <= bound).all())
        if out is x:
            break
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("sections,order", [
    ([8, 12, 12], "blocks"), ([12, 10, 10], "cycled"), ([32], "blocks"), ([32], "cycled"), ([16, 16], "cycled"),
    ([1, 30, 1], "blocks"), ([29, 1, 2], "cycled"), ([8, 8, 8, 8], "blocks"), ([8, 8, 8, 8], "cycled"),
    ([3, 5, 7, 17], "blocks"), ([20, 4, 3, 5], "cycled")])
@pytest.mark.parametrize("B,S,N,H,offset", [(2, 5, 128, 64, 0), (3, 7, 5, 192, 128), (1, 33, 64, 128, 0), (2, 3, 6, 70, 5)])
def test_rotation(dtype, layout, sections, order, B, S, N, H, offset):
    g = _gen(B * 1000 + S * 10 + H)
    x = torch.randn(B, S, N, H, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 5000, (len(sections), B, S), generator=g, device="cuda", dtype=torch.int32)
    _check(x, pos, sections, layout, order, offset, inverse=bool(S & 1))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("sections,order,H,offset", [([1], "blocks", 2, 0), ([2, 1], "cycled", 6, 0), ([64, 32, 32], "blocks", 256, 0),
                                                     ([44, 42, 42], "cycled", 300, 44), ([5, 3], "blocks", 17, 1)])
def test_widths(layout, sections, order, H, offset):
    """From one pair to the widest head; heads that are no whole 16-byte pieces."""
    g = _gen(H)
    for dtype in UNIT:
        x = torch.randn(2, 9, 3, H, generator=g, device="cuda").to(dtype)
        pos = torch.randint(0, 70000, (len(sections), 2, 9), generator=g, device="cuda", dtype=torch.int32)
        _check(x, pos, sections, layout, order, offset)


@pytest.mark.parametrize("order", ["blocks", "cycled"])
def test_text_turns_as_on_one_axis(order):
    g = _gen(1)
    x = torch.randn(2, 40, 8, 64, generator=g, device="cuda").bfloat16()
    pos = torch.randint(0, 900, (2, 40), generator=g, device="cuda", dtype=torch.int32)
    table = dsa.rotary_table(900, 64)
    for layout in ("interleaved", "half"):
        one = dsa.rotary_embedding(x, table, pos, layout=layout)
        for sections in ([11, 11, 10], [16, 16]):
            got = dsa.rotary_embedding_axes(x, table, pos.expand(len(sections), 2, 40), sections, layout=layout, order=order)
            assert torch.equal(got, one)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_strided_views_tokens_first_and_in_place(layout):
    g = _gen(11)
    wide = torch.randn(2, 9, 6, 192, generator=g, device="cuda").bfloat16()
    pos = torch.randint(0, 99, (3, 2, 9), generator=g, device="cuda")          # int64
    a = _check(wide[..., 128:], pos, [8, 12, 12], layout)
    _check(wide.transpose(1, 2).contiguous().transpose(1, 2)[..., 128:], pos, [8, 12, 12], layout)
    _check(wide[:, ::2, 1::2, 3:73], pos[:, :, ::2], [8, 12, 12], layout, "blocks", 5)    # no aligned base
    _check(wide.transpose(2, 3)[..., :64, :].transpose(2, 3)[:, :, :, ::2], pos, [4, 4, 8], layout)   # no contiguous last dim
    got = _check(wide.reshape(18, 6, 192)[..., 128:], pos.reshape(3, 18), [8, 12, 12], layout)
    assert torch.equal(got, a.reshape(18, 6, 64))
    into = torch.zeros(2, 9, 6, 100, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(_check(wide[..., 128:], pos, [8, 12, 12], layout, out=into[..., 4:68]), a)
    assert not into[..., :4].any() and not into[..., 68:].any()
    mine = wide.clone()[..., 128:]
    assert _check(mine, pos, [8, 12, 12], layout, out=mine) is mine and torch.equal(mine, a)
    with pytest.raises(ValueError, match="overlaps"):
        dsa.rotary_embedding_axes(mine, dsa.rotary_table(99, 64), pos, [8, 12, 12], layout=layout, out=wide.clone()[..., :64].set_(
            mine.untyped_storage(), 64, mine.shape, mine.stride()))


def test_without_tokens():
    table = dsa.rotary_table(9, 64)
    for shape in ((0, 3, 4, 64), (2, 0, 4, 64), (2, 3, 0, 64)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        assert dsa.rotary_embedding_axes(x, table, torch.zeros(3, *shape[:2], device="cuda", dtype=torch.int32), [8, 12, 12]).shape == shape


@pytest.mark.parametrize("axis", [0, 1, 2])
def test_a_position_outside_the_table_gives_zeros_and_is_reported(axis):
    g = _gen(2)
    x = torch.randn(1, 6, 5, 64, generator=g, device="cuda").bfloat16()
    table = dsa.rotary_table(50, 64)
    pos = torch.randint(0, 50, (3, 1, 6), generator=g, device="cuda")
    good = dsa.rotary_embedding_axes(x, table, pos, [8, 12, 12])
    for layout, H in (("interleaved", 64), ("half", 64)):
        pos[axis, 0, 1], pos[axis, 0, 4] = -1, 50 + (1 << 33)
        got = dsa.rotary_embedding_axes(x, table, pos, [8, 12, 12], layout=layout)
        with pytest.raises(RuntimeError, match="bits 0x4"):
            dsa.check_device_errors()
        assert not got[0, [1, 4]].any()
        if layout == "interleaved":
            assert torch.equal(got[0, [0, 2, 3, 5]], good[0, [0, 2, 3, 5]])


def test_tokens_past_one_launch():
    """More than 2^30 pieces: the launch is divided, and offsets pass 32 bits."""
    n = (1 << 27) + 77
    x = torch.zeros(n, 1, 64, device="cuda", dtype=torch.bfloat16)
    pos = torch.zeros(2, n, device="cuda", dtype=torch.int32)
    pos[0, -1], pos[1, -1] = 3, 5
    x[-1] = 1.0
    table = dsa.rotary_table(8, 64)
    got = dsa.rotary_embedding_axes(x, table, pos, [16, 16], out=x)
    one = torch.ones(1, 1, 64, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(got[-1:], dsa.rotary_embedding_axes(one, table, pos[:, -1:].contiguous(), [16, 16]))
    assert not got[:-1].any()


@pytest.mark.parametrize("layout,order", [("interleaved", "cycled"), ("half", "blocks")])
def test_gradient(layout, order):
    """Against the formula's (autograd through the rotation in 64 bits), against differences, and the
    gradient's own gradient."""
    g = _gen(4)
    sections, offset = [12, 10, 10], 32
    pos = torch.randint(0, 3000, (3, 2, 5), generator=g, device="cuda", dtype=torch.int32)
    table = dsa.rotary_table(3000, 64)
    x = torch.randn(2, 5, 3, 96, generator=g, device="cuda", requires_grad=True)
    w = torch.randn(2, 5, 3, 96, generator=g, device="cuda", requires_grad=True)
    turn = lambda t: dsa.RotaryEmbeddingAxesFunction.apply(t, table, pos, sections, layout, order, offset)
    (got,) = torch.autograd.grad((turn(x) * w).sum(), x, create_graph=True)
    axis_of = _axes(sections, order)
    x64 = x.detach().double().requires_grad_()
    ang = pos.double()[axis_of].movedim(0, -1).unsqueeze(-2) * torch.tensor(dsa.rotary_frequencies(64), dtype=torch.float64, device="cuda")
    i = torch.arange(32, device="cuda")
    ia = offset + (2 * i if layout == "interleaved" else i)
    ib = ia + (1 if layout == "interleaved" else 32)
    a, b, w64 = x64[..., ia], x64[..., ib], w.detach().double()
    keep = [j for j in range(96) if j < offset]
    loss = ((a * ang.cos() - b * ang.sin()) * w64[..., ia] + (a * ang.sin() + b * ang.cos()) * w64[..., ib]).sum() \
        + (x64[..., keep] * w64[..., keep]).sum()
    (ref,) = torch.autograd.grad(loss, x64)
    bound = torch.zeros_like(ref)
    mag = w64[..., ia].abs() + w64[..., ib].abs()
    for at in (ia, ib):
        bound[..., at] = 2.0 ** -22 * mag + 2.0 ** -24 * ref[..., at].abs()
    assert bool(((got.double() - ref).abs() <= bound).all())
    # a linear map: its difference quotient is exact but for roundings (of values up to 10, 2^-20 each)
    step = torch.randn(x.shape, generator=g, device="cuda")
    slope = ((turn(x + step) - turn(x)) * w).sum().double()
    off = float((slope - (got * step).sum()).detach())
    assert abs(off) <= 2.0 ** -18 * float(((x.abs() + step.abs()) * w.abs()).detach().sum())
    # d(grad . v) / dw is the rotation of v
    v = torch.randn(x.shape, generator=g, device="cuda")
    (again,) = torch.autograd.grad((got * v).sum(), w)
    assert torch.equal(again, turn(v))


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_captured_on_another_stream_and_after(layout):
    g = _gen(5)
    x = torch.randn(2, 7, 16, 64, generator=g, device="cuda").bfloat16()
    pos = torch.randint(0, 90, (3, 2, 7), generator=g, device="cuda", dtype=torch.int32)
    table = dsa.rotary_table(90, 64)
    call = lambda: dsa.rotary_embedding_axes(x, table, pos, [12, 10, 10], layout=layout, order="cycled")
    ref = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert torch.equal(got, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    pos.copy_(89 - pos)
    graph.replay()
    assert torch.equal(got, call()) and not torch.equal(got, ref)


@pytest.mark.parametrize("order", ["blocks", "cycled"])
def test_backward_captured(order):
    """A step of forward and backward in a graph, run on a side stream before the capture; no graph of
    autograd's own outlives its run."""
    g = _gen(6)
    x = torch.randn(3, 5, 8, 64, generator=g, device="cuda").half().requires_grad_()
    w = torch.randn(3, 5, 8, 64, generator=g, device="cuda").half()
    pos = torch.randint(0, 50, (2, 3, 5), generator=g, device="cuda", dtype=torch.int32)
    table = dsa.rotary_table(50, 64)

    def step():
        out = dsa.RotaryEmbeddingAxesFunction.apply(x, table, pos, (17, 15), "half", order)
        return torch.autograd.grad(out, x, w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        pos.copy_(49 - pos)
        w.neg_()
        graph.replay()
        assert torch.equal(got, dsa.rotary_embedding_axes(w, table, pos, (17, 15), "half", order, inverse=True))
