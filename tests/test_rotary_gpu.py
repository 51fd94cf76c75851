"""rotary_embedding against the rotation in 64 bits, and its gradient (GPU).

Tolerance: the kernel forms a c - b s and a s + b c in fp32 from table entries rounded once to
fp32, so each product is off by at most 2^-23 of |a| + |b| times the amplitude, and the result is
rounded once to the element type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32 of its size).  The bound used
is 2^-22 A (|a| + |b|) + u |result| with that u; copied values are exact.
"""
import math

import pytest
import torch

import dsa_triton_ascend_b200 as dsa

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _expect(x, positions, freq, amplitude, layout, offset, inverse):
    """(value, bound) in 64 bits, from the definition."""
    half = len(freq)
    ang = positions.double()[..., None, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    c, s = amplitude * ang.cos(), amplitude * ang.sin() * (-1 if inverse else 1)
    i = torch.arange(half, device=x.device)
    ia = offset + (2 * i if layout == "interleaved" else i)
    ib = ia + (1 if layout == "interleaved" else half)
    ref = x.double().clone()
    a, b = x.double()[..., ia], x.double()[..., ib]
    ref[..., ia], ref[..., ib] = a * c - b * s, a * s + b * c
    bound = torch.zeros_like(ref)
    for at in (ia, ib):
        bound[..., at] = 2.0 ** -22 * amplitude * (a.abs() + b.abs()) + UNIT[x.dtype] * ref[..., at].abs()
        if x.dtype == torch.float16:
            bound[..., at] += 2.0 ** -25   # half a step among the subnormal values
    return ref, bound


def _check(x, positions, dim, layout, offset, inverse=False, out=None, **scaling):
    amplitude = scaling.get("amplitude", 1.0)
    maxp = int(positions.max()) + 1 if positions.numel() else 1
    table = dsa.rotary_table(max(maxp, 1), dim, **scaling)
    scaling.pop("amplitude", None)
    freq = dsa.rotary_frequencies(dim, **scaling)
    ref, bound = _expect(x, positions, freq, amplitude, layout, offset, inverse)
    got = dsa.rotary_embedding(x, table, positions, layout=layout, offset=offset, inverse=inverse, out=out)
    dsa.check_device_errors()
    assert got.shape == x.shape and got.dtype == x.dtype
    assert bool(((got.double() - ref).abs() <= bound).all())
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("B,S,N,H,dim,offset", [
    (1, 1, 1, 64, 64, 0), (2, 5, 128, 64, 64, 0), (3, 7, 5, 192, 64, 128), (1, 33, 64, 128, 64, 0),
    (2, 3, 6, 160, 32, 64), (1, 257, 3, 256, 256, 0),
    (2, 4, 3, 10, 6, 1), (1, 3, 2, 7, 2, 5), (2, 2, 9, 36, 12, 20)])   # no whole 16-byte pieces
def test_rotation(dtype, layout, inverse, B, S, N, H, dim, offset):
    g = _gen(B * 1000 + S * 10 + H)
    x = torch.randn(B, S, N, H, generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 5000, (B, S), generator=g, device="cuda", dtype=torch.int32)
    _check(x, pos, dim, layout, offset, inverse)


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=8.0), dict(scaling="ntk", factor=4.0),
                                dict(scaling="yarn", factor=16.0, original_positions=4096, amplitude=1.2772588722),
                                dict(base=500000.0)])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_scaled_angles_at_long_positions(kw, layout):
    """At position 131071 an angle formed in fp32 would be off by up to 2^-8 radians."""
    g = _gen(3)
    x = torch.randn(1, 4, 3, 64, generator=g, device="cuda")
    pos = torch.tensor([[0, 1, 100001, 131071]], dtype=torch.int32, device="cuda")
    _check(x, pos, 64, layout, 0, **kw)


def test_yarn_keeps_fast_pairs_and_divides_slow_ones():
    plain = dsa.rotary_frequencies(64)
    yarn = dsa.rotary_frequencies(64, scaling="yarn", factor=16.0, original_positions=4096)
    turns = [4096 * f / (2 * math.pi) for f in plain]
    for f, y, t in zip(plain, yarn, turns):
        if t > 32 * plain[0] / plain[1]:
            assert y == f
        if t < 1 * plain[1] / plain[0]:
            assert y == pytest.approx(f / 16.0, rel=1e-12)
        assert f / 16.0 <= y * (1 + 1e-12) and y <= f * (1 + 1e-12)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_strided_views_tokens_first_and_in_place(layout):
    g = _gen(11)
    wide = torch.randn(2, 9, 6, 192, generator=g, device="cuda").bfloat16()
    pos = torch.randint(0, 99, (2, 9), generator=g, device="cuda")          # int64
    a = _check(wide[..., 128:], pos, 64, layout, 0)
    _check(wide.transpose(1, 2).contiguous().transpose(1, 2)[..., 128:], pos, 64, layout, 0)
    _check(wide[:, ::2, 1::2, 3:73], pos[:, ::2], 64, layout, 5)              # no aligned base
    t = wide.reshape(18, 6, 192)[..., 128:]
    assert torch.equal(_check(t, pos.reshape(18), 64, layout, 0), a.reshape(18, 6, 64))
    into = torch.zeros(2, 9, 6, 100, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(_check(wide[..., 128:], pos, 64, layout, 0, out=into[..., 4:68]), a)
    assert not into[..., :4].any() and not into[..., 68:].any()
    mine = wide.clone()[..., 128:]
    table = dsa.rotary_table(99, 64)
    assert dsa.rotary_embedding(mine, table, pos, layout=layout, out=mine) is mine
    assert torch.equal(mine, a)


@pytest.mark.parametrize("H,dim,offset", [(64, 64, 0), (10, 6, 1)])
def test_positions_outside_the_table(H, dim, offset):
    x = torch.ones(1, 4, 2, H, device="cuda", dtype=torch.bfloat16)
    table = dsa.rotary_table(8, dim)
    for dtype in (torch.int32, torch.int64):
        pos = torch.tensor([[3, -1, 8, 7]], device="cuda", dtype=dtype)
        if dtype == torch.int64:
            pos[0, 1], pos[0, 2] = -(1 << 40), 1 << 40
        got = dsa.rotary_embedding(x, table, pos, offset=offset)
        with pytest.raises(RuntimeError, match="bits 0x4"):
            dsa.check_device_errors()
        assert not got[0, 1:3].any() and bool(got[0, 0].any()) and bool(got[0, 3].any())


def test_empty():
    table = dsa.rotary_table(8, 64)
    for shape in ((0, 3, 2, 64), (2, 0, 2, 64), (2, 3, 0, 64)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        assert dsa.rotary_embedding(x, table, torch.zeros(shape[:2], device="cuda", dtype=torch.int32)).shape == shape
    dsa.check_device_errors()


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient(layout):
    """Against the formula (the transposed rotation) and against central differences.  The map
    is linear, so a difference quotient has no truncation error; in fp32 with steps of 1 it
    carries the rounding of two results of size <= |x| + 1 each: 2 * 2^-22 * (6 + 1) = 3.4e-6."""
    g = _gen(7)
    x = torch.randn(1, 3, 2, 12, generator=g, device="cuda").clamp(-6, 6).requires_grad_()
    pos = torch.tensor([[0, 5, 1000]], device="cuda", dtype=torch.int32)
    table = dsa.rotary_table(1001, 8, amplitude=1.0)
    w = torch.randn(x.shape, generator=g, device="cuda")
    y = dsa.RotaryEmbeddingFunction.apply(x, table, pos, layout, 2)
    y.backward(w)
    ref, bound = _expect(w, pos, dsa.rotary_frequencies(8), 1.0, layout, 2, True)
    assert bool(((x.grad.double() - ref).abs() <= bound).all())
    with torch.no_grad():
        flat = x.detach().reshape(-1)
        for i in range(0, flat.numel(), 5):
            up, down = flat.clone(), flat.clone()
            up[i] += 1.0
            down[i] -= 1.0
            f = lambda v: dsa.rotary_embedding(v.reshape(x.shape), table, pos, layout=layout, offset=2).double()
            step = (up[i] - down[i]).double()
            quotient = ((f(up) - f(down)) * w.double()).sum() / step
            # the difference touches two outputs, each weighted by |w| <= 5
            assert abs(float(quotient - x.grad.reshape(-1)[i].double())) <= 2 * 5 * 3.4e-6
    dsa.check_device_errors()


def test_gradient_of_an_expanded_result():
    """d(out) of a sum over tokens is an expanded tensor (stride 0)."""
    x = torch.randn(2, 3, 4, 64, generator=_gen(1), device="cuda").requires_grad_()
    pos = torch.arange(6, device="cuda", dtype=torch.int32).reshape(2, 3)
    table = dsa.rotary_table(6, 64)
    dsa.RotaryEmbeddingFunction.apply(x, table, pos).sum().backward()
    ref, bound = _expect(torch.ones_like(x), pos, dsa.rotary_frequencies(64), 1.0, "interleaved", 0, True)
    assert bool(((x.grad.double() - ref).abs() <= bound).all())


def test_on_another_stream():
    x = torch.randn(1, 512, 64, 64, generator=_gen(2), device="cuda").bfloat16()
    pos = torch.arange(512, device="cuda", dtype=torch.int32)[None]
    table = dsa.rotary_table(512, 64)
    ref = dsa.rotary_embedding(x, table, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dsa.rotary_embedding(x, table, pos)
    side.synchronize()
    assert torch.equal(got, ref)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_gradient_of_the_gradient(layout):
    """The gradient is linear in d(out), so it has a gradient of its own: the rotation again.  With
    g = R^T w, the sum of g v has the derivative R v in w."""
    x = torch.randn(1, 3, 2, 12, generator=_gen(8), device="cuda", requires_grad=True)
    w = torch.randn(x.shape, generator=_gen(9), device="cuda", requires_grad=True)
    v = torch.randn(x.shape, generator=_gen(10), device="cuda")
    pos = torch.tensor([[0, 5, 1000]], device="cuda", dtype=torch.int32)
    table = dsa.rotary_table(1001, 8)
    y = dsa.RotaryEmbeddingFunction.apply(x, table, pos, layout, 2)
    g, = torch.autograd.grad(y, x, w, create_graph=True)
    for got, arg, inverse in ((g, w, True), (torch.autograd.grad(g, w, v)[0], v, False)):
        ref, bound = _expect(arg.detach(), pos, dsa.rotary_frequencies(8), 1.0, layout, 2, inverse)
        assert bool(((got.detach().double() - ref).abs() <= bound).all())
