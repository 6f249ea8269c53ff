"""Rotary positions against a plain 64-bit form.

With x the pair (a, b) and m the factor an output is a sum of two products of fp32 numbers: cos and sin are off by at most
2 units of 2^-24 (sincospif, and the first-order term), times m by one more, each product and the sum by one:
(|a| + |b|) m 2^-21 covers them, and the output's rounding is half a step of its type.  Angles are reduced in
double: 2^-50 of a position times a frequency, below 2^-29 for positions up to 2^21."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from rldx_b200.rope import B200Rope  # noqa: E402

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def axis_of(pair, sections, interleaved):
    if sections is None:
        return 0
    if interleaved:
        a = pair % len(sections)
        return a if pair < len(sections) * sections[a] else 0
    a, end = 0, sections[0]
    while pair >= end:
        a += 1
        end += sections[a]
    return a


def angles(positions, freqs, sections=None, interleaved_sections=False):
    p = positions.reshape(-1, positions.shape[-1]).double()
    return torch.stack([p[axis_of(i, sections, interleaved_sections)] * freqs[i] for i in range(freqs.numel())], 1)


def turned(x, angle, factor, interleaved, inverse):
    """x [T, H, d] -> its 64-bit rotation and |a| + |b| of every value's pair."""
    n = angle.shape[1]
    c, s = (angle.cos() * factor).unsqueeze(1), (angle.sin() * factor).unsqueeze(1)
    s = -s if inverse else s
    x = x.double()
    y, size = x.clone(), torch.zeros_like(x)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * abs(factor)
    return y, size


def close(got, want, size):
    # half a step of the type, also of its subnormal numbers
    info = torch.finfo(got.dtype)
    room = size * 2.0 ** -21 + want.abs() * info.eps / 2 + info.tiny * info.eps / 2
    assert bool(((got.double() - want).abs() <= room * (1 + 1e-6)).all())


def check(rope, q, k, positions, **kw):
    got = rope(q, k, positions, **kw)
    angle = angles(positions, rope.freqs, rope.sections, rope.interleaved_sections)
    for g, x in zip(got, (q, k)):
        if x is None:
            assert g is None
            continue
        assert g.shape == x.shape and g.dtype == x.dtype
        close(g, *turned(x, angle, rope.factor, rope.interleaved, kw.get("inverse", False)))


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("d,rotary", [(128, 128), (64, 32), (72, 72), (72, 36), (80, 20), (256, 64), (6, 2), (2, 2), (1024, 1024)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_heads_and_parts(cuda, dtype, d, rotary, interleaved):
    g = torch.Generator(device=cuda).manual_seed(d + rotary)
    rope = B200Rope(d, theta=1e4, rotary_dim=rotary, interleaved=interleaved, device=cuda)
    for tokens, hq, hk in ((1, 16, 2), (3, 5, 5), (67, 8, 1), (300, 1, 3)):
        q, k = (torch.randn(tokens, h, d, device=cuda, generator=g).to(dtype) for h in (hq, hk))
        at = torch.randint(5000, (tokens,), device=cuda, generator=g)
        check(rope, q, k, at)
        check(rope, q, None, at.int(), inverse=True)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("sections,interleaved", [((24, 20, 20), False), ((24, 20, 20), True), ((0, 64, 0), False), ((1, 1, 1, 61), True),
                                                  ((30, 34), True), ((64,), False)])
def test_axes(cuda, dtype, sections, interleaved):
    g = torch.Generator(device=cuda).manual_seed(sum(sections[:2]))
    rope = B200Rope(128, theta=1e6, sections=sections, interleaved_sections=interleaved, device=cuda)
    for t in (1, 530):
        at = torch.randint(2000, (len(sections), t), device=cuda, generator=g)
        x = torch.randn(t, 20 * 128, device=cuda, generator=g).to(dtype).unflatten(1, (20, 128))
        check(rope, x[:, :16], x[:, 16:18], at)
        cos, sin = rope.rows(at, dtype=dtype)
        angle = angles(at, rope.freqs, sections, interleaved).repeat(1, 2)
        for got, want in ((cos, angle.cos()), (sin, angle.sin())):
            close(got, want, torch.ones_like(want))
    same = torch.arange(40, device=cuda).expand(len(sections), -1)  # text: one place on every axis
    y = torch.randn(40, 2, 128, device=cuda, generator=g).to(dtype)
    one = B200Rope(128, theta=1e6, device=cuda)
    assert torch.equal(rope(y, None, same)[0], one(y, None, same[0])[0])


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 8.0}, {"type": "ntk", "factor": 4.0},
                                     {"type": "yarn", "factor": 16.0, "original": 4096}])
def test_far_and_negative_positions(cuda, scaling):
    g = torch.Generator(device=cuda).manual_seed(3)
    rope = B200Rope(64, theta=1e4, scaling=scaling, device=cuda)
    at = torch.tensor([0, 1, -1, 7, 2 ** 20, 2 ** 21 - 1, -(2 ** 20), 999983], device=cuda)
    q = torch.randn(8, 3, 64, device=cuda, generator=g)
    check(rope, q, None, at)
    check(rope, q.to(BF), None, at.int())
    cos, sin = rope.rows(at)
    angle = angles(at, rope.freqs).repeat(1, 2)
    close(cos, angle.cos() * rope.factor, torch.full_like(angle, rope.factor))
    close(sin, angle.sin() * rope.factor, torch.full_like(angle, rope.factor))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strides_and_alignment(cuda, dtype):
    """Rows of wider buffers, odd strides and starts, heads before tokens, one position for every axis, broadcast heads."""
    g = torch.Generator(device=cuda).manual_seed(5)
    rope = B200Rope(32, theta=1e4, rotary_dim=16, device=cuda)
    at = torch.arange(50, device=cuda) + 100
    wide = torch.randn(50, 5 * 32 + 7, device=cuda, generator=g).to(dtype)
    for shift in (0, 1, 2, 4):
        x = wide[:, shift: shift + 160].unflatten(1, (5, 32))
        check(rope, x[:, :3], x[:, 3:], at)
    odd = torch.randn(50, 4, 37, device=cuda, generator=g).to(dtype)[..., 3:35]
    check(rope, odd, odd[:, 1:2], at)
    heads_first = torch.randn(6, 50, 32, device=cuda, generator=g).to(dtype).transpose(0, 1)
    check(rope, heads_first, heads_first[:, ::2], at)
    check(rope, odd[:, :1].expand(-1, 7, -1), odd[:1].expand(50, -1, -1), at)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [128, 48])
def test_in_place_and_given_outputs(cuda, interleaved, rotary):
    g = torch.Generator(device=cuda).manual_seed(6)
    rope = B200Rope(128, theta=1e4, rotary_dim=rotary, interleaved=interleaved, device=cuda)
    at = torch.arange(333, device=cuda)
    qkv = torch.randn(333, 10 * 128 + 8, device=cuda, generator=g).to(BF)
    keep = qkv.clone()
    q, k = qkv[:, : 6 * 128].unflatten(1, (6, 128)), qkv[:, 6 * 128: 8 * 128].unflatten(1, (2, 128))
    want = [t.clone() for t in rope(q, k, at)]
    given = torch.full((6, 400, 128), 7.0, dtype=BF, device=cuda)  # heads before tokens, room behind
    out_q = given[:, :333].transpose(0, 1)
    got = rope(q, k, at, out_q=out_q)
    assert got[0] is out_q or got[0].data_ptr() == out_q.data_ptr()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and bool((given[:, 333:] == 7).all())
    rope(q, k, at, out_q=q, out_k=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(qkv[:, 8 * 128:], keep[:, 8 * 128:])
    one = keep[:, : 6 * 128].unflatten(1, (6, 128))
    rope(one, None, at, out_q=one)
    assert torch.equal(one, want[0])


def test_inverse_is_the_transpose(cuda):
    """<R x, y> = <x, R^-1 y> and R^-1 R x = x, up to the two rotations' roundings; differences give the same."""
    g = torch.Generator(device=cuda).manual_seed(7)
    rope = B200Rope(64, theta=1e4, rotary_dim=48, device=cuda)
    at = torch.randint(9000, (200,), device=cuda, generator=g)
    x, y = (torch.randn(200, 3, 64, device=cuda, generator=g) for _ in range(2))
    a, b = rope(x, None, at)[0], rope(y, None, at, inverse=True)[0]
    dots = (a.double() * y.double()).sum(), (x.double() * b.double()).sum()
    # each value is off by 2^-21 (|a| + |b|) at most
    room = 2 * 2.0 ** -21 * 2 * float((x.double().abs().amax() * y.double().abs()).sum() + (y.double().abs().amax() * x.double().abs()).sum())
    assert abs(float(dots[0] - dots[1])) <= room
    back = rope(a, None, at, inverse=True)[0]
    pair = turned(x, angles(at, rope.freqs), 1.0, False, False)[1]
    assert bool(((back.double() - x.double()).abs() <= 2 * pair * 2.0 ** -20 + 2.0 ** -23 * x.double().abs()).all())


def test_other_values_pass_unchanged(cuda):
    """NaN and infinities stay in their pairs; values past the rotated part keep their bits."""
    rope = B200Rope(64, theta=1e4, rotary_dim=32, device=cuda)
    x = torch.randn(20, 2, 64, device=cuda)
    x[3, 0, 5], x[4, 1, 20], x[5, 0, 40] = math.nan, math.inf, math.nan
    y = rope(x, None, torch.arange(20, device=cuda))[0]
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[3, 0, [5, 21]] = True
    want[4, 1, [4, 20]] = True
    want[5, 0, 40] = True
    assert torch.equal(bad, want)
    assert torch.equal(y[..., 32:].view(torch.int32), x[..., 32:].contiguous().view(torch.int32))


def test_captured_and_on_another_stream(cuda):
    rope = B200Rope(128, theta=1e6, device=cuda)
    q, k = torch.randn(77, 4, 128, device=cuda).to(BF), torch.randn(77, 2, 128, device=cuda).to(BF)
    at = torch.arange(77, device=cuda)
    want = rope(q, k, at)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        here = rope(q, k, at)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(here, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = rope(q, k, at)
        cos, _ = rope.rows(at)
    at += 1000
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, rope(q, k, at))) and torch.equal(cos, rope.rows(at)[0])


def test_no_tokens(cuda):
    rope = B200Rope(128, device=cuda)
    at = torch.empty(0, dtype=torch.int64, device=cuda)
    q, k = rope(torch.empty(0, 4, 128, device=cuda), torch.empty(0, 2, 128, device=cuda), at)
    assert q.shape == (0, 4, 128) and k.shape == (0, 2, 128) and rope.rows(at)[0].shape == (0, 128)


def test_offsets_past_32_bits(cuda):
    """Tokens of a stride that takes the last ones past 2^31 elements."""
    rope = B200Rope(64, theta=1e4, device=cuda)
    buffer = torch.empty(5 * 10 ** 8 * 5 + 64, dtype=BF, device=cuda)
    x = buffer.as_strided((6, 1, 64), (5 * 10 ** 8, 64, 1))
    x.copy_(torch.randn(6, 1, 64, device=cuda))
    at = torch.arange(6, device=cuda) + 5
    check(rope, x, None, at)
    want = rope(x, None, at)[0]
    rope(x, None, at, out_q=x)
    assert torch.equal(x, want)
