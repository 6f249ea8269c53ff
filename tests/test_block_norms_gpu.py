"""The norms after and before a block against a plain 64-bit form.

Roundings: a value passes at most 64 fp32 operations (16 of a thread's sum and 10 of the tree for each of up to four
sums, the rest products), so with u = 2^-18 = 64 x 2^-24 an intermediate is off by u times the size of the terms
it is made of.  With A = |h| + |scale gate| (|x^ w| + mean|y| inv |w| + |b|) that is u A for the sum; the pre
norm takes the sum's error times inv, that of the mean and of the mean square (at most the rows' root mean square of A)
and its own u.  The results' own rounding is half a step of their type."""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -18


def norm(x, kind, w, b, plus, eps):
    """The norm, and the size of the terms it is made of."""
    if kind is None:
        return x, x.abs()
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    inv = 1.0 / ((x - mean).pow(2).mean(1, keepdim=True) + eps).sqrt()
    w = 1.0 if w is None else w.double() + (1.0 if plus else 0.0)
    b = 0.0 if b is None else b.double()
    w_size = abs(w)
    size = ((x - mean).abs() + (x.abs().mean(1, keepdim=True) if kind == "layer" else 0.0)) * inv * w_size + abs(b)
    return (x - mean) * inv * w + b, size


def of_rows(v, rows, group):
    if v is None or v.dim() == 1:
        return v if v is None else v.double()
    return v.double()[torch.arange(rows, device=v.device) // group]


def check(branch, residual, *, post=None, post_weight=None, post_bias=None, gate=None, scale=1.0, pre="rms", pre_weight=None, pre_bias=None,
          mod_scale=None, mod_shift=None, rows_per_group=0, weight_plus_one=False, eps=1e-6, **out):
    rows = branch.shape[0]
    y, h0 = branch.double(), residual.double()
    got_h, got_n = ops.block_norms(branch, residual, post=post, post_weight=post_weight, post_bias=post_bias, gate=gate, scale=scale, pre=pre,
                                   pre_weight=pre_weight, pre_bias=pre_bias, mod_scale=mod_scale, mod_shift=mod_shift,
                                   rows_per_group=rows_per_group, weight_plus_one=weight_plus_one, eps=eps, **out)
    y, size = norm(y, post, post_weight, post_bias, weight_plus_one, eps)
    g = of_rows(gate, rows, rows_per_group)
    g = scale if g is None else scale * g
    h = h0 + g * y
    a = h0.abs() + abs(g) * size

    def close(got, want, off):
        info = torch.finfo(got.dtype)
        room = off + (want.abs() + off) * info.eps / 2 + info.tiny * info.eps / 2
        wrong = ~((got.double() - want).abs() <= room)
        assert not bool(wrong.any()), ((got.double() - want).abs() / room).max()

    assert got_h.dtype == residual.dtype and got_h.shape == branch.shape
    close(got_h, h, U * a)
    if pre is None:
        assert got_n is None
        return got_h, got_n
    n, n_size = norm(h, pre, pre_weight, pre_bias, weight_plus_one, eps)
    mean = h.mean(1, keepdim=True) if pre == "layer" else 0.0
    inv = 1.0 / ((h - mean).pow(2).mean(1, keepdim=True) + eps).sqrt()
    w = 1.0 if pre_weight is None else (pre_weight.double() + (1.0 if weight_plus_one else 0.0)).abs()
    bent = (h - mean).abs() * inv  # how much an error of inv weighs
    off = U * ((a + a.mean(1, keepdim=True) + bent * a.pow(2).mean(1, keepdim=True).sqrt()) * inv * w + n_size)
    s, t = of_rows(mod_scale, rows, rows_per_group), of_rows(mod_shift, rows, rows_per_group)
    if s is not None:
        n, off = n * (1 + s), off * (1 + s.abs()) + U * n.abs() * (1 + s.abs())
    if t is not None:
        n, off = n + t, off + U * t.abs()
    assert got_n.dtype == branch.dtype and got_n.shape == branch.shape
    close(got_n, n, off)
    return got_h, got_n


TYPES = [(BF, BF), (BF, F32), (F16, F16), (F16, F32), (F32, F32)]


def rows_of(g, dev, n, w, dtype, size=1.0, pad=0, shift=0):
    x = torch.empty(n, w + pad + shift, dtype=dtype, device=dev)[:, shift: shift + w]
    return x.copy_(size * torch.randn(n, w, device=dev, generator=g) + 0.2)


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("width", [1, 2, 7, 16, 64, 100, 513, 1001, 1536, 2048, 5000, 14336])
def test_kinds(cuda, dtype, stream, width):
    g = torch.Generator(device=cuda).manual_seed(width)
    n = 37 if width < 5000 else 5
    y, h = rows_of(g, cuda, n, width, dtype), rows_of(g, cuda, n, width, stream, 3.0)
    vec = lambda *shape: (0.5 * torch.randn(*shape, width, device=cuda, generator=g)).to(dtype)  # noqa: E731
    for post, pre in itertools.product((None, "rms", "layer"), repeat=2):
        check(y, h, post=post, pre=pre, eps=1e-5)
        check(y, h, post=post, post_weight=vec() if post else None, post_bias=vec() if post else None, gate=vec(), scale=0.3, pre=pre,
              pre_weight=vec() if pre else None, pre_bias=vec() if pre else None, mod_scale=vec(-(-n // 5)) if pre else None,
              mod_shift=vec() if pre else None, rows_per_group=5)
        check(y, h, post=post, post_weight=vec() if post else None, pre=pre, pre_weight=vec() if pre else None, weight_plus_one=True, gate=vec(-(-n // 4)),
              rows_per_group=4)


@pytest.mark.parametrize("dtype,stream", TYPES)
def test_strides_groups_and_vector_types(cuda, dtype, stream):
    g = torch.Generator(device=cuda).manual_seed(2)
    for width, pad, shift in ((96, 8, 0), (96, 4, 4), (97, 3, 1), (1000, 0, 2), (1001, 7, 0), (2050, 6, 0)):
        y, h = rows_of(g, cuda, 23, width, dtype, pad=pad, shift=shift), rows_of(g, cuda, 23, width, stream, 2.0, pad=pad, shift=shift)
        for vt in (dtype, F32):
            wide = torch.randn(6, 2 * width + 1, device=cuda, generator=g).to(vt)
            one = torch.randn(width + 1, device=cuda, generator=g).to(vt)
            check(y, h, post="rms", post_weight=one[1:], gate=wide[:, :width], scale=-0.7, pre="layer", pre_weight=one[:-1],
                  mod_scale=wide[:, width: 2 * width], mod_shift=wide[:, 1: 1 + width], rows_per_group=4)
            check(y, h, gate=wide[:1, :width], pre="rms", mod_shift=wide[:1, :width], rows_per_group=40)
    one_row = rows_of(g, cuda, 1, 200, dtype)
    check(one_row.expand(9, -1), rows_of(g, cuda, 9, 200, stream))


@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("width", [8, 128, 512, 1536, 4096, 4104])
def test_groups_of_few_and_of_many_rows(cuda, dtype, stream, width):
    """Rows enough that a CTA goes over several, groups that end inside its run, behind it and in each row."""
    g = torch.Generator(device=cuda).manual_seed(width)
    n = 9001 if width <= 512 else 2003
    y, h = rows_of(g, cuda, n, width, dtype), rows_of(g, cuda, n, width, stream, 2.0)
    for group in (1, 3, 15, 16, 700, n, n + 5, 2 ** 40):
        count = -(-n // group)
        wide = (0.5 * torch.randn(count, 2 * width, device=cuda, generator=g)).to(dtype)
        gate = (0.5 * torch.randn(count, width, device=cuda, generator=g)).to(dtype)
        check(y, h, post="rms", gate=gate, pre="layer", mod_scale=wide[:, :width], mod_shift=wide[:, width:], rows_per_group=group)
        check(y, h, gate=gate[0], pre="rms", mod_shift=wide[:, :width], rows_per_group=group)
        check(y, h, post="layer", post_bias=gate[0], gate=gate, pre=None, rows_per_group=group)


@pytest.mark.parametrize("dtype,stream", [(BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("width", [40, 2048, 1001])
def test_in_place(cuda, dtype, stream, width):
    g = torch.Generator(device=cuda).manual_seed(4)
    y, h = rows_of(g, cuda, 300, width, dtype, pad=5), rows_of(g, cuda, 300, width, stream, pad=5)
    # (rows of one stride: sums of others may be taken in another order)
    want = ops.block_norms(y, h, post="rms", pre="layer", out=torch.empty_like(y._base)[:, :width], out_residual=torch.empty_like(h._base)[:, :width])
    y2, h2 = torch.empty_like(y._base).copy_(y._base)[:, :width], torch.empty_like(h._base).copy_(h._base)[:, :width]
    got = ops.block_norms(y2, h2, post="rms", pre="layer", out_residual=h2, out=y2)
    assert got[0].data_ptr() == h2.data_ptr() and got[1].data_ptr() == y2.data_ptr()
    assert torch.equal(h2, want[0]) and torch.equal(y2, want[1])
    if dtype == stream:  # the other way round
        y3, h3 = y.clone(), h.clone()
        want = ops.block_norms(y3, h3, post="rms", pre="layer")
        ops.block_norms(y3, h3, post="rms", pre="layer", out_residual=y3, out=h3)
        assert torch.equal(y3, want[0]) and torch.equal(h3, want[1])


def test_large_means_small_spreads_and_special_values(cuda):
    g = torch.Generator(device=cuda).manual_seed(5)
    y = 1000.0 + 0.01 * torch.randn(6, 1536, device=cuda, generator=g)
    check(y, torch.zeros_like(y), post="layer", pre="layer")  # the variance is not a difference of large sums
    check(1e-20 * y, 1e-20 * y, post=None, pre="rms")
    check(1e15 * y, 1e15 * y, post="rms", pre="rms")
    zero = torch.zeros(4, 512, device=cuda, dtype=BF)
    h, n = ops.block_norms(zero, zero, post="layer", pre="rms")
    assert not bool(h.any()) and not bool(n.any())
    y = torch.randn(4, 512, device=cuda)
    y[1, 3], y[2, 5] = float("nan"), float("inf")
    h, n = ops.block_norms(y, torch.ones_like(y), post=None, pre="rms")
    assert bool(torch.isfinite(n[[0, 3]]).all()) and bool(torch.isnan(n[1]).all()) and bool(torch.isnan(n[2, 5]))
    f16 = torch.full((2, 64), 60000.0, device=cuda, dtype=F16)
    h, n = ops.block_norms(f16, f16, post=None, pre="rms")
    assert bool(torch.isinf(h).all()) and bool((n == 1).all())  # the norm takes the sum before its rounding


def test_rows_do_not_depend_on_the_batch(cuda):
    g = torch.Generator(device=cuda).manual_seed(6)
    y, h = rows_of(g, cuda, 1000, 1536, BF), rows_of(g, cuda, 1000, 1536, BF)
    whole = ops.block_norms(y, h, post="rms", pre="layer")
    for r in (0, 501, 999):
        one = ops.block_norms(y[r: r + 1], h[r: r + 1], post="rms", pre="layer")
        assert all(torch.equal(a[r: r + 1], b) for a, b in zip(whole, one))
    h0, n0 = ops.block_norms(y[:0], h[:0])
    assert h0.shape == n0.shape == (0, 1536)


def test_captured_and_on_another_stream(cuda):
    g = torch.Generator(device=cuda).manual_seed(7)
    y, h = rows_of(g, cuda, 100, 2048, BF), rows_of(g, cuda, 100, 2048, F32)
    want = ops.block_norms(y, h, post="rms")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        here = ops.block_norms(y, h, post="rms")
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(here, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a, n = ops.block_norms(y, h, post="rms")
        b, n = ops.block_norms(n, a, post="layer", out=n)
    y.mul_(-2)
    graph.replay()
    a2, n2 = ops.block_norms(y, h, post="rms")
    b2, n2 = ops.block_norms(n2, a2, post="layer")
    assert torch.equal(b, b2) and torch.equal(n, n2)


def test_offsets_past_32_bits(cuda):
    buffer = torch.empty(4 * 10 ** 8 * 6 + 800, dtype=BF, device=cuda)
    y, h = buffer.as_strided((7, 256), (4 * 10 ** 8, 1)), buffer.as_strided((7, 256), (4 * 10 ** 8, 1), 512)  # (as aligned as dense rows)
    y.copy_(torch.randn(7, 256, device=cuda)), h.copy_(torch.randn(7, 256, device=cuda))
    check(y, h, post="rms", pre="layer")
    want = ops.block_norms(y, h, post="rms", pre="layer")
    ops.block_norms(y, h, post="rms", pre="layer", out_residual=h, out=y)
    assert torch.equal(h, want[0]) and torch.equal(y, want[1])
