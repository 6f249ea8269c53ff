"""Sampling against a plain row-by-row implementation with exact sums.

The weights are by definition whole numbers of the fp32 exponential; the plain form takes that
exponential from torch, sums Python integers, and has to give the same tokens and counts.
logprob is one rounding of a 64-bit logarithm (2^-24 relative, plus 2^-50 of the sums)."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import _lib, ops  # noqa: E402

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def plain(logits, u, t, k, p, m):
    """One row, in the order of the definition."""
    x = torch.where(torch.isnan(logits), torch.full_like(logits, -math.inf), logits.float() + 0.0)
    top = x.max()
    if top == -math.inf:
        return -1, -math.inf, 0
    if not t > 0:
        return int((x == top).nonzero()[0]), 0.0, 1
    d = torch.where(x == top, torch.zeros_like(x), (x - top) / torch.tensor(max(t, 1e-30), dtype=F32, device=x.device))
    w = (d.exp() * 4294967296.0).to(torch.int64).tolist()
    order = torch.argsort(x, descending=True, stable=True).tolist()
    if 0 < k < len(order):
        order = order[:k]
    total, before, kept = sum(w[i] for i in order), 0, []
    for rank, i in enumerate(order):
        if w[i] > 0 and (rank == 0 or not p < 1 or before < p * total) and w[i] >= min(max(m, 0.0), 1.0) * 4294967296.0:
            kept.append(i)
        before += w[i]
    kept.sort()
    total = sum(w[i] for i in kept)
    goal, reach = min(max(int(u * float(total)), 0), total - 1), 0
    for i in kept:
        reach += w[i]
        if reach > goal:
            return i, math.log(w[i] / total), len(kept)


def f32(v):
    return torch.tensor(v, dtype=F32).item()


def run_and_check(logits, u, t=None, k=None, p=None, m=None):
    dev, rows = logits.device, logits.shape[0]

    def vec(v, dtype):
        return None if v is None else torch.tensor(v, dtype=dtype, device=dev)

    uu = torch.tensor(u, dtype=F32, device=dev)
    token, logprob, kept = ops.sample(logits, uu, temperature=vec(t, F32), top_k=vec(k, I32), top_p=vec(p, F32), min_p=vec(m, F32))
    torch.cuda.synchronize()
    for r in range(rows):
        want = plain(logits[r], f32(u[r]), 1.0 if t is None else f32(t[r]), 0 if k is None else k[r],
                     1.0 if p is None else f32(p[r]), 0.0 if m is None else f32(m[r]))
        got = (token[r].item(), logprob[r].item(), kept[r].item())
        assert got[0] == want[0] and got[2] == want[2], (r, got, want)
        if math.isfinite(want[1]):
            assert abs(got[1] - want[1]) <= 2.0 ** -24 * abs(want[1]) + 2.0 ** -50, (r, got, want)
        else:
            assert got[1] == want[1]


def rows_of(g, dev, rows, vocab, dtype, spread=2.0, pad=0, shift=0):
    wide = torch.empty(rows, vocab + pad + shift, dtype=dtype, device=dev)
    x = wide[:, shift: shift + vocab]
    x.copy_(spread * torch.randn(rows, vocab, device=dev, generator=g) - 3.0)
    hot = torch.randint(vocab, (rows, max(1, vocab // 50)), device=dev, generator=g)
    x.scatter_add_(1, hot, (3.0 * torch.rand(hot.shape, device=dev, generator=g)).to(dtype))
    return x


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab,pad,shift", [(1, 0, 0), (7, 2, 1), (1000, 0, 0), (4097, 3, 5), (32003, 0, 3), (50257, 7, 0)])
def test_filters(cuda, dtype, vocab, pad, shift):
    g = torch.Generator(device=cuda).manual_seed(vocab + pad)
    x = rows_of(g, cuda, 12, vocab, dtype, pad=pad, shift=shift)
    u = torch.rand(12, generator=torch.Generator().manual_seed(vocab)).tolist()
    run_and_check(x, u)
    run_and_check(x, u, t=[0.5, 1.0, 2.0, 0.0, 1.3, 0.9, 1.0, 0.7, 1.0, 5.0, 1e-3, 100.0])
    run_and_check(x, u, k=[1, 2, 5, 50, 1000, 0, -1, vocab, vocab - 1, vocab + 9, 333, 20])
    run_and_check(x, u, p=[0.0, 0.1, 0.5, 0.9, 0.95, 0.99, 0.9999, 1.0, 1.5, 1e-9, 0.3, 0.7])
    run_and_check(x, u, m=[0.0, 0.01, 0.05, 0.5, 1.0, 2.0, -1.0, 1e-6, 0.2, 0.1, 0.3, 0.9])
    run_and_check(x, u, t=[0.8] * 6 + [1.5] * 6, k=[50, 40, 1000, 3, 0, 7] * 2, p=[0.95, 0.5, 0.9, 0.99, 0.8, 1.0] * 2,
                  m=[0.0, 0.02, 0.1] * 4)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [9, 2048, 40000])
def test_ties_go_to_the_lowest_id(cuda, dtype, vocab):
    """Rows of one value, of two and of a few: cuts that fall among equal logits."""
    g = torch.Generator(device=cuda).manual_seed(vocab)
    x = torch.zeros(8, vocab, dtype=dtype, device=cuda)
    x[1] = -2.5
    x[2, ::2] = 1.0
    x[3:] = torch.randint(-2, 3, (5, vocab), device=cuda, generator=g).to(dtype) * 0.5
    x[4, ::3] = -0.0
    u = [0.0, 0.3, 0.999999, 0.5, 0.7, 0.9, 0.1, 0.25]
    for k in (1, 3, vocab // 2 + 1, vocab - 1):
        run_and_check(x, u, k=[k] * 8)
        run_and_check(x, u, k=[k] * 8, p=[0.6] * 8, m=[0.1] * 8)
    for p in (0.001, 0.5, 0.77):
        run_and_check(x, u, p=[p] * 8)
    run_and_check(x, u, t=[0.0] * 8)


@pytest.mark.parametrize("dtype", [F32, BF])
@pytest.mark.parametrize("vocab", [300, 5000, 33000])
def test_list_lengths_and_ties_at_the_cut(cuda, dtype, vocab):
    """Cuts by count from one token to more than any list holds, on values that many tokens share, with top-p and min-p after."""
    g = torch.Generator(device=cuda).manual_seed(vocab)
    ks = [1, 2, 90, 100, 127, 128, 129, 200, 1000, 1500, 1536, 1537, 2500]
    rows = 3 * len(ks)
    x = torch.randn(rows, vocab, device=cuda, generator=g)
    x[len(ks): 2 * len(ks)] = (2 * x[len(ks): 2 * len(ks)]).round()  # a few values only
    x[2 * len(ks):] *= 4
    u = torch.rand(rows, device=cuda, generator=g).tolist()
    pick = lambda values: [values[i % len(values)] for i in range(rows)]  # noqa: E731
    run_and_check(x.to(dtype), u, t=pick([1.0, 0.7, 1.9, 0.25]), k=ks * 3)
    run_and_check(x.to(dtype), u, t=pick([1.0, 0.7, 1.9]), k=ks * 3, p=pick([0.9, 0.5, 0.999, 0.05, 1.0]), m=pick([0.0, 0.1]))


@pytest.mark.parametrize("dtype", [F32, BF])
def test_masks_of_the_lowest_value_and_large_logits(cuda, dtype):
    g = torch.Generator(device=cuda).manual_seed(4)
    vocab, low = 9000, torch.finfo(dtype).min
    x = torch.randn(10, vocab, device=cuda, generator=g)
    x[0] = low  # every token masked: all equal
    x[1, 5:] = low
    x[2, ::2] = low
    x[3] = x[3] * 1e30
    x[4] = x[4] * 100 + 1e6
    x[5] = x[5] * 100 - 1e6
    x[6] = -x[6].abs() * 1e-30
    x[7] = x[7] * 1e-3 - 3e4
    x[8, : vocab - 2] = -math.inf
    x[9] = low
    x[9, 8999] = -low
    x = x.to(dtype)
    u = torch.rand(10, device=cuda, generator=g).tolist()
    for t in (1.0, 0.01, 1e-30, 1e30, 3e38):
        for k, p in ((0, 0.5), (0, 0.9), (50, 0.9), (4000, 1.0), (4000, 0.7), (0, 1.0)):
            run_and_check(x, u, t=[t] * 10, k=[k] * 10, p=[p] * 10)


def test_special_rows(cuda):
    """Infinities, NaN, rows that a mask empties, values of a type's range, draws at the ends."""
    v = 300
    x = torch.randn(10, v, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 5:] = -math.inf
    x[3, 7], x[3, 250] = math.inf, math.inf
    x[4, ::2] = math.nan
    x[5] = torch.finfo(F32).min
    x[6, :150] = torch.finfo(F32).min
    x[7, 100] = torch.finfo(F32).max
    x[8] = torch.linspace(-1e-38, 1e-38, v, device=cuda)
    x[9, 1:] = -math.inf
    for u in (0.0, 0.5, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0):
        for kw in ({}, {"k": [3] * 10}, {"p": [0.8] * 10}, {"t": [0.0] * 10}, {"t": [1e-35] * 10}, {"t": [1e30] * 10},
                   {"k": [150] * 10, "p": [0.5] * 10, "m": [0.5] * 10}):
            run_and_check(x, [u] * 10, **kw)
    nan = float("nan")
    run_and_check(x, [0.4] * 10, t=[nan] * 10)
    uu = torch.full((10,), 0.4, device=cuda)
    want = ops.sample(x, uu)
    got = ops.sample(x, uu, top_p=torch.full((10,), nan, device=cuda), min_p=torch.full((10,), nan, device=cuda))
    assert all(torch.equal(a, b) for a, b in zip(want, got))  # NaN limits are off


def test_wide_spread_crosses_inside_one_bin(cuda):
    """fp32 logits a few ulps apart: the cut is found by ordered bits inside a bin, across zero too."""
    v = 20000
    base = torch.arange(v, device=cuda, dtype=F32)
    x = torch.stack([5.0 + base * 2.0 ** -21, (base - v // 2) * 1e-12, (base - v // 2) * 1e-41, -1e-3 * base / v])
    x = x[:, torch.randperm(v, device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))]
    u = [0.1, 0.5, 0.9, 0.99]
    run_and_check(x, u, k=[1, 77, 9999, 19999])
    run_and_check(x, u, p=[0.2, 0.5, 0.9, 0.999])
    run_and_check(x, u, k=[5000, 12000, 19000, 3], p=[0.2, 0.5, 0.9, 0.999])


def test_the_draw_does_not_depend_on_the_batch(cuda):
    g = torch.Generator(device=cuda).manual_seed(11)
    x = rows_of(g, cuda, 40, 30011, BF, pad=5)
    u = torch.rand(40, device=cuda, generator=g)
    p = torch.full((40,), 0.9, device=cuda)
    whole = ops.sample(x, u, top_p=p)
    for r in (0, 17, 39):
        one = ops.sample(x[r: r + 1], u[r: r + 1], top_p=p[r: r + 1])
        assert all(torch.equal(a[r: r + 1], b) for a, b in zip(whole, one))


def test_frequencies(cuda):
    """Draws over a grid of u take each kept token as often as its share says."""
    x = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5]], device=cuda).repeat(4096, 1)
    u = (torch.arange(4096, device=cuda) + 0.5) / 4096
    token, logprob, kept = ops.sample(x, u.float(), top_k=torch.full((4096,), 4, dtype=I32, device=cuda))
    w = torch.softmax(x[0].double().index_fill(0, torch.tensor([2], device=cuda), -math.inf), -1)
    share = torch.bincount(token, minlength=5).double() / 4096
    assert (share - w).abs().max() <= 1.0 / 4096
    assert bool((kept == 4).all()) and (logprob.double() - w[token].log()).abs().max() <= 1e-6


def test_refusals(cuda):
    x, u = torch.randn(3, 100, device=cuda), torch.rand(3, device=cuda)
    with pytest.raises(TypeError):
        ops.sample(x.half(), u)
    with pytest.raises(ValueError):
        ops.sample(x.cpu(), u)
    with pytest.raises(ValueError):
        ops.sample(x.t(), u)
    with pytest.raises(ValueError):
        ops.sample(x, u[:2])
    with pytest.raises(ValueError):
        ops.sample(x, u.double())
    with pytest.raises(ValueError):
        ops.sample(x, u, top_k=torch.ones(3, device=cuda))
    with pytest.raises(ValueError):
        ops.sample(x, u, min_p=torch.ones(1, device=cuda))
    with pytest.raises(_lib.RldxError, match="at most"):
        ops.sample(torch.empty(1, 400000, device=cuda), u[:1])
    token, logprob, kept = ops.sample(x[:0], u[:0])
    assert token.shape == logprob.shape == kept.shape == (0,)
