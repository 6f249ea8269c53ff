"""Log probabilities of given tokens against a plain 64-bit form; ranks and alternatives have to be equal.

Roundings, in units of 2^-24: with D the mean of |d| under the distribution and D2 that of its square, a weight is off by
3 |d| (the difference, the product with log2 e and that constant) and 4 of the exponential unit, and the sum by 8 (a vector) +
8 (a thread's vectors) + chunks of a row (one each, at most 25 here) + 13 (the tree) + 5 a move of the reference, at
most 25: 180 in all covers it.  ln S is off by that, and T / S by it times D with 3 D2 more; the results' own
roundings are a few units of their size."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def check(logits, tokens, top):
    lp, entropy, rank, ids, values = ops.token_logprobs(logits, tokens, top=top)
    rows, vocab = logits.shape
    assert lp.shape == entropy.shape == rank.shape == (rows,) and ids.shape == values.shape == (rows, top)
    assert (lp.dtype, entropy.dtype, rank.dtype, ids.dtype, values.dtype) == (F32, F32, torch.int32, torch.int64, F32)
    x = logits.double() + 0.0
    m = x.amax(1, keepdim=True)
    good = torch.isfinite(m[:, 0]) & ~torch.isnan(x).any(1)
    nan = torch.full_like(m[:, 0], math.nan)
    p = torch.softmax(x, 1)
    d = torch.where(p > 0, x - m, torch.zeros_like(x))
    logs = x - m - (x - m).exp().sum(1, keepdim=True).log()
    mean, square = (p * d.abs()).sum(1), (p * d * d).sum(1)
    off = 2.0 ** -24 * (180 + 3 * mean)
    want_h = -(p * torch.where(p > 0, logs, torch.zeros_like(logs))).sum(1)

    def close(got, want, room):
        want, room = want.double(), room + want.double().abs() * 2.0 ** -22
        same = torch.isnan(got) & torch.isnan(want) | (got == want.float())  # (2 max below 0 is -inf in fp32)
        assert bool((same | ((got.double() - want).abs() <= room)).all()), (got.double() - want).abs().max()

    close(entropy, torch.where(good, want_h, nan), off * (1 + mean) + 3 * 2.0 ** -24 * square)
    given = tokens >= 0
    at = tokens.clamp_min(0).unsqueeze(1)
    mine = x.gather(1, at)
    want = torch.where(good, logs.gather(1, at)[:, 0], nan)
    close(lp, torch.where(given, want, torch.zeros_like(want)), off + 2.0 ** -23 * (mine - m)[:, 0].abs().nan_to_num(0, 0, 0))
    order = torch.arange(vocab, device=x.device)
    want_rank = ((x > mine) | ((x == mine) & (order < at))).sum(1)
    assert torch.equal(rank.long(), torch.where(given & good, want_rank, torch.full_like(want_rank, -1)))
    if top:
        by = torch.sort(x, dim=1, descending=True, stable=True)
        assert torch.equal(ids, torch.where(good.unsqueeze(1), by.indices[:, :top], torch.full_like(ids, -1)))
        best = torch.where(good.unsqueeze(1), logs.gather(1, by.indices[:, :top]), nan.unsqueeze(1))
        close(values, best, off.unsqueeze(1) + 2.0 ** -23 * (by.values[:, :top] - m).abs().nan_to_num(0, 0, 0))
    return lp, entropy, rank, ids, values


def rows_of(g, dev, rows, vocab, dtype, spread=2.0, pad=0, shift=0):
    x = torch.empty(rows, vocab + pad + shift, dtype=dtype, device=dev)[:, shift: shift + vocab]
    x.copy_(spread * torch.randn(rows, vocab, device=dev, generator=g) - 3.0)
    return x


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("vocab,pad,shift", [(1, 0, 0), (5, 2, 1), (33, 0, 3), (1000, 0, 0), (2049, 3, 5), (4097, 1, 0), (32003, 0, 1), (50257, 7, 0),
                                             (151680, 0, 0)])
def test_sizes(cuda, dtype, vocab, pad, shift):
    g = torch.Generator(device=cuda).manual_seed(vocab + pad)
    for rows in (1, 9):
        x = rows_of(g, cuda, rows, vocab, dtype, pad=pad, shift=shift)
        tokens = torch.randint(-1, vocab, (rows,), device=cuda, generator=g)
        for top in {0, 1, min(5, vocab), min(32, vocab)}:
            check(x, tokens, top)


@pytest.mark.parametrize("dtype,vocab,rows", [(BF, 4096, 700), (F32, 1500, 600), (F16, 20011, 450), (BF, 32003, 60), (F32, 151680, 500)])
def test_many_rows(cuda, dtype, vocab, rows):
    """Rows of one CTA, of two and more."""
    g = torch.Generator(device=cuda).manual_seed(rows)
    x = rows_of(g, cuda, rows, vocab, dtype, spread=4.0)
    tokens = torch.randint(vocab, (rows,), device=cuda, generator=g)
    whole = check(x, tokens, 20)
    for r in (0, rows // 2, rows - 1):  # ranks and alternatives are the same in every batch
        one = ops.token_logprobs(x[r: r + 1], tokens[r: r + 1], top=20)
        assert all(torch.equal(a[r: r + 1], b) for a, b in zip(whole[2:4], one[2:4]))


@pytest.mark.parametrize("dtype,vocab,shift,rows", [
    (F32, 511, 0, 5), (F32, 512, 0, 5), (F32, 1023, 1, 5), (F32, 1024, 0, 5), (BF, 4096, 0, 592), (BF, 4096, 0, 593), (BF, 4091, 3, 1184),
    (F16, 4096, 0, 1185), (F16, 8191, 5, 1185), (BF, 4104, 0, 2368), (BF, 8191, 1, 2369), (F32, 16384, 0, 1200), (F32, 16388, 0, 1200)])
def test_threads_of_a_row(cuda, dtype, vocab, shift, rows):
    """The sizes at which a row goes to 64, 128 or 256 threads, from both sides, with rows of each awkward kind among the others."""
    g = torch.Generator(device=cuda).manual_seed(rows + vocab)
    x = rows_of(g, cuda, rows, vocab, dtype, spread=3.0, shift=shift)
    n = torch.arange(vocab, device=cuda).float()
    for first in {0, rows - 5}:
        x[first] = 1.25
        x[first + 1] = 30 * n / vocab
        x[first + 2, : vocab * 9 // 10] = -math.inf
        x[first + 3] = torch.finfo(dtype).min
        x[first + 4] = (x[first + 4].float() * 2).round()
    if rows > 20:
        x[rows // 2] = -math.inf
        x[rows // 2 + 1, vocab - 1] = math.nan
    tokens = torch.randint(-1, vocab, (rows,), device=cuda, generator=g)
    for top in (0, 1, 32):
        check(x, tokens, top)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("vocab", [40, 3001, 40000, 151680])
@pytest.mark.parametrize("rows", [12, 480])
def test_ties_masks_and_orders(cuda, dtype, vocab, rows):
    """Equal logits, a few values only, ascending and descending rows, masks of -inf and of the type's lowest value: in front,
    behind, everywhere but a few tokens."""
    if rows * vocab > 2 ** 25:
        rows = 2 ** 25 // vocab
    g = torch.Generator(device=cuda).manual_seed(vocab)
    low = torch.finfo(dtype).min
    x = torch.randn(rows, vocab, device=cuda, generator=g)
    n = torch.arange(vocab, device=cuda).float()
    x[0] = 1.25
    x[1] = (x[1] * 2).round()
    x[2] = 30 * n / vocab
    x[3] = -30 * n / vocab
    x[4, : vocab * 9 // 10] = -math.inf
    x[5, vocab // 10:] = -math.inf
    x[6] = -math.inf
    x[6, vocab // 2], x[6, vocab - 1] = 2.0, -0.0
    x[7] = low
    x[8, 3:] = low
    x[9] = 0.0
    x[9, ::3] = -0.0
    x[10, : vocab // 2] = 5.0
    x[11] = torch.where(n % 7 == 3, 2.0, -1.0)
    x[12:] = (x[12:] * 3).round() / 2
    x = x.to(dtype)
    tokens = torch.randint(vocab, (rows,), device=cuda, generator=g)
    tokens[6] = vocab // 2
    for top in (1, 7, 32):
        check(x, tokens, top)
    check(x, torch.zeros_like(tokens), 32)
    check(x, torch.full_like(tokens, vocab - 1), 0)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_special_rows(cuda, dtype):
    """NaN, infinities, rows that a mask empties, logits of a type's whole range."""
    vocab, big = 9001, torch.finfo(dtype).max
    x = torch.randn(10, vocab, device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    x[0] = -math.inf
    x[1, 77] = math.nan
    x[2, 9000] = math.inf
    x[3] = math.nan
    x[4, 1:] = -math.inf
    x[5] = -big
    x[5, 5] = big
    x[6] = big
    x[7] = -big
    x[7, 100:] = -math.inf
    x[8] = 3e4
    x = x.to(dtype)
    for t in (0, 5, 9000):
        lp, entropy, rank, ids, values = check(x, torch.full((10,), t, device=cuda), 32)
        assert bool(torch.isnan(entropy[:4]).all()) and bool((rank[:4] == -1).all()) and bool((ids[:4] == -1).all())
    assert entropy[4] == 0 and values[4, 0] == 0 and bool((values[4, 1:] == -math.inf).all())
    assert entropy[5] == 0 and abs(float(entropy[6]) - math.log(vocab)) <= 2.0 ** -24 * 200


def test_tokens_that_are_none_or_outside(cuda):
    x = torch.randn(5, 300, device=cuda)
    tokens = torch.tensor([-1, 3, -100, 299, -(2 ** 40)], device=cuda)
    lp, _, rank, _, _ = check(x, tokens, 3)
    assert lp[[0, 2, 4]].tolist() == [0, 0, 0] and rank[[0, 2, 4]].tolist() == [-1, -1, -1]
    assert ops.device_error() == 0
    tokens = torch.tensor([300, 3, 2 ** 40, 299, 4], device=cuda)
    lp, entropy, rank, ids, _ = ops.token_logprobs(x, tokens, top=2)
    assert torch.isnan(lp).tolist() == [True, False, True, False, False] and rank[[0, 2]].tolist() == [-1, -1]
    assert bool(torch.isfinite(entropy).all()) and bool((ids >= 0).all())
    assert ops.device_error() == 0x503 and ops.device_error() == 0


def test_broadcast_rows_and_no_rows(cuda):
    x = torch.randn(1, 500, device=cuda)
    tokens = torch.arange(40, device=cuda)
    lp = check(x.expand(40, -1), tokens, 4)[0]
    # sums over every token: probabilities add up to one
    every = ops.token_logprobs(x.expand(500, -1), torch.arange(500, device=cuda))[0]
    assert abs(float(every.double().exp().sum()) - 1) <= 200 * 2.0 ** -24 and torch.equal(every[:40], lp)
    out = ops.token_logprobs(x[:0], tokens[:0], top=3)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0,), (0, 3), (0, 3)]


def test_captured_and_on_another_stream(cuda):
    g = torch.Generator(device=cuda).manual_seed(8)
    x = rows_of(g, cuda, 6, 60000, BF)
    tokens = torch.randint(60000, (6,), device=cuda, generator=g)
    want = ops.token_logprobs(x, tokens, top=9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        here = ops.token_logprobs(x, tokens, top=9)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(here, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.token_logprobs(x, tokens, top=9)
    x.copy_(rows_of(g, cuda, 6, 60000, BF))
    tokens += 1
    tokens %= 60000
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, ops.token_logprobs(x, tokens, top=9)))


def test_offsets_past_32_bits(cuda):
    buffer = torch.empty(5 * 10 ** 8 * 5 + 5000, dtype=BF, device=cuda)
    x = buffer.as_strided((6, 5000), (5 * 10 ** 8, 1))
    x.copy_(torch.randn(6, 5000, device=cuda))
    check(x, torch.arange(6, device=cuda) * 900, 6)
