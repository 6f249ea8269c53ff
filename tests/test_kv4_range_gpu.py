"""The 4-bit cache's attention over the rest of its range: batches of several launches, values of any size, rows
and pages that the host cannot see to be missing.  Plain forms and their tolerances: test_kv4_gpu.py."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from test_kv4_gpu import U, check_attention, cumulative, filled_cache, stored  # noqa: E402

BF, F64, I32 = torch.bfloat16, torch.float64, torch.int32


# ------------------------------------------------------------------------------------------------
# more sequences than one launch takes (1024)
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("seqs", [1024, 1025, 1043, 2050])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (24, 24, 64)])
@pytest.mark.parametrize("longest", [1000, 8192])  # of a launch that cuts no segment, and of one that may
def test_many_sequences(cuda, seqs, hq, hkv, d, longest):
    """The last launch holds a few sequences only: it keeps the plan of the first, with or without a workspace."""
    g = torch.Generator(device=cuda).manual_seed(seqs + d)
    lens = [(7 * b) % 41 for b in range(seqs)]
    lens[3], lens[-1] = 150, 150
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, 32, g, fill=0xFF)
    new = [min(1, n) for n in lens]
    q = torch.randn(sum(new), hq, d, device=cuda, generator=g).mul(1.5).to(BF)
    cu = cumulative(cuda, new)
    wide = torch.full((seqs, -(-longest // 32)), -1, dtype=I32, device=cuda)  # room for `longest` tokens a sequence
    wide[:, : table.shape[1]] = table[:, : wide.shape[1]]
    out = ops.kv4_attention(q, cache, wide, lengths, cu, max_new=1, max_len=longest)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    some = [b for b in range(seqs) if lens[b] and (b < 40 or b % 37 == 0 or b > 1000)]
    rows = cu[:-1][some].long()
    check_attention(q[rows], cache, table[some], lengths[some], cumulative(cuda, [1] * len(some)), out[rows])


# ------------------------------------------------------------------------------------------------
# values and weights of any size
# ------------------------------------------------------------------------------------------------
def cache_of(dev, k, v, d, page=64):
    """A cache of one sequence that holds k, v [n, heads, d] (k is normed per head on the way in)."""
    n, hkv = k.shape[0], k.shape[1]
    pages = -(-n // page)
    cache = ops.kv4_cache(pages, hkv, d, page, device=dev).fill_(0xFF)
    table, lengths = torch.arange(pages, dtype=I32, device=dev)[None], torch.tensor([n], dtype=I32, device=dev)
    one, cos, sin = torch.ones(d, device=dev).to(BF), torch.ones(1, d, device=dev), torch.zeros(1, d, device=dev)
    qkv = torch.cat([torch.zeros_like(k), k, v], 1).flatten(1).to(BF)
    ops.qkv_rope_append(qkv, one, one, cos, sin, torch.zeros(n, dtype=I32, device=dev), cache, table, lengths,
                        cumulative(dev, [n]), q_heads=hkv)
    return cache, table, lengths


def check_by_weights(q, cache, table, lengths, out, scale):
    """Every element of the rows q [new, heads, d] of one sequence, and the rows' norm.

    With w the softmax weights and B = sum_k w_k max_c |v_kc|, what the kernels round moves an element by no more than
      2^-8 |o|                   the output's rounding to bf16
      2 x 2^-11 x 2 B            p, and p scale or V rebuilt, to fp16 (numerator and sum; scale code <= 2 max |v|)
      2^-14 B                    fp32 scores, exponentials and sums
      2 x 2^-11 S B              K rebuilt to fp16 (chunks), S = sum_c |q_c k_c| scale, of the largest row
      2^-32 n w_max max |v|      fp16's last bits: p is held at 2^7 and more times the largest weight's 1
    """
    n, new = lengths.item(), q.shape[0]
    k, v = (stored(cache, table, 0, n, w) for w in (0, 1))
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("ihd,khd->ihk", q.to(F64), k) * scale
    hidden = torch.arange(n, device=q.device) > (n - new + torch.arange(new, device=q.device))[:, None, None]
    w = s.masked_fill(hidden, -math.inf).softmax(-1)
    ref = torch.einsum("ihk,khd->ihd", w, v)
    top = v.abs().amax(-1).t()  # [heads, keys]
    big = (w * top).sum(-1, keepdim=True)
    spread = torch.einsum("ihd,khd->ihk", q.to(F64).abs(), k.abs()).amax(-1, keepdim=True) * scale
    tol = U * ref.abs() + (2.0 ** -9 + 2.0 ** -14 + 2.0 ** -10 * spread) * big
    tol = tol + 2.0 ** -32 * n * w.amax(-1, keepdim=True) * top.amax(-1)[:, None]
    err = (out.to(F64) - ref).abs()
    assert bool((err <= tol).all()), ((err / tol).max().item(), (err.norm() / ref.norm()).item())
    return (err.norm() / ref.norm()).item()


@pytest.mark.parametrize("new", [1, 5, 300])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-4, 1e3])
def test_values_of_any_size(cuda, size, d, new):
    """V's scales from fp16's last bits to its thousands: the error stays what rounding the output makes it."""
    g = torch.Generator(device=cuda).manual_seed(d + new)
    n, hkv, hq = 4001, 2, 16
    k, v = (torch.randn(n, hkv, d, device=cuda, generator=g) for _ in range(2))
    cache, table, lengths = cache_of(cuda, k, v * size, d)
    q = torch.randn(new, hq, d, device=cuda, generator=g).mul(1.5).to(BF)
    out = ops.kv4_attention(q, cache, table, lengths, cumulative(cuda, [new]), max_new=new, max_len=n)
    # bf16's rounding alone is 2^-8 / sqrt(3) at most, in the mean over a row
    assert check_by_weights(q, cache, table, lengths, out, d ** -0.5) <= 2.0 ** -8


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_grow_along_the_sequence(cuda, d, new):
    """Sizes from 1e-4 to 1e3 in one sequence, up, down and mixed: the running power of two follows."""
    g = torch.Generator(device=cuda).manual_seed(d)
    n = 3000
    sizes = 10.0 ** torch.linspace(-4, 3, n, device=cuda)
    for order in (torch.arange(n), torch.arange(n).flip(0), torch.randperm(n, generator=torch.Generator().manual_seed(1))):
        k, v = (torch.randn(n, 2, d, device=cuda, generator=g) for _ in range(2))
        cache, table, lengths = cache_of(cuda, k, v * sizes[order.to(cuda)][:, None, None], d)
        q = torch.randn(new, 16, d, device=cuda, generator=g).to(BF)
        out = ops.kv4_attention(q, cache, table, lengths, cumulative(cuda, [new]), max_new=new, max_len=n)
        check_by_weights(q, cache, table, lengths, out, d ** -0.5)


@pytest.mark.parametrize("new", [1, 3, 300, 2000])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bits", [9.3, 17.3, 22.415, 24.415])
def test_small_weights_beside_a_large_one(cuda, bits, d, new):
    """The first token takes nearly all weight and holds zeros; the others, 2^-bits of its weight each, make the result."""
    g = torch.Generator(device=cuda).manual_seed(d)
    n, hkv, hq = 2000, 2, 16
    k = torch.randn(1, hkv, d, device=cuda, generator=g).expand(n, hkv, d).clone()
    k[0] = 1.0 - 2.0 * (torch.arange(d, device=cuda) % 2)
    v = 0.02 * (1.0 + 0.3 * torch.randn(n, hkv, d, device=cuda, generator=g))
    v[0] = 0.0
    cache, table, lengths = cache_of(cuda, k, v, d)
    q = k[0, 0].to(BF).expand(new, hq, d).contiguous()
    held = stored(cache, table, 0, n, 0)
    gap = torch.einsum("d,khd->kh", q[0, 0].to(F64), held[:2])
    scale = bits * math.log(2.0) / (gap[0] - gap[1]).min().item()  # one kv head at `bits`, the other a little past it
    out = ops.kv4_attention(q, cache, table, lengths, cumulative(cuda, [new]), max_new=new, max_len=n, scale=scale)
    check_by_weights(q, cache, table, lengths, out, torch.tensor(scale, dtype=torch.float32).item())


# ------------------------------------------------------------------------------------------------
# what only the device can see
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("new,old", [([1], [700]), ([4, 1], [500, 90]), ([300, 2], [1200, 10]), ([40] * 20, [100] * 20),
                                     ([2000], [0])])
@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("d", [64, 128])
def test_tokens_without_a_page_are_hidden(cuda, d, window, new, old):
    """Pages of the first sequence that its table does not name (-1, or past the pool) count for nothing, whichever kernel
    runs and whatever was read before: the other tokens' attention, and the code of the table."""
    g = torch.Generator(device=cuda).manual_seed(d + new[0])
    lens = [a + b for a, b in zip(new, old)]
    page, hq, hkv = 32, 16, 2
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, page, g, fill=0xFF, offset=8.0)
    held = -(-lens[0] // page)
    lost = sorted({0, 3, 4, held // 2, held - 2, held - 1} & set(range(held)))
    torn = table.clone()
    for i, p in enumerate(lost):
        torn[0, p] = -1 if i % 2 else cache.shape[0]
    q = torch.randn(sum(new), hq, d, device=cuda, generator=g).mul(1.5).to(BF)
    cu = cumulative(cuda, new)
    assert ops.device_error() == 0
    out = ops.kv4_attention(q, cache, torn, lengths, cu, max_new=max(new), max_len=max(lens), window=window)
    assert ops.device_error() == 0x500 and ops.device_error() == 0
    k, v = (stored(cache, table, 0, lens[0], w) for w in (0, 1))
    key = torch.arange(lens[0], device=cuda)
    there = ~torch.isin(key // page, torch.tensor(lost, device=cuda))
    rows = [i for i in range(new[0]) if i < 40 or i % 29 == 0]
    pos = old[0] + torch.tensor(rows, device=cuda)[:, None]
    seen = there & (key <= pos) & ((pos - key < window) if window else True)
    s = torch.einsum("ihd,khd->ihk", q[rows].to(F64), k.repeat_interleave(hq // hkv, 1)) * d ** -0.5
    w = s.masked_fill(~seen[:, None], -math.inf).softmax(-1).nan_to_num(0.0)  # no token left: zeros
    ref = torch.einsum("ihk,khd->ihd", w, v.repeat_interleave(hq // hkv, 1))
    # as check_attention's: the output's bf16, fp16 of p and of p scale or V, K in fp16, against the largest value
    tol = U * ref.abs() + 2.0 ** -9 * v.abs().max()
    assert bool(((out[rows].to(F64) - ref).abs() <= tol).all()), (out[rows].to(F64) - ref).abs().max().item()
    if len(new) > 1:  # the other sequences have all their pages
        some = list(range(1, len(new)))
        last = cu[1:].long()[some] - 1
        check_attention(q[last], cache, table[some], lengths[some], cumulative(cuda, [1] * len(some)), out[last], window)


@pytest.mark.parametrize("new,old,max_new,max_len", [
    ([1, 1, 0, 1, 1], [40, 700, 3, 90, 5], 1, 100),  # the second is longer than the call says
    ([3, 7, 0, 2], [40, 20, 3, 90], 4, 100),         # the second has more new tokens
    ([40, 300, 17, 600], [500, 20, 33, 0], 300, 545),  # chunks, the last breaks both
    ([300, 2100], [100, 0], 300, 3000),              # chunks whose keys are shared out
])
def test_rows_that_get_no_attention_are_zero(cuda, new, old, max_new, max_len):
    """Rows of a sequence that breaks the call's bounds (0x502), and rows before the first or past the last sequence's."""
    g = torch.Generator(device=cuda).manual_seed(sum(new))
    d, lens, head, tail = 128, [a + b for a, b in zip(new, old)], 3, 5
    cache, table, lengths = filled_cache(cuda, lens, 2, d, 64, g, fill=0xFF)
    cu = cumulative(cuda, new) + head
    q = torch.randn(head + sum(new) + tail, 16, d, device=cuda, generator=g).to(BF)
    out = torch.full_like(q, math.nan)
    ops.kv4_attention(q, cache, table, lengths, cu, max_new=max_new, max_len=max_len, out=out)
    assert ops.device_error() == 0x502 and ops.device_error() == 0
    assert bool((out[:head] == 0).all()) and bool((out[-tail:] == 0).all())
    for b, (n, length) in enumerate(zip(new, lens)):
        rows = slice(cu[b].item(), cu[b + 1].item())
        if n > max_new or length > max_len:
            assert bool((out[rows] == 0).all()), b
        elif n:
            assert not bool(torch.isnan(out[rows].float()).any()), b
            last = rows.stop - 1
            check_attention(q[last: last + 1], cache, table[b: b + 1], lengths[b: b + 1], cumulative(cuda, [1]), out[last: last + 1])


def test_rows_outside_every_launch(cuda):
    """Batches of several launches: the rows around them are zeroed once, those between are not."""
    g = torch.Generator(device=cuda).manual_seed(1)
    seqs = 1030
    lens = [1 + b % 9 for b in range(seqs)]
    cache, table, lengths = filled_cache(cuda, lens, 2, 64, 32, g)
    cu = cumulative(cuda, [1] * seqs) + 2
    q = torch.randn(seqs + 6, 16, 64, device=cuda, generator=g).to(BF)
    out = torch.full_like(q, math.nan)
    ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=9, out=out)
    assert ops.device_error() == 0
    assert bool((out[:2] == 0).all()) and bool((out[-4:] == 0).all())
    check_attention(q[2:-4], cache, table, lengths, cumulative(cuda, [1] * seqs), out[2:-4])


@pytest.mark.parametrize("seqs", [2, 1030])
def test_append_stores_rows_of_sequences_only(cuda, seqs):
    """Rows before the first sequence's and past the last one's change no byte of the cache, where there is a page too."""
    g = torch.Generator(device=cuda).manual_seed(2)
    d, hkv, lens = 64, 2, [20] * seqs
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, 32, g)
    one, cos, sin = torch.ones(d, device=cuda).to(BF), torch.ones(1, d, device=cuda), torch.zeros(1, d, device=cuda)
    lengths = lengths + 1  # one new token each, of pages that have room
    plain, want = cache.clone(), None
    qkv = torch.randn(seqs + 7, 3 * hkv * d, device=cuda, generator=g).to(BF)

    def append(pool, rows, cu):
        return ops.qkv_rope_append(rows, one, one, cos, sin, torch.zeros(rows.shape[0], dtype=I32, device=cuda), pool, table,
                                   lengths, cu, q_heads=hkv)

    want = append(plain, qkv[3:-4], cumulative(cuda, [1] * seqs))
    assert ops.device_error() == 0
    q = append(cache, qkv, cumulative(cuda, [1] * seqs) + 3)
    assert ops.device_error() == 0x502 and ops.device_error() == 0
    assert torch.equal(cache, plain) and torch.equal(q[3:-4], want)
    k, v = ops.kv4_read(cache, table, lengths, cumulative(cuda, [1] * seqs) + 3, tokens=seqs + 7)
    assert ops.device_error() == 0x502 and ops.device_error() == 0
    assert not bool(k[:3].any()) and not bool(k[-4:].any()) and not bool(v[-4:].any()) and bool(k[3:-4].any(2).all())


def test_launches_of_few_sequences_where_lengths_may_be_huge(cuda):
    """A max_len of 368 million tokens leaves two sequences to a launch, whose sums are 32-bit."""
    g = torch.Generator(device=cuda).manual_seed(3)
    new, old = [20, 1, 3, 20, 7], [100, 0, 3000, 12, 1]
    lens = [a + b for a, b in zip(new, old)]
    cache, table, lengths = filled_cache(cuda, lens, 24, 64, 32, g, fill=0xFF)
    wide = torch.full((5, 11_500_000), -1, dtype=I32, device=cuda)
    wide[:, : table.shape[1]] = table
    q = torch.randn(sum(new), 24, 64, device=cuda, generator=g).mul(1.5).to(BF)
    cu = cumulative(cuda, new)
    out = ops.kv4_attention(q, cache, wide, lengths, cu, max_new=20, max_len=wide.shape[1] * 32)
    assert ops.device_error() == 0
    check_attention(q, cache, table, lengths, cu, out)


@pytest.mark.parametrize("new,hidden", [(6, 4), (90, 40), (600, 130)])
@pytest.mark.parametrize("window", [999, 1000, 1001, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 3])
def test_windows_as_long_as_the_sequence_and_longer(cuda, new, hidden, window, sinks):
    """Such a window hides nothing, with rows before position 0 too (whose positions less the window pass 32 bits)."""
    g = torch.Generator(device=cuda).manual_seed(8)
    cache, table, _ = filled_cache(cuda, [1000], 2, 128, 64, g)
    lengths = torch.tensor([new - hidden], dtype=I32, device=cuda)
    q = torch.randn(new, 16, 128, device=cuda, generator=g).to(BF)
    cu = cumulative(cuda, [new])
    out = ops.kv4_attention(q, cache, table, lengths, cu, max_new=new, max_len=1000, window=window, sinks=sinks)
    want = ops.kv4_attention(q, cache, table, lengths, cu, max_new=new, max_len=1000)
    assert bool((out[:hidden] == 0).all()) and ops.device_error() == 0
    # 999 still runs as a window, whose units may be split in other places
    assert torch.equal(out, want) or (window == 999 and (out.float() - want.float()).abs().max() <= 2.0 ** -6)
