"""The 4-bit cache operators against plain 64-bit implementations: qkv_rope_append (RMSNorm, RoPE,
quantised write), kv4_read and kv4_attention.

The plain forms here find a token's codes by the description of the unit's layout, one element at a
time in index arithmetic.  Tolerances: a bf16 result is within half an ulp (U = eps / 2 = 2^-8) of its
fp32 value; a stored value is within half a step of its input plus the rounding of scale and low
(fp16, 2^-11 of the range's ends each); attention adds p's rounding to fp16 (2^-11) and p scale's
(2^-11) to the output's rounding, against the largest value it averages."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import _lib, ops  # noqa: E402

BF, F64, I32 = torch.bfloat16, torch.float64, torch.int32
U = torch.finfo(BF).eps / 2


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def stored(cache, table, b, length, which):
    """[length, Hkv, d] values in 64 bits of sequence b's tokens (which: 0 K, 1 V)."""
    d = cache.shape[3] // 40
    page = cache.shape[2] * 32
    G = d // 32
    dev = cache.device
    j = torch.arange(length, device=dev)
    units = cache[table[b, j // page].long(), :, j % page // 32]  # [n, Hkv, 40 d]
    tau = (j % 32).view(-1, 1, 1)
    c = torch.arange(d, device=dev).view(1, 1, -1)
    grp = c // 32
    blk, h, t, e = tau // 16, tau // 8 % 2, tau // 2 % 4, tau % 2
    if which == 0:
        word = c % 32 // 8
        byte = tau * (d // 2) + 4 * (word * G + grp) + c % 8 // 2
        scale = 32 * d + 4 * G * tau + 2 * grp
        low = scale + 2 * G
    else:
        g = c % 32 // 4
        byte = 16 * d + 8 * d * blk + 4 * d * h + 4 * G * (4 * g + t) + 2 * G * e + 2 * grp + c % 4 // 2
        scale = 32 * d + 128 * G + 32 * G * blk + 16 * G * h + 4 * G * t + 4 * grp + 2 * e
        low = scale + 64 * G

    def gather(at):
        return units.gather(2, at.expand(units.shape[0], units.shape[1], d)).long()

    def fp16(at):
        return (gather(at) | gather(at + 1) << 8).to(torch.int32).to(torch.int16).view(torch.float16).to(F64)

    code = gather(byte) >> 4 * (c % 2) & 15
    return fp16(scale) * code + fp16(low)


def reference_attention(q, cache, table, lengths, cu, window, sinks, scale):
    out = torch.zeros(q.shape, dtype=F64, device=q.device)
    for b, length in enumerate(lengths.tolist()):
        r0, r1 = cu[b].item(), cu[b + 1].item()
        if r1 == r0 or length == 0:
            continue
        k, v = (stored(cache, table, b, length, w) for w in (0, 1))
        group = q.shape[1] // k.shape[1]
        j = torch.arange(length, device=q.device)
        for i in range(r0, r1):
            p = length - (r1 - i)
            ok = j <= p
            if window:
                ok &= (j > p - window) | (j < sinks)
            if not bool(ok.any()):
                continue
            kk, vv = k[ok].repeat_interleave(group, 1), v[ok].repeat_interleave(group, 1)
            w = torch.softmax(torch.einsum("hd,khd->hk", q[i].to(F64), kk) * scale, -1)
            out[i] = torch.einsum("hk,khd->hd", w, vv)
    return out


def make_tables(dev, lens, page, g, extra=2, spare_pages=3):
    held = [-(-n // page) for n in lens]
    pages = sum(held) + spare_pages
    order = torch.randperm(pages, device=dev, generator=g).to(I32)
    table = torch.full((len(lens), max(held) + extra), -1, dtype=I32, device=dev)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at: at + n]
        at += n
    return table, pages


def cumulative(dev, new):
    return torch.tensor([0] + list(new), device=dev).cumsum(0).to(I32)


def filled_cache(dev, lens, hkv, d, page, g, fill=None, offset=1.0):
    """A cache that holds random tokens, written by the append operator itself; unwritten bytes are
    `fill`."""
    table, pages = make_tables(dev, lens, page, g)
    cache = ops.kv4_cache(pages, hkv, d, page, device=dev)
    cache.fill_(0 if fill is None else fill)
    t = sum(lens)
    qkv = torch.randn(t, 3 * hkv * d, device=dev, generator=g)
    qkv[:, 2 * hkv * d:] += offset * torch.randn(hkv * d, device=dev, generator=g)
    one, cos, sin = torch.ones(d, device=dev).to(BF), torch.ones(1, d, device=dev), torch.zeros(1, d, device=dev)
    lengths = torch.tensor(lens, dtype=I32, device=dev)
    ops.qkv_rope_append(qkv.to(BF), one, one, cos, sin, torch.zeros(t, dtype=I32, device=dev), cache, table, lengths,
                        cumulative(dev, lens), q_heads=hkv)
    return cache, table, lengths


def check_attention(q, cache, table, lengths, cu, out, window=0, sinks=0, scale=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    ref = reference_attention(q, cache, table, lengths, cu, window, sinks, scale)
    biggest = max([1e-30] + [stored(cache, table, b, n, 1).abs().max().item() for b, n in enumerate(lengths.tolist()) if n])
    # bf16 of the result, fp16 of p, fp16 of p scale, fp32 sums and exponentials
    tol = 2.0 ** -9 * ref.abs() + (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -16) * 2 * biggest
    assert bool(((out.to(F64) - ref).abs() <= tol).all()), (out.to(F64) - ref).abs().max().item()
    err = (out.to(F64) - ref).norm() / ref.norm().clamp_min(1e-30)
    assert err <= 2.0 ** -8 or ref.norm() == 0


# ------------------------------------------------------------------------------------------------
# append and read
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rope", [torch.float32, BF])
@pytest.mark.parametrize("hq,hkv,d,page", [(16, 2, 128, 64), (24, 24, 64, 32), (6, 3, 128, 96), (5, 1, 64, 128), (8, 8, 128, 32)])
@pytest.mark.parametrize("new,old", [([1], [0]), ([1, 1, 1], [63, 64, 31]), ([5, 0, 33, 2], [0, 7, 95, 1000])])
def test_append_and_read(cuda, hq, hkv, d, page, new, old, rope):
    g = torch.Generator(device=cuda).manual_seed(hq * 100 + d + sum(new))
    lens = [a + b for a, b in zip(new, old)]
    t = sum(new)
    table, pages = make_tables(cuda, lens, page, g)
    cache = ops.kv4_cache(pages, hkv, d, page, device=cuda).fill_(0xA5)
    before = cache.clone()
    wide = torch.randn(t, (hq + 2 * hkv) * d + 24, device=cuda, generator=g).mul(2.0).to(BF)
    qkv = wide[:, 8: 8 + (hq + 2 * hkv) * d]  # a view with a row stride
    qn, kn = ((1 + 0.2 * torch.randn(d, device=cuda, generator=g)).to(BF) for _ in range(2))
    ang = torch.outer(torch.arange(1200, device=cuda).float(), 1e4 ** (-torch.arange(0, d, 2, device=cuda).float() / d))
    cos, sin = (torch.cat([f, f], -1).to(rope) for f in (ang.cos(), ang.sin()))
    pos = torch.randint(0, 1200, (t,), device=cuda, generator=g).to(I32)
    lengths, cu = torch.tensor(lens, dtype=I32, device=cuda), cumulative(cuda, new)
    q = ops.qkv_rope_append(qkv, qn, kn, cos, sin, pos, cache, table, lengths, cu, q_heads=hq)
    k, v = ops.kv4_read(cache, table, lengths, cu, tokens=t)
    torch.cuda.synchronize()
    assert ops.device_error() == 0

    x = qkv.to(F64).reshape(t, hq + 2 * hkv, d)
    w = torch.cat([qn.to(F64).expand(hq, d), kn.to(F64).expand(hkv, d)])
    y = x[:, : hq + hkv]
    y = y * torch.rsqrt(y.pow(2).mean(-1, keepdim=True) + 1e-6) * w
    half = torch.cat([-y[..., d // 2:], y[..., : d // 2]], -1)
    y = y * cos.to(F64)[pos.long()][:, None] + half * sin.to(F64)[pos.long()][:, None]
    # fp32 arithmetic, then bf16
    assert bool(((q.to(F64) - y[:, :hq]).abs() <= U * y[:, :hq].abs() + 2.0 ** -20 * y[:, :hq].abs().amax(-1, keepdim=True)).all())
    for got, want in ((k, y[:, hq:]), (v, x[:, hq + hkv:])):
        grp = want.reshape(t, hkv, d // 32, 32)
        top, low = grp.amax(-1, keepdim=True), grp.amin(-1, keepdim=True)
        step = (top - low) / 15
        # half a step (a little wider after rounding), the ends lost to low's and scale's fp16, bf16
        ends = 2.0 ** -11 * (low.abs() + 15 * step) + 2.0 ** -24 * 16
        tol = (0.5 * step * (1 + 2.0 ** -10) + ends + U * (grp.abs() + step)).reshape(want.shape)
        assert bool(((got.to(F64) - want).abs() <= tol).all())
    # the cache holds, by its layout, what kv4_read returned, and nothing else changed
    used = torch.zeros_like(cache, dtype=torch.bool)
    for b, (n, length) in enumerate(zip(new, lens)):
        if not n:
            continue
        rows = slice(cu[b].item(), cu[b + 1].item())
        for which, got in ((0, k), (1, v)):
            held = stored(cache, table, b, length, which)[length - n:]
            assert bool(((got[rows].to(F64) - held).abs() <= U * held.abs() + 1e-30).all())
        p = torch.arange(length - n, length, device=cuda)
        used[table[b, p // page].long(), :, p % page // 32] = True  # units touched
    assert torch.equal(cache[~used], before[~used])


def test_append_leaves_neighbours_alone(cuda):
    """A second append into the same unit changes its own token's bytes only."""
    g = torch.Generator(device=cuda).manual_seed(3)
    d, hkv, n = 128, 2, 32
    cache, table, lengths = filled_cache(cuda, [n], hkv, d, 32, g)
    k0, v0 = (stored(cache, table, 0, n, w) for w in (0, 1))
    for tau in (0, 1, 7, 8, 17, 31):
        one = torch.ones(d, device=cuda).to(BF)
        qkv = torch.randn(1, 3 * hkv * d, device=cuda, generator=g).to(BF)
        ops.qkv_rope_append(qkv, one, one, torch.ones(1, d, device=cuda), torch.zeros(1, d, device=cuda),
                            torch.zeros(1, dtype=I32, device=cuda), cache, table,
                            torch.tensor([tau + 1], dtype=I32, device=cuda), cumulative(cuda, [1]), q_heads=hkv)
        for which, old in ((0, k0), (1, v0)):
            now = stored(cache, table, 0, n, which)
            same = torch.arange(n, device=cuda) != tau
            assert torch.equal(now[same], old[same])
            assert not torch.equal(now[tau], old[tau])
            old.copy_(now)


def test_append_special_values(cuda):
    """Constant groups, zeros, infinities (saturate) and NaN (stays in its group)."""
    d, hkv = 64, 1
    table = torch.zeros(1, 1, dtype=I32, device=cuda)
    cache = ops.kv4_cache(1, hkv, d, 32, device=cuda)
    v = torch.zeros(4, d, device=cuda)
    v[0] = 3.0
    v[1, 5] = math.inf
    v[2, 40] = math.nan
    v[3, :32] = torch.linspace(-7.5, 7.5, 32, device=cuda)
    qkv = torch.cat([torch.ones(4, 2 * d, device=cuda), v], 1).to(BF)
    one = torch.ones(d, device=cuda).to(BF)
    cu = cumulative(cuda, [4])
    lengths = torch.tensor([4], dtype=I32, device=cuda)
    ops.qkv_rope_append(qkv, one, one, torch.ones(1, d, device=cuda), torch.zeros(1, d, device=cuda),
                        torch.zeros(4, dtype=I32, device=cuda), cache, table, lengths, cu, q_heads=1)
    k, got = ops.kv4_read(cache, table, lengths, cu, tokens=4)
    got = got[:, 0].float()
    assert bool((got[0] == 3.0).all())
    assert got[1, 5] > 6e4 and bool((got[1, 32:] == 0).all()) and bool(torch.isfinite(got[1]).all())
    assert bool(torch.isnan(got[2, 32:]).all()) and bool((got[2, :32] == 0).all())
    assert (got[3, :32] - v[3, :32]).abs().max() <= 0.5 + 2 ** -5
    assert bool(torch.isfinite(k.float()).all())


# ------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------
HEADS = [(16, 2, 128, 64), (24, 24, 64, 32), (6, 2, 128, 96), (8, 1, 64, 64), (32, 2, 64, 128), (40, 2, 128, 64)]


@pytest.mark.parametrize("hq,hkv,d,page", HEADS)
@pytest.mark.parametrize("lens", [[1], [33, 0, 7, 64], [300, 2, 95, 96, 97], [2111]])
def test_single_tokens(cuda, hq, hkv, d, page, lens):
    g = torch.Generator(device=cuda).manual_seed(hq + d + sum(lens))
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, page, g, fill=0xFF)
    new = [min(1, n) for n in lens]
    q = torch.randn(sum(new), hq, d, device=cuda, generator=g).mul(1.5).to(BF)
    cu = cumulative(cuda, new)
    out = ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=max(lens))
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    check_attention(q, cache, table, lengths, cu, out)


@pytest.mark.parametrize("hq,hkv,d,page", HEADS)
@pytest.mark.parametrize("new,old", [([2, 3], [0, 40]), ([5, 1, 0, 8], [90, 0, 12, 1]), ([33], [200]), ([70, 9], [0, 131])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (17, 3), (64, 40)])
def test_chunks(cuda, hq, hkv, d, page, new, old, window, sinks):
    g = torch.Generator(device=cuda).manual_seed(hq + d + sum(new) + window)
    lens = [a + b for a, b in zip(new, old)]
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, page, g, fill=0xFF)
    wide = torch.randn(sum(new), hq * d + 16, device=cuda, generator=g).mul(1.5).to(BF)
    q = wide[:, : hq * d].unflatten(1, (hq, d))  # a token stride of its own
    cu = cumulative(cuda, new)
    out = ops.kv4_attention(q, cache, table, lengths, cu, max_new=max(new), max_len=max(lens) + 50, window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    check_attention(q, cache, table, lengths, cu, out, window, sinks)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1000, 0), (1000, 5), (129, 200), (5000, 4)])
@pytest.mark.parametrize("d", [64, 128])
def test_long_lengths(cuda, d, window, sinks):
    """More units than one split holds, few sequences: the split over the length and its join."""
    g = torch.Generator(device=cuda).manual_seed(d + window)
    lens = [9001, 12, 4097]
    cache, table, lengths = filled_cache(cuda, lens, 2, d, 64, g, fill=0xFF)
    q = torch.randn(3, 16, d, device=cuda, generator=g).mul(1.5).to(BF)
    cu = cumulative(cuda, [1, 1, 1])
    out = ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=9001, window=window, sinks=sinks)
    again = ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=9001, window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert torch.equal(out, again)  # the join has one order
    check_attention(q, cache, table, lengths, cu, out, window, sinks)


@pytest.mark.parametrize("new", [1, 4, 40])
def test_row_without_keys_is_zero(cuda, new):
    """lengths says fewer tokens than there are new rows: the rows before position 0 see nothing."""
    g = torch.Generator(device=cuda).manual_seed(new)
    cache, table, _ = filled_cache(cuda, [64], 2, 128, 64, g)
    lengths = torch.tensor([new - 1], dtype=I32, device=cuda)
    q = torch.randn(new, 16, 128, device=cuda, generator=g).to(BF)
    out = ops.kv4_attention(q, cache, table, lengths, cumulative(cuda, [new]), max_new=new, max_len=64)
    assert bool((out[0] == 0).all())
    if new > 1:
        ref = reference_attention(q[1:], cache, table, lengths, cumulative(cuda, [new - 1]), 0, 0, 128 ** -0.5)
        assert (out[1:].to(F64) - ref).abs().max() <= 2.0 ** -8 * ref.abs().max()


@pytest.mark.parametrize("new", [6, 40])
def test_nan_of_a_hidden_token_stays_hidden(cuda, new):
    """NaN in K and V of one token reaches the rows that see it and no other."""
    g = torch.Generator(device=cuda).manual_seed(9 + new)
    d, hkv, n, bad = 128, 2, 100, 100 - new + 3
    cache, table, lengths = filled_cache(cuda, [n], hkv, d, 64, g, fill=0xFF)
    qkv = torch.full((1, 3 * hkv * d), math.nan, device=cuda).to(BF)
    one = torch.ones(d, device=cuda).to(BF)
    ops.qkv_rope_append(qkv, one, one, torch.ones(1, d, device=cuda), torch.zeros(1, d, device=cuda),
                        torch.zeros(1, dtype=I32, device=cuda), cache, table,
                        torch.tensor([bad + 1], dtype=I32, device=cuda), cumulative(cuda, [1]), q_heads=hkv)
    q = torch.randn(new, 16, d, device=cuda, generator=g).to(BF)
    for window in (0, 2):
        out = ops.kv4_attention(q, cache, table, lengths, cumulative(cuda, [new]), max_new=new, max_len=n, window=window)
        for i in range(new):
            p = n - new + i
            sees = p >= bad and (not window or p - bad < window)
            assert bool(torch.isnan(out[i].float()).any()) == sees, (window, i)


@pytest.mark.parametrize("hq,hkv,d,page", HEADS)
@pytest.mark.parametrize("new,old", [([40, 1, 0, 17] * 6, [30, 0, 5, 160] * 6), ([200, 0, 9], [1400, 70, 3000]), ([67], [5000]),
                                     ([530, 31], [0, 600])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 5), (1100, 0)])
def test_chunk_forms(cuda, hq, hkv, d, page, new, old, window, sinks):
    """Many sequences (longest tiles first), and few whose keys are shared out between CTAs and joined."""
    g = torch.Generator(device=cuda).manual_seed(hq + d + sum(new) + window)
    lens = [a + b for a, b in zip(new, old)]
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, page, g, fill=0xFF)
    q = torch.randn(sum(new), hq, d, device=cuda, generator=g).mul(1.5).to(BF)
    cu = cumulative(cuda, new)
    out = ops.kv4_attention(q, cache, table, lengths, cu, max_new=max(new), max_len=max(lens), window=window, sinks=sinks)
    again = ops.kv4_attention(q, cache, table, lengths, cu, max_new=max(new), max_len=max(lens), window=window, sinks=sinks)
    torch.cuda.synchronize()
    assert ops.device_error() == 0
    assert torch.equal(out, again)
    # every row would take minutes in 64 bits: the first and last eight of a sequence and every 29th between
    cum = cu.tolist()
    for b in range(len(new)):
        rows = [i for i in range(new[b]) if i < 8 or i >= new[b] - 8 or i % 29 == 0]
        for i in rows:
            at = cum[b] + i
            length = torch.tensor([lens[b] - new[b] + i + 1], dtype=I32, device=cuda)
            check_attention(q[at: at + 1], cache, table[b: b + 1], length, cumulative(cuda, [1]), out[at: at + 1], window, sinks)


@pytest.mark.parametrize("new,old", [([300, 2], [1200, 10]), ([40] * 20, [60] * 20)])
def test_chunk_nan_stays_hidden(cuda, new, old):
    """NaN in K and V of one token of the first sequence reaches the rows that see it and no other, whole or shared out."""
    g = torch.Generator(device=cuda).manual_seed(new[0])
    d, hkv, hq = 128, 2, 8
    lens = [a + b for a, b in zip(new, old)]
    cache, table, lengths = filled_cache(cuda, lens, hkv, d, 64, g, fill=0xFF)
    for bad in (old[0] + 3, 1):
        qkv = torch.full((1, 3 * hkv * d), math.nan, device=cuda).to(BF)
        one = torch.ones(d, device=cuda).to(BF)
        ops.qkv_rope_append(qkv, one, one, torch.ones(1, d, device=cuda), torch.zeros(1, d, device=cuda),
                            torch.zeros(1, dtype=I32, device=cuda), cache, table[:1],
                            torch.tensor([bad + 1], dtype=I32, device=cuda), cumulative(cuda, [1]), q_heads=hkv)
        q = torch.randn(sum(new), hq, d, device=cuda, generator=g).to(BF)
        for window in (5, 0):
            out = ops.kv4_attention(q, cache, table, lengths, cumulative(cuda, new), max_new=max(new), max_len=max(lens), window=window)
            p = old[0] + torch.arange(new[0], device=cuda)
            sees = torch.zeros_like(p, dtype=torch.bool)
            for x in {bad, old[0] + 3}:
                sees |= (p >= x) & ((p - x < window) if window else torch.ones_like(sees))
            nan = torch.isnan(out.float())
            assert torch.equal(nan[: new[0]].all(2).all(1), sees) and torch.equal(nan[: new[0]].any(2).any(1), sees)
            assert not bool(nan[new[0]:].any())


def test_chunk_rows_without_keys(cuda):
    """Rows before position 0 of a chunk whose keys are shared out see nothing: zeros."""
    g = torch.Generator(device=cuda).manual_seed(8)
    cache, table, _ = filled_cache(cuda, [1000], 2, 128, 64, g)
    new, hidden = 600, 130
    lengths = torch.tensor([new - hidden], dtype=I32, device=cuda)
    q = torch.randn(new, 16, 128, device=cuda, generator=g).to(BF)
    out = ops.kv4_attention(q, cache, table, lengths, cumulative(cuda, [new]), max_new=new, max_len=1000)
    assert bool((out[:hidden] == 0).all())
    check_attention(q[hidden: hidden + 40], cache, table, torch.tensor([40], dtype=I32, device=cuda), cumulative(cuda, [40]),
                    out[hidden: hidden + 40])


@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("mag", [1e-30, 1e-6, 1e6, 1e30])
def test_query_range(cuda, mag, new):
    """bf16 queries far outside fp16's range keep their scores (scale chosen to give them size 1)."""
    g = torch.Generator(device=cuda).manual_seed(5)
    cache, table, lengths = filled_cache(cuda, [150], 2, 128, 64, g)
    q = (torch.randn(new, 16, 128, device=cuda, generator=g) * mag).to(BF)
    scale = 128 ** -0.5 / mag
    if not 0 < scale < 1e30:
        scale = 1e29
    cu = cumulative(cuda, [new])
    out = ops.kv4_attention(q, cache, table, lengths, cu, max_new=new, max_len=150, scale=scale)
    check_attention(q, cache, table, lengths, cu, out, scale=scale)


def test_long_cache_past_32_bit_offsets(cuda):
    """Pages that lie past 2^32 bytes of the pool."""
    g = torch.Generator(device=cuda).manual_seed(6)
    d, hkv, page = 128, 2, 64
    pages = (1 << 32) // (hkv * page // 32 * 40 * d) + 8
    cache = ops.kv4_cache(pages, hkv, d, page, device=cuda)
    small, table, lengths = filled_cache(cuda, [130], hkv, d, page, g)
    far = torch.tensor([[pages - 1, pages - 3, 1]], dtype=I32, device=cuda)
    for i in range(3):
        cache[far[0, i].item()] = small[table[0, i].item()]
    q = torch.randn(1, 16, d, device=cuda, generator=g).to(BF)
    cu = cumulative(cuda, [1])
    a = ops.kv4_attention(q, cache, far, lengths, cu, max_new=1, max_len=130)
    b = ops.kv4_attention(q, small, table, lengths, cu, max_new=1, max_len=130)
    assert torch.equal(a, b)


def test_another_stream_and_graph(cuda):
    g = torch.Generator(device=cuda).manual_seed(8)
    cache, table, lengths = filled_cache(cuda, [500, 77], 2, 128, 64, g)
    q = torch.randn(2, 16, 128, device=cuda, generator=g).to(BF)
    cu = cumulative(cuda, [1, 1])
    want = ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=500)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=500)
    s.synchronize()
    assert torch.equal(got, want)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=500, out=out)
    lengths.copy_(torch.tensor([400, 60], device=cuda))  # the device's lengths count, not the captured ones
    graph.replay()
    torch.cuda.synchronize()
    check_attention(q, cache, table, lengths, cu, out)


# ------------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------------
def test_refusals(cuda):
    g = torch.Generator(device=cuda).manual_seed(4)
    cache, table, lengths = filled_cache(cuda, [40], 2, 128, 64, g)
    cu = cumulative(cuda, [1])
    q = torch.randn(1, 16, 128, device=cuda).to(BF)

    def attend(**kw):
        a = dict(q=q, cache=cache, table=table, lengths=lengths, cu_seqlens=cu, max_new=1, max_len=40)
        a.update(kw)
        return ops.kv4_attention(**a)

    attend()
    with pytest.raises(TypeError):
        attend(q=q.float())
    with pytest.raises(ValueError):
        attend(q=q.cpu())
    with pytest.raises(ValueError):
        attend(q=q[:, :, :64])
    with pytest.raises(ValueError):
        attend(q=q.transpose(0, 1).contiguous().transpose(0, 1)[:, ::2])
    with pytest.raises(ValueError):
        attend(cache=cache[..., :1280])
    with pytest.raises(ValueError):
        attend(cache=cache[:, :1])
    with pytest.raises(ValueError):
        attend(table=table.long())
    with pytest.raises(ValueError):
        attend(lengths=lengths.repeat(2))
    with pytest.raises(ValueError):
        attend(cu_seqlens=cu.long())
    with pytest.raises(_lib.RldxError):
        attend(q=torch.randn(1, 15, 128, device=cuda).to(BF))
    for bad in (dict(max_new=0), dict(max_len=0), dict(window=-1), dict(sinks=-2), dict(scale=0.0), dict(scale=math.nan)):
        with pytest.raises(_lib.RldxError):
            attend(**bad)
    assert attend(q=q[:0], cu_seqlens=torch.zeros(2, dtype=I32, device=cuda)).shape == (0, 16, 128)

    one = torch.ones(128, device=cuda).to(BF)
    cos, sin = torch.ones(4, 128, device=cuda), torch.zeros(4, 128, device=cuda)
    pos = torch.zeros(1, dtype=I32, device=cuda)
    qkv = torch.randn(1, 20 * 128, device=cuda).to(BF)

    def append(**kw):
        a = dict(qkv=qkv, q_norm=one, k_norm=one, cos=cos, sin=sin, rope_pos=pos, cache=cache, table=table, lengths=lengths,
                 cu_seqlens=cu, q_heads=16)
        a.update(kw)
        return ops.qkv_rope_append(**a)

    append()
    for bad in (dict(qkv=qkv.float()), dict(cos=cos.half(), sin=sin.half()), dict(sin=sin.to(BF)), dict(rope_pos=pos.long())):
        with pytest.raises(TypeError):
            append(**bad)
    for bad in (dict(qkv=qkv[:, 128:]), dict(q_heads=15), dict(q_norm=one[:64]), dict(cos=cos[:, :64], sin=sin[:, :64]),
                dict(rope_pos=pos.repeat(2)), dict(out=torch.empty(1, 16, 64, dtype=BF, device=cuda))):
        with pytest.raises(ValueError):
            append(**bad)
    with pytest.raises(ValueError):
        ops.kv4_cache(4, 2, 96)
    with pytest.raises(ValueError):
        ops.kv4_cache(4, 2, 128, page_size=48)
    assert ops.device_error() == 0


def test_device_side_bounds_are_reported(cuda):
    """What only the device can see is skipped and reported: pages outside the pool, RoPE rows outside
    the table, sequences longer than the call said."""
    g = torch.Generator(device=cuda).manual_seed(4)
    cache, table, lengths = filled_cache(cuda, [40], 2, 128, 64, g)
    before = cache.clone()
    cu = cumulative(cuda, [1])
    q = torch.randn(1, 16, 128, device=cuda).to(BF)
    bad = torch.full_like(table, cache.shape[0])
    ops.kv4_attention(q, cache, bad, lengths, cu, max_new=1, max_len=40)
    assert ops.device_error() == 0x500
    ops.kv4_attention(q, cache, table, lengths, cu, max_new=1, max_len=4)
    assert ops.device_error() == 0x502
    one = torch.ones(128, device=cuda).to(BF)
    qkv = torch.randn(1, 20 * 128, device=cuda).to(BF)
    cos, sin = torch.ones(4, 128, device=cuda), torch.zeros(4, 128, device=cuda)
    for t, length in ((bad, 40), (table, 64 * table.shape[1] + 1), (table, 0)):
        ops.qkv_rope_append(qkv, one, one, cos, sin, torch.zeros(1, dtype=I32, device=cuda), cache, t,
                            torch.tensor([length], dtype=I32, device=cuda), cu, q_heads=16)
        assert ops.device_error() == 0x500
    assert torch.equal(cache, before)
    for row in (4, -1):
        ops.qkv_rope_append(qkv, one, one, cos, sin, torch.full((1,), row, dtype=I32, device=cuda), cache, table, lengths, cu, q_heads=16)
        assert ops.device_error() == 0x501
    assert ops.device_error() == 0
