"""B200TextDecoder's calls without a GPU: what they refuse before the cache changes, and what they hand on."""

import math

import pytest
import torch

import rldx_b200  # noqa: F401
from rldx_b200 import _lib, decoder
from rldx_b200.decoder import B200TextDecoder
from rldx_b200.rope import B200Rope

from test_decoder_host import BF, HEAD, HIDDEN, ROWS, VOCAB, layer, make, refused, state, weight


def roped(**kw):
    return B200TextDecoder([layer(), layer()], weight(HIDDEN), torch.zeros(VOCAB, HIDDEN), torch.zeros(VOCAB, HIDDEN), device="cpu",
                           rope=B200Rope(HEAD, sections=(16, 8, 8), device="cpu"), **kw)


@pytest.mark.parametrize("build", [make, roped])
def test_ids_are_whole_numbers(build):
    """Floats and bools were cut to whole numbers and ran."""
    dec, u = build(), torch.zeros(2, 2)
    cache = dec.new_cache(2, 256)
    before = state(cache)
    for ids in ([0.4, 3.6], [1.0, 2.0], [math.nan], torch.tensor([1.0]), [True, False], torch.tensor([True, False]), torch.tensor([1 + 2j])):
        with pytest.raises(ValueError, match="ids must be whole numbers"):
            dec.generate([[1], ids], 2, u=u, cache=cache)
        with pytest.raises(ValueError, match="ids must be whole numbers"):
            dec.score([[1], ids], cache=cache)
    for ids in (torch.tensor(3), [[1, 2]], torch.zeros(1, 2, HIDDEN, dtype=torch.int64)):
        with pytest.raises(ValueError, match="a prompt is ids"):
            dec.generate([[1], ids], 2, u=u, cache=cache)
    for target in ([0.4, 3.6], [1.0, 2.0], [math.nan, 1.0], [True, False], torch.tensor([1.0, 2.0])):
        with pytest.raises(ValueError, match="targets must be whole numbers"):
            dec.score([[1], [2, 3]], targets=[[1], target], cache=cache)
    assert state(cache) == before


def test_positions_are_whole_numbers():
    u = torch.zeros(2, 2)
    tables, rope = make(), roped()
    cache = tables.new_cache(2, 256)
    before = state(cache)
    for bad in ([0.5, 1.0], [math.nan, 1.0], [math.inf, 1.0], [True, False], torch.tensor([0.0, 1.5])):
        for dec in (tables, rope):
            with pytest.raises(ValueError, match="positions must be whole numbers"):
                dec.generate([[1], [2, 3]], 2, u=u, positions=[[0], bad], cache=cache)
            with pytest.raises(ValueError, match="positions must be whole numbers"):
                dec.score([[1], [2, 3]], positions=[[0], bad], cache=cache)
        for dec in (tables, rope):
            with pytest.raises(ValueError, match="next_positions must be whole numbers"):
                dec.generate([[1], [2, 3]], 2, u=u, positions=[[0], [0, 1]], next_positions=bad, cache=cache)
        refused(tables, cache, ValueError, "positions must be whole numbers", torch.zeros(2, HIDDEN, dtype=BF), [0, 2], positions=torch.as_tensor(bad))
        with pytest.raises(ValueError, match="deepstack_rows must be whole numbers"):
            tables.forward(torch.zeros(2, HIDDEN, dtype=BF), cache, [0, 2], deepstack_features=[torch.zeros(2, HIDDEN)], deepstack_rows=bad)
    with pytest.raises(ValueError, match="rows of the RoPE tables"):  # (cut to 32 bits it was row 5)
        tables.generate([[1], [2, 3]], 2, u=u, positions=[[2 ** 32 + 5], [0, 1]], cache=cache)
    assert state(cache) == before


def test_whole_positions_of_any_type_are_handed_on(monkeypatch):
    dec, seen = make(), []

    def forward(hidden, cache, new, positions=None):
        seen.append(positions.tolist())
        cache.extend(new)

    monkeypatch.setattr(decoder.ops, "sample", lambda *a, **kw: (torch.tensor([1, 2]), None, None))
    monkeypatch.setattr(decoder.ops, "device_error", lambda: 0)
    monkeypatch.setattr(dec, "forward", forward)
    for p in ([0.0, 4.0], torch.tensor([0, 4], dtype=torch.uint8), torch.tensor([0, 4], dtype=torch.int32)):
        for follow in ([5, 9], (5.0, 9.0), iter([5, 9]), torch.tensor([5, 9], dtype=torch.int16), [torch.tensor(5), torch.tensor(9)]):
            dec.generate([[1], [2, 3]], 2, u=torch.zeros(2, 2), positions=[[ROWS - 1], p], next_positions=follow)
            assert seen == [[ROWS - 1, 0, 4], [5, 9]]
            del seen[:]


class Stop(Exception):
    pass


def first_norm(monkeypatch, dec):
    """What a step hands to its first norm, in place of running it."""
    seen = []

    def norm(x, weight):
        seen.append(x)
        raise Stop

    monkeypatch.setattr(dec, "_here", lambda *a, **kw: None)
    monkeypatch.setattr(dec, "_rmsnorm", norm)
    return seen


@pytest.mark.parametrize("scale", [1.0, 0.5])
def test_rows_of_any_layout_are_run(monkeypatch, scale):
    """Columns first or off 16 bytes, they were refused in mid-step: the cache had their tokens."""
    dec = make(residual_scale=scale)
    seen = first_norm(monkeypatch, dec)
    rows = torch.randn(5, HIDDEN).to(BF)
    off = torch.zeros(5 * HIDDEN + 1, dtype=BF)[1:].view(5, HIDDEN)
    wide = torch.zeros(5, HIDDEN + 3, dtype=BF)[:, 1: 1 + HIDDEN]
    for x in (rows, rows.t().contiguous().t(), off.copy_(rows), wide.copy_(rows)):
        with pytest.raises(Stop):
            dec.forward(x, dec.new_cache(1, 64), [5])
        got = seen.pop()
        assert torch.equal(got, rows) and got.is_contiguous() and got.data_ptr() % 16 == 0
    assert rows.is_contiguous()


def test_positions_of_any_layout_reach_the_rope(monkeypatch):
    """[axes, rows] that lie the other way round, or every other one, were refused; an axis' positions go side by side."""
    dec, seen = roped(), []
    first_norm(monkeypatch, dec)

    def rows(positions):
        seen.append(positions)
        return torch.zeros(4, HEAD), torch.zeros(4, HEAD)

    monkeypatch.setattr(dec.rope, "rows", rows)
    at = torch.arange(12).view(3, 4)
    every = torch.zeros(3, 8, dtype=torch.int32)[:, ::2]
    for p in (at, at.t().contiguous().t(), every.copy_(at), at.to(torch.int16)):
        with pytest.raises(Stop):
            dec.forward(torch.zeros(4, HIDDEN, dtype=BF), dec.new_cache(1, 64), [4], p)
        got = seen.pop()
        assert torch.equal(got, at) and got.dtype == torch.int64 and got.stride(1) == 1
    one = torch.arange(8)[::2]
    with pytest.raises(Stop):
        dec.forward(torch.zeros(4, HIDDEN, dtype=BF), dec.new_cache(1, 64), [4], one)
    got = seen.pop()
    assert torch.equal(got, one.expand(3, -1)) and got.stride(1) == 1


def test_counts_may_come_from_an_iterator(monkeypatch):
    """They were used up before the last rows were picked: no logits."""
    dec, last = make(), []
    monkeypatch.setattr(dec, "_run", lambda hidden, cache, new, *a: last.append(list(new)) or (lambda rows: last.append(rows.tolist()) or torch.zeros(len(rows), HIDDEN)))
    monkeypatch.setattr(decoder.ops, "linear", lambda x, w: x)
    for new in ([2, 0, 3], iter([2, 0, 3]), (n for n in (2, 0, 3)), torch.tensor([2, 0, 3])):
        assert dec.forward(torch.zeros(5, HIDDEN, dtype=BF), None, new).shape == (2, HIDDEN)
        assert last == [[2, 0, 3], [1, 4]]
        del last[:]


@pytest.mark.parametrize("n", [2.5, 2.0, "2", math.nan, None])
def test_numbers_of_alternatives_are_whole(n, monkeypatch):
    """A fraction was refused behind the step, which had filled the cache."""
    dec = make()
    cache = dec.new_cache(2, 256)
    before = state(cache)
    for name in ("_run", "forward"):
        monkeypatch.setattr(dec, name, lambda *a, **kw: pytest.fail("a step was run"))
    with pytest.raises(TypeError):
        dec.score([[1], [2, 3]], top=n, cache=cache)
    if n is not None:  # (None: no scores)
        with pytest.raises(TypeError):
            dec.generate([[1], [2, 3]], 2, u=torch.zeros(2, 2), logprobs=n, cache=cache)
    assert state(cache) == before


def scored(monkeypatch, dec, code=0):
    """score() with no device: logits of zeros, and scores that count the rows."""
    made = []

    def run(hidden, cache, new, *a):
        cache.extend(new)
        return lambda rows: hidden[rows]

    def logprobs(logits, tokens, top):
        n, first = len(tokens), sum(made)
        made.append(n)
        row = torch.arange(first, first + n)
        return row.float(), row.float(), tokens.int(), row[:, None].expand(n, top), row[:, None].expand(n, top).float()

    monkeypatch.setattr(dec, "_run", run)
    monkeypatch.setattr(decoder.ops, "linear", lambda x, w: x)
    monkeypatch.setattr(decoder.ops, "token_logprobs", logprobs)
    monkeypatch.setattr(decoder.ops, "device_error", lambda: code)
    return made


def test_score_reports_device_errors(monkeypatch):
    """As generate() does: scores of what a kernel left out came back as if they were whole."""
    dec = make()
    scored(monkeypatch, dec, 0x500)
    with pytest.raises(_lib.RldxError, match="0x500") as e:
        dec.score([[1], [2, 3]])
    assert e.value.code == _lib.RLDX_ERR_DEVICE
    scored(monkeypatch, dec)
    assert [s.rank.tolist() for s in dec.score([[1], [2, 3]], top=2)] == [[-1], [3, -1]]


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 100])
def test_scores_of_pieces_join(monkeypatch, rows):
    """Logits are made for some rows at a time; the pieces end inside prompts."""
    dec = make()
    made = scored(monkeypatch, dec)
    dec.score_logits = rows * VOCAB + VOCAB - 1
    got = dec.score([[1, 2, 3, 4], [5], [6, 7]], top=2)
    assert made == [min(rows, 7 - a) for a in range(0, 7, rows)]
    assert [s.rank.tolist() for s in got] == [[2, 3, 4, -1], [-1], [7, -1]]
    assert [s.logprob.tolist() for s in got] == [[0, 1, 2, 3], [4], [5, 6]] and [s.top_ids.tolist() for s in got][2] == [[5, 5], [6, 6]]


def test_a_layers_own_window_is_not_left_out(monkeypatch):
    """Layers with a sliding window ran over the whole sequence where the decoder was given none."""
    def build(*windows, **kw):
        return make([layer(sliding_window=w) for w in windows], **kw)

    rows = torch.zeros(9, HIDDEN, dtype=BF)
    for dec in (build(None, 8), build(8, 12), build(8, 8)):
        cache = dec.new_cache(2, 256)
        refused(dec, cache, ValueError, r"sliding window \(8\)", rows, [0, 9])
        refused(dec, cache, ValueError, r"sliding window \(8\)", rows, [0, 9], positions=torch.arange(9))
        cache.extend([0, 5])
        refused(dec, cache, ValueError, r"sliding window \(8\)", rows[:4], [0, 4])
        refused(dec, cache, ValueError, "no CPU path", rows[:3], [0, 3])  # everything else is right
        with pytest.raises(ValueError, match="sliding window"):
            dec.generate([[1], [2] * 5], 5, u=torch.zeros(5, 2))
    for dec in (build(None, None), build(8, 8, window=8), make()):
        refused(dec, dec.new_cache(2, 256), ValueError, "no CPU path", rows, [0, 9])
