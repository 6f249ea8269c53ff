"""B200TextDecoder's host side without a GPU: what it hands to the library, and what it refuses before any device work
with the cache as it was."""

from types import SimpleNamespace as NS

import pytest
import torch

import rldx_b200  # noqa: F401
from rldx_b200 import _lib, decoder
from rldx_b200.decoder import B200TextDecoder

BF = torch.bfloat16
HIDDEN, HEAD, HQ, HKV, FFN, VOCAB, ROWS = 64, 64, 2, 1, 96, 50, 40


def weight(*shape, bias=None):
    return NS(weight=torch.zeros(*shape), bias=bias)


def layer(**attn):
    a = dict(q_proj=weight(HQ * HEAD, HIDDEN), k_proj=weight(HKV * HEAD, HIDDEN), v_proj=weight(HKV * HEAD, HIDDEN),
             o_proj=weight(HIDDEN, HQ * HEAD), q_norm=weight(HEAD), k_norm=weight(HEAD))
    a.update(attn)
    return NS(input_layernorm=weight(HIDDEN), post_attention_layernorm=weight(HIDDEN), self_attn=NS(**a),
              mlp=NS(gate_proj=weight(FFN, HIDDEN), up_proj=weight(FFN, HIDDEN), down_proj=weight(HIDDEN, FFN)))


def make(layers=None, **kw):
    return B200TextDecoder(layers or [layer(), layer()], weight(HIDDEN), torch.zeros(VOCAB, HIDDEN), torch.zeros(VOCAB, HIDDEN),
                           torch.zeros(ROWS, HEAD), torch.zeros(ROWS, HEAD), device="cpu", **kw)


def test_norm_hands_over_rows_of_one_stride(monkeypatch):
    """Input and output share a row stride: a view of wider rows is copied, and the output is its own rows long."""
    seen = []

    class Lib:
        @staticmethod
        def rldx_res_rmsnorm(seg, n, eps, stream):
            s = seg._obj
            seen.append((s.rows, s.D, s.ld, s.x, s.ln_out))
            return _lib.RLDX_OK

    monkeypatch.setattr(_lib, "load", lambda: Lib)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: NS(cuda_stream=0))
    wide = torch.zeros(5, 3 * HIDDEN, dtype=BF)
    for x in (wide[:, HIDDEN: 2 * HIDDEN], wide[:, :HIDDEN], torch.zeros(5, HIDDEN, dtype=BF), torch.zeros(HIDDEN, 5, dtype=BF).t()):
        out = make()._rmsnorm(x, torch.zeros(HIDDEN, dtype=BF))
        rows, width, ld, src, dst = seen.pop()
        assert (rows, width, ld) == (5, HIDDEN, HIDDEN) and dst == out.data_ptr()
        assert out.shape == (5, HIDDEN) and out.stride() == (HIDDEN, 1)
        assert (src == x.data_ptr()) == x.is_contiguous()


def state(cache):
    return list(cache.tokens), cache.lengths.tolist(), cache.table.tolist(), cache.free_tokens


def refused(dec, cache, error, match, hidden, new, **kw):
    before = state(cache)
    with pytest.raises(error, match=match):
        dec.forward(hidden, cache, new, **kw)
    assert state(cache) == before


def test_other_devices_are_refused(monkeypatch):
    """On the host, before any launch: a CPU decoder, tensors of another device, another current device."""
    launches = []
    monkeypatch.setattr(_lib, "load", lambda: launches.append(1))
    dec = make()
    cache = dec.new_cache(1, 64)
    refused(dec, cache, ValueError, "no CPU path", torch.zeros(3, HIDDEN, dtype=BF), [3])
    meta = torch.zeros(3, HIDDEN, dtype=BF, device="meta")  # stands for another device
    refused(dec, cache, ValueError, "hidden is on meta", meta, [3])
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    dec.embed = NS(device=torch.device("cuda", 1))  # a decoder of device 1 while 0 is current
    on_one = NS(shape=(3, HIDDEN), dtype=BF, device=torch.device("cuda", 1))
    refused(dec, cache, ValueError, "cache is on cpu", on_one, [3])
    there = NS(tokens=[0], table=NS(device=torch.device("cuda", 1)), pools=cache.pools)
    with pytest.raises(ValueError, match="not the current CUDA device"):
        dec.forward(on_one, there, [3])
    assert not launches


def test_a_refused_forward_leaves_the_cache_alone():
    dec = make()
    cache = dec.new_cache(2, 256)
    rows = lambda n: torch.zeros(n, HIDDEN, dtype=BF)  # noqa: E731
    refused(dec, cache, ValueError, "longer than the RoPE tables", rows(ROWS + 4), [3, ROWS + 1])
    refused(dec, cache, ValueError, "hidden must be", rows(3).float(), [1, 2])
    refused(dec, cache, ValueError, "hidden must be", rows(4), [1, 2])
    refused(dec, cache, ValueError, "count for each", rows(3), [3])
    refused(dec, cache, ValueError, "count for each", rows(3), [4, -1])
    refused(dec, cache, ValueError, "one of them positive", rows(0), [0, 0])
    refused(dec, cache, ValueError, "positions must be", rows(3), [1, 2], positions=torch.zeros(2, dtype=torch.int32))
    for bad in ([0, 1, ROWS], [-1, 0, 1]):
        refused(dec, cache, ValueError, "rows of the RoPE tables", rows(3), [1, 2], positions=torch.tensor(bad))
    cache.extend([30, 0])
    refused(dec, cache, ValueError, "longer than the RoPE tables", rows(11), [11, 0])


def test_generate_refuses_what_it_could_not_finish(monkeypatch):
    """Before the first step: the tables' length, the cache's pages and its sequences for the whole run."""
    dec = make()
    monkeypatch.setattr(dec, "forward", lambda *a, **kw: pytest.fail("a step was run"))
    cache = dec.new_cache(2, 256, page_size=32)
    before = state(cache)

    def run(prompts, n, cache=cache):
        return dec.generate(prompts, n, u=torch.zeros(n, len(prompts)), cache=cache)

    with pytest.raises(ValueError, match="longer than the RoPE tables"):
        run([[1] * 10, [2] * 5], ROWS - 10 + 2)
    with pytest.raises(ValueError, match="the cache has 2 sequences"):
        run([[1]], 3)
    with pytest.raises(ValueError, match="no token"):
        run([torch.tensor([1]), torch.zeros(0, dtype=torch.long)], 3)
    small = dec.new_cache(2, 1, page_size=32)  # three pages
    with pytest.raises(RuntimeError, match="free pages"):
        run([[1] * 30, [2] * 30], 10, cache=small)
    assert state(cache) == before and small.tokens == [0, 0]
    cache.extend([20, 0])
    with pytest.raises(ValueError, match="longer than the RoPE tables"):
        run([[1] * 10, [2] * 5], ROWS - 30 + 2)


def test_other_models_caches_and_tables_are_refused():
    """A cache of fewer layers would run fewer layers; tables of another width would be refused in mid-step."""
    dec = make()
    rows = torch.zeros(2, HIDDEN, dtype=BF)
    for other in (make([layer()]), make([layer()] * 3)):
        refused(dec, other.new_cache(1, 64), ValueError, "not one of 2 layers", rows, [2])
    two = layer(k_proj=weight(2 * HEAD, HIDDEN), v_proj=weight(2 * HEAD, HIDDEN))
    refused(dec, make([two, two]).new_cache(1, 64), ValueError, "1 key / value heads of 64", rows, [2])
    for cos, sin in ((torch.zeros(9, 32), torch.zeros(9, 32)), (torch.zeros(9, HEAD), torch.zeros(8, HEAD)),
                     (torch.zeros(9, HEAD).half(), torch.zeros(9, HEAD).half()), (torch.zeros(9, HEAD), torch.zeros(9, HEAD, dtype=BF))):
        with pytest.raises(ValueError, match="cos and sin must be"):
            B200TextDecoder([layer()], weight(HIDDEN), torch.zeros(VOCAB, HIDDEN), torch.zeros(VOCAB, HIDDEN), cos, sin, device="cpu")


def scripted(monkeypatch, dec, tokens, code=0):
    """generate() over drawn tokens given per step, with no device."""
    steps = iter(tokens)
    monkeypatch.setattr(dec, "forward", lambda hidden, cache, new, *a, **kw: cache.extend(new))
    monkeypatch.setattr(decoder.ops, "sample", lambda *a, **kw: (torch.tensor(next(steps)), None, None))
    monkeypatch.setattr(decoder.ops, "device_error", lambda: code)


def test_generate_reports_rows_without_a_token(monkeypatch):
    dec = make()
    u = torch.zeros(3, 2)
    scripted(monkeypatch, dec, [[4, 5], [6, -1], [7, 8]])
    with pytest.raises(RuntimeError, match="sequence 1 has no logit that is a number at its token 1"):
        dec.generate([[1], [2, 3]], 3, u=u)
    scripted(monkeypatch, dec, [[4, 9], [6, -1], [7, 8]])  # past its end: of no interest
    assert dec.generate([[1], [2, 3]], 3, u=u, stop_ids=[9]) == [[4, 6, 7], [9]]


def test_generate_reports_device_errors(monkeypatch):
    dec = make()
    scripted(monkeypatch, dec, [[4], [5]], code=0x500)
    with pytest.raises(_lib.RldxError, match="0x500") as e:
        dec.generate([[1]], 2, u=torch.zeros(2, 1))
    assert e.value.code == _lib.RLDX_ERR_DEVICE
    scripted(monkeypatch, dec, [[4], [5]])
    assert dec.generate([[1]], 2, u=torch.zeros(2, 1)) == [[4, 5]]


def test_layers_that_it_does_not_run_are_refused():
    """Video-token compression, biases and layers without the per-head norms, each of which was left out without a word."""
    wrapped = [NS(layer=layer(), internal_projection=1, layer_idx=i) for i in range(3)]
    with pytest.raises(NotImplementedError, match="layer 1 compresses video tokens"):
        make(wrapped)
    assert len(make(wrapped, ignore_compression=True).layers) == 3
    assert len(make(wrapped[:1]).layers) == 1  # this one's wrapper never compresses
    with pytest.raises(NotImplementedError, match="bias"):
        make([layer(), layer(v_proj=weight(HKV * HEAD, HIDDEN, bias=torch.zeros(HEAD)))])
    biased = layer()
    biased.mlp.down_proj.bias = torch.zeros(HIDDEN)
    with pytest.raises(NotImplementedError, match="bias"):
        make([layer(), biased])
    with pytest.raises(NotImplementedError, match="q_norm"):
        make([layer(), layer(k_norm=None)])


def test_generate_hands_on_positions(monkeypatch):
    dec = make()
    seen = []

    def forward(hidden, cache, new, positions=None):
        seen.append(None if positions is None else positions.tolist())
        cache.extend(new)

    monkeypatch.setattr(decoder.ops, "sample", lambda *a, **kw: (torch.tensor([1, 2]), None, None))
    monkeypatch.setattr(decoder.ops, "device_error", lambda: 0)
    monkeypatch.setattr(dec, "forward", forward)
    prompts, u = [[5, 6, 7], torch.zeros(2, HIDDEN)], torch.zeros(3, 2)
    dec.generate(prompts, 3, u=u)
    dec.generate(prompts, 3, u=u, positions=[[0, 4, 4], torch.tensor([1, 0])])
    dec.generate(prompts, 3, u=u, positions=[[0, 4, 4], [1, 0]], next_positions=[ROWS - 2, 9])
    assert seen == [None] * 3 + [[0, 4, 4, 1, 0], [5, 2], [6, 3]] + [[0, 4, 4, 1, 0], [ROWS - 2, 9], [ROWS - 1, 10]]
    del seen[:]
    for kw in (dict(positions=[[0, 1, 2], [0]]), dict(positions=[[0, 1, 2]]), dict(positions=[[0, 1, ROWS], [0, 1]]),
               dict(positions=[[0, -1, 2], [0, 1]]), dict(positions=[[0, 1, ROWS - 2], [0, 1]]), dict(next_positions=[3, 3]),
               dict(positions=[[0, 1, 2], [0, 1]], next_positions=[3]), dict(positions=[[0, 1, 2], [0, 1]], next_positions=[3, ROWS - 1])):
        with pytest.raises(ValueError, match="positions"):
            dec.generate(prompts, 3, u=u, **kw)
    assert not seen


def test_deepstack_that_does_not_fit_is_refused():
    dec = make()
    cache, rows = dec.new_cache(2, 256), torch.zeros(5, HIDDEN, dtype=BF)
    f = torch.zeros(2, HIDDEN)
    for kw, match in ((dict(deepstack_features=[f]), "need deepstack_rows"), (dict(deepstack_rows=torch.tensor([1, 2])), "go with"),
                      (dict(deepstack_features=[f], deepstack_rows=torch.tensor([1, 5])), "different rows of the 5"),
                      (dict(deepstack_features=[f], deepstack_rows=torch.tensor([-1, 2])), "different rows"),
                      (dict(deepstack_features=[f], deepstack_rows=torch.tensor([2, 2])), "different rows"),
                      (dict(deepstack_features=[f, f, f], deepstack_rows=torch.tensor([1, 2])), "at most 2"),
                      (dict(deepstack_features=[f, f[:1]], deepstack_rows=torch.tensor([1, 2])), "at most 2"),
                      (dict(deepstack_features=[f[:, 1:]], deepstack_rows=torch.tensor([1, 2])), "at most 2")):
        refused(dec, cache, ValueError, match, rows, [2, 3], **kw)
    with pytest.raises(ValueError, match="go with"):
        dec.generate([[1], [2]], 2, u=torch.zeros(2, 2), deepstack_rows=torch.tensor([0]))
