"""Calls of the operators around a decoder's products that are refused before any device work."""

import math

import pytest
import torch

import rldx_b200  # noqa: F401
from rldx_b200 import _lib, ops  # noqa: F401
from rldx_b200.rope import B200Rope, frequencies  # noqa: F401

BF, F64 = torch.bfloat16, torch.float64


def test_logprobs_pointers_are_aligned(lib):
    """Tokens and results that begin inside a word would fault on the device."""
    def call(tokens=256, logprob=256, entropy=256, rank=256, ids=256, values=256, top=2):
        return lib.rldx_token_logprobs(256, 50, 3, 50, 2, tokens, top, logprob, entropy, rank, ids, values, None)

    for kw in (dict(tokens=260), dict(tokens=257), dict(logprob=258), dict(entropy=257), dict(rank=258), dict(ids=260), dict(values=258)):
        assert call(**kw) == _lib.RLDX_ERR_ARG, kw
        assert b"misaligned" in lib.rldx_last_error()


def test_rope_results_are_apart_from_positions_and_freqs():
    """A block may turn its tokens while another still reads them."""
    words = torch.zeros(1024, dtype=torch.int64)
    heads = words.view(BF)[: 6 * 4 * 64].unflatten(0, (6, 4, 64))
    q, at, f = torch.zeros(6, 4, 64, dtype=BF), torch.arange(6), torch.ones(32, dtype=F64)
    for kw, match in ((dict(at=words[:6]), "out_q shares memory with positions"), (dict(at=words[383:389]), "out_q shares memory with positions"),
                      (dict(at=words[:18].view(3, 6), sections=(16, 8, 8)), "out_q shares memory with positions"),
                      (dict(f=words[100:132].view(F64)), "out_q shares memory with freqs"), (dict(at=words[384:390]), "CUDA")):
        place, freqs = kw.pop("at", at), kw.pop("f", f)
        with pytest.raises(ValueError, match=match):
            ops.rope(q, None, place, freqs, out_q=heads, **kw)
    with pytest.raises(ValueError, match="out_k shares memory with freqs"):
        ops.rope(torch.zeros(6, 4, 64, dtype=BF), q, at, words[100:132].view(F64), out_k=heads)


def test_a_scalings_factor_needs_its_type():
    """Without one it divided every frequency."""
    for scaling in ({"factor": 4.0}, {"type": None, "factor": 4.0}):
        with pytest.raises(ValueError, match="needs its type"):
            frequencies(64, 1e4, scaling)
    for scaling in (None, {}, {"type": None}, {"type": "linear"}):
        f, m = frequencies(64, 1e4, scaling)
        assert m == 1.0 and torch.equal(f, frequencies(64, 1e4)[0])


def test_yarn_divides_every_pair_that_turns_too_little():
    """The fastest pair was kept, however little it turns; with theta below 1 pairs were blended the wrong way round."""
    f, _ = frequencies(128, 1e6)
    for kw in (dict(original=5), dict(original=128, beta_fast=32.0, beta_slow=32.0), dict(original=128, beta_fast=64.0, beta_slow=21.0)):
        assert kw["original"] / (2 * math.pi) < kw.get("beta_slow", 1.0)
        y, _ = frequencies(128, 1e6, {"type": "yarn", "factor": 8.0, **kw})
        assert torch.allclose(y, f / 8, rtol=1e-15, atol=0)
    y, _ = frequencies(128, 1e6, {"type": "yarn", "factor": 8.0, "original": 7})  # one pair turns more than once
    assert y[0] == f[0] and torch.allclose(y[2:], f[2:] / 8, rtol=1e-15, atol=0)
    for theta in (0.5, 1.0):
        with pytest.raises(ValueError, match="theta above 1"):
            frequencies(128, theta, {"type": "yarn", "factor": 8.0, "original": 4096})


def test_rope_refusals_say_what_is_wrong():
    q, at, f = torch.zeros(6, 4, 64, dtype=BF), torch.arange(6), torch.ones(32, dtype=F64)
    for match, kw in (("sections must be a sequence", dict(sections=5)), ("integer", dict(sections=(16.0, 16))), ("real number", dict(factor="two"))):
        with pytest.raises(TypeError, match=match):
            ops.rope(q, None, at, f, **kw)
        with pytest.raises(TypeError, match=match):
            ops.rope_rows(at, f, **kw)
