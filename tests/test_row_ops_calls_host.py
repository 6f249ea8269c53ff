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
