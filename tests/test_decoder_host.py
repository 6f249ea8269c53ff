"""B200TextDecoder's host side without a GPU: what it hands to the library, and what it refuses before any device work
with the cache as it was."""

from types import SimpleNamespace as NS

import pytest
import torch

import rldx_b200  # noqa: F401
from rldx_b200 import _lib
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
