"""Which layers B200TextDecoder takes: what it would run otherwise than they do is refused when it is built."""

import math
from types import SimpleNamespace as NS

import pytest
import torch
import torch.nn as nn

import rldx_b200  # noqa: F401
from rldx_b200.decoder import B200TextDecoder
from rldx_b200.rope import B200Rope

from test_decoder_host import HEAD, HIDDEN, VOCAB, layer, weight


class Norm(nn.Module):
    """x / rms(x) * (plus + weight), as layers write it."""

    def __init__(self, n, plus=0.0, weight=None, dtype=torch.float32):
        super().__init__()
        self.plus, self.eps = plus, 1e-6
        self.weight = nn.Parameter((torch.ones(n) if weight is None else weight).to(dtype))

    def forward(self, x):
        y = x.float() * torch.rsqrt(x.float().pow(2).mean(-1, keepdim=True) + self.eps)
        return (y * (self.plus + self.weight.float())).to(x.dtype)


def build(layers, norm=None, **kw):
    return B200TextDecoder(layers, norm or Norm(HIDDEN), torch.zeros(VOCAB, HIDDEN), torch.zeros(VOCAB, HIDDEN),
                           rope=B200Rope(HEAD, device="cpu"), device="cpu", **kw)


NORMS = ("input_layernorm", "post_attention_layernorm", "pre_feedforward_layernorm", "post_feedforward_layernorm", "q_norm", "k_norm")


def four_norms(**put):
    m = layer()
    for name in NORMS:
        n = HEAD if name[1:] == "_norm" else HIDDEN
        setattr(m.self_attn if name[1:] == "_norm" else m, name, put.get(name, Norm)(n))
    return m


def test_layers_of_plain_norms_are_taken():
    g = torch.Generator().manual_seed(0)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        plain = {name: lambda n: Norm(n, weight=1 + 0.5 * torch.randn(n, generator=g), dtype=dtype) for name in NORMS}
        assert build([four_norms(), four_norms(**plain)], norm=Norm(HIDDEN, weight=torch.zeros(HIDDEN), dtype=dtype)).after
    m = four_norms()
    m.mlp.act_fn, m.self_attn.scaling, m.self_attn.attn_logit_softcapping = nn.SiLU(), HEAD ** -0.5, None
    assert build([m]).after
    m.mlp.act_fn = "silu"
    assert build([m]).after
    m.mlp.act_fn = torch.nn.functional.silu
    assert build([m]).after


@pytest.mark.parametrize("name", NORMS)
def test_norms_of_one_plus_weight_are_refused(name):
    """Their weights begin at zero, which a norm of w alone would multiply by."""
    g = torch.Generator().manual_seed(1)
    for w in (torch.zeros, lambda n: torch.randn(n, generator=g), lambda n: 10 + torch.randn(n, generator=g)):
        with pytest.raises(NotImplementedError, match=f"layer 1's {name} is not"):
            build([four_norms(), four_norms(**{name: lambda n: Norm(n, plus=1.0, weight=w(n))})])


def test_other_norms_are_refused():
    with pytest.raises(NotImplementedError, match="the final norm is not"):
        build([layer()], norm=Norm(HIDDEN, plus=1.0, weight=torch.zeros(HIDDEN)))
    with pytest.raises(NotImplementedError, match="has a bias"):
        build([four_norms(input_layernorm=nn.LayerNorm)])
    with pytest.raises(NotImplementedError, match="layer 0's input_layernorm is not"):
        build([four_norms(input_layernorm=lambda n: nn.LayerNorm(n, bias=False))])


@pytest.mark.parametrize("act", [nn.GELU("tanh"), nn.GELU(), nn.ReLU(), torch.tanh, lambda x: x * torch.sigmoid(1.702 * x), "gelu"])
def test_other_activations_are_refused(act):
    m = layer()
    m.mlp.act_fn = act
    with pytest.raises(NotImplementedError, match="layer 1's MLP"):
        build([layer(), m])


def test_other_scores_are_refused():
    for kw, match in ((dict(scaling=1 / 16), "scales by"), (dict(scaling=math.sqrt(HEAD)), "scales by"), (dict(attn_logit_softcapping=50.0), "caps")):
        with pytest.raises(NotImplementedError, match=match):
            build([layer(), layer(**kw)])


def sized(hidden=HIDDEN, head=HEAD, hq=2, hkv=1, ffn=96, **put):
    """A decoder of one layer of these sizes, or with other weights put in the place of some."""
    m = NS(input_layernorm=weight(hidden), post_attention_layernorm=weight(hidden),
           self_attn=NS(q_proj=weight(hq * head, hidden), k_proj=weight(hkv * head, hidden), v_proj=weight(hkv * head, hidden),
                        o_proj=weight(hidden, hq * head), q_norm=weight(head), k_norm=weight(head)),
           mlp=NS(gate_proj=weight(ffn, hidden), up_proj=weight(ffn, hidden), down_proj=weight(hidden, ffn)))
    for name, shape in put.items():
        at = next((p for p in (m, m.self_attn, m.mlp) if hasattr(p, name)), m)
        setattr(at, name, weight(*shape))
    return B200TextDecoder([m], weight(put.get("norm", (hidden,))[0]), torch.zeros(VOCAB, hidden), torch.zeros(*put.get("lm_head", (VOCAB, hidden))),
                           rope=B200Rope(head, device="cpu"), device="cpu")


def test_models_that_no_step_could_run_are_refused():
    """They were built, and refused by a kernel in mid-step, when the cache had the new tokens already."""
    assert sized(hidden=4096).hidden == 4096 and sized(head=128, hq=4, hkv=4).kv_heads == 4
    for kw, match in ((dict(hidden=4104), "4096 at most"), (dict(hidden=8192), "4096 at most"), (dict(hidden=60), "multiple of 8"),
                      (dict(head=32), "64 or 128"), (dict(hq=3, hkv=2), "as many query heads"), (dict(ffn=100), "multiple of 8")):
        with pytest.raises(NotImplementedError, match=match):
            sized(**kw)
    for kw in (dict(q_proj=(2 * HEAD, 32)), dict(k_proj=(2 * HEAD, HIDDEN)), dict(v_proj=(2 * HEAD, HIDDEN)), dict(o_proj=(HIDDEN, HEAD)),
               dict(k_norm=(128,)), dict(up_proj=(104, HIDDEN)), dict(down_proj=(HIDDEN, 104)), dict(input_layernorm=(72,)),
               dict(post_attention_layernorm=(72,)), dict(norm=(72,)), dict(lm_head=(VOCAB, 72))):
        if "k_proj" in kw:  # (counts the key / value heads)
            kw["v_proj"] = (HEAD, HIDDEN)
        with pytest.raises(ValueError, match="must be"):
            sized(**kw)
    with pytest.raises(ValueError, match="lm_head has no tokens"):
        sized(lm_head=(0, HIDDEN))
    for kw in (dict(window=-1), dict(sinks=-1)):
        with pytest.raises(ValueError, match="must not be negative"):
            build([layer()], **kw)
    with pytest.raises(ValueError, match="layer 1's k_proj must be"):
        build([layer(), layer(k_proj=weight(2 * HEAD, HIDDEN), v_proj=weight(2 * HEAD, HIDDEN))])
