"""The decoding path (B200TextDecoder over the 4-bit cache) against the layers in plain fp32 operations,
rounded to bf16 at the decoder's rounding points, with keys and values quantised by the plain formula.

The plain form rounds where the decoder does because a code moves by a whole step where its input
moves across a boundary.  Tolerance: sums of another order move a bf16 rounding now and then, and with
it a code; the backbone's prefill is held to cosine 0.9999 on such stacks without codes, here 0.999."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from oracle import qwen3_oracle as oq  # noqa: E402
from rldx_b200 import ops  # noqa: E402
from rldx_b200.decoder import B200TextDecoder  # noqa: E402

BF = torch.bfloat16
CFG = oq.Qwen3Config(hidden=256, q_heads=8, kv_heads=2, head_dim=64, ffn=512, layers=3)
VOCAB = 777


def quantised(x):
    g = x.unflatten(-1, (-1, 32))
    low, top = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s, lo = ((top - low) / 15).half().float(), low.half().float()
    return (((g - lo) / s.clamp_min(1e-30)).round().clamp(0, 15) * s + lo).flatten(-2)


def r(x):
    """The value that bf16 holds."""
    return x.to(BF).float()


def rms(x, w):
    return r(w * r(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)))


def normed(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w


def plain_logits(stack, embed, head, ids, cos, sin, window=0, sinks=0):
    """Logits of every position of one sequence, rounded to bf16 where the decoder rounds."""
    h, n = embed[ids], len(ids)
    pos = torch.arange(n, device=h.device)
    seen = pos <= pos[:, None]
    if window:
        seen &= (pos[:, None] - pos < window) | (pos < sinks)
    c, s = cos[:n, None], sin[:n, None]
    for m in stack.layers:
        a = m.self_attn
        x = rms(h, m.input_layernorm.weight)
        q, k, v = (r(p(x)).unflatten(-1, (-1, CFG.head_dim)) for p in (a.q_proj, a.k_proj, a.v_proj))
        q, k = normed(q, a.q_norm.weight), normed(k, a.k_norm.weight)
        q, k = r(q * c + oq.rotate_half(q) * s), k * c + oq.rotate_half(k) * s
        k, v = (quantised(t).repeat_interleave(CFG.q_heads // CFG.kv_heads, 1) for t in (k, v))
        w = torch.einsum("qhd,khd->hqk", q, k) * CFG.head_dim ** -0.5
        w = w.masked_fill(~seen, float("-inf")).softmax(-1)
        h = r(r(a.o_proj(r(torch.einsum("hqk,khd->qhd", w, v).flatten(1)))) + h)
        x = rms(h, m.post_attention_layernorm.weight)
        gate, up = r(m.mlp.gate_proj(x)), r(m.mlp.up_proj(x))
        h = r(r(m.mlp.down_proj(r(r(torch.nn.functional.silu(gate)) * up))) + h)
    return r(rms(h, stack.norm.weight) @ head.t())


def make(dev, **kw):
    stack = oq.init_weights(oq.TextStack(CFG), seed=3, std=0.05).to(dev)
    g = torch.Generator(device=dev).manual_seed(5)
    embed, head = torch.randn(VOCAB, CFG.hidden, device=dev, generator=g), torch.randn(VOCAB, CFG.hidden, device=dev, generator=g) * 0.1
    with torch.no_grad():
        for p in stack.parameters():
            p.copy_(p.to(BF))
    embed, head = embed.to(BF).float(), head.to(BF).float()
    cos, sin = oq.rope_tables(CFG, torch.arange(600))
    cos, sin = cos.to(dev), sin.to(dev)
    return stack, embed, head, cos, sin, B200TextDecoder(stack.layers, stack.norm, embed, head, cos, sin, device=dev, **kw)


def close(got, want):
    got, want = got.double(), want.double()
    cos = torch.nn.functional.cosine_similarity(got, want, dim=-1)
    assert bool((cos >= 0.999).all()), cos.min().item()


@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 4)])
@torch.no_grad()
def test_prefill_then_steps_match_plain_layers(cuda, window, sinks):
    stack, embed, head, cos, sin, dec = make(cuda, window=window, sinks=sinks)
    g = torch.Generator().manual_seed(7)
    seqs = [torch.randint(VOCAB, (n,), generator=g).to(cuda) for n in (97, 5, 230)]
    want = [plain_logits(stack, embed, head, s, cos, sin, window, sinks) for s in seqs]
    cache = dec.new_cache(3, 600)
    rows = dec.embed[torch.cat([s[:-4] for s in seqs])]
    got = dec.forward(rows, cache, [len(s) - 4 for s in seqs])
    close(got, torch.stack([w[len(s) - 5] for s, w in zip(seqs, want)]))
    for step in range(4, 1, -1):  # one token each
        got = dec.forward(dec.embed[torch.stack([s[len(s) - step] for s in seqs])], cache, [1, 1, 1])
        close(got, torch.stack([w[len(s) - step] for s, w in zip(seqs, want)]))
    got = dec.forward(dec.embed[seqs[2][-1:]], cache, [0, 0, 1])  # two sequences rest
    close(got, want[2][-1:])
    assert ops.device_error() == 0


@torch.no_grad()
def test_generate(cuda):
    _, _, _, _, _, dec = make(cuda)
    prompts = [[1, 5, 9, 200], list(range(40, 140)), [700]]
    u = torch.rand(9, 3, generator=torch.Generator().manual_seed(1))
    out = dec.generate(prompts, 9, u=u, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    assert [len(o) for o in out] == [9, 9, 9] and all(0 <= t < VOCAB for o in out for t in o)
    assert dec.generate(prompts, 9, u=u, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01) == out
    greedy = dec.generate(prompts, 5, u=u[:5], temperature=0.0)
    cache = dec.new_cache(3, 400)
    logits = dec.forward(dec.embed[torch.tensor(sum(prompts, []), device=cuda)], cache, [len(p) for p in prompts])
    assert [o[0] for o in greedy] == logits.float().argmax(-1).tolist()
    stop = out[1][3]
    cut = dec.generate(prompts, 9, u=u, temperature=0.9, top_k=40, top_p=0.95, min_p=0.01, stop_ids=[stop])
    assert cut[1] == out[1][: out[1].index(stop) + 1]
    with pytest.raises(ValueError):
        dec.generate(prompts, 3, u=u)
    with pytest.raises(ValueError):
        dec.forward(dec.embed[:2], cache, [1, 0, 0])
    with pytest.raises(RuntimeError, match="free pages"):
        dec.forward(dec.embed[torch.zeros(500, dtype=torch.long, device=cuda)], cache, [500, 0, 0])
