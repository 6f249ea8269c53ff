"""B200TextDecoder beyond plain prompts: rows that cannot be drawn from, prompts with positions and features of their
own.  Plain forms and their tolerance: test_decoder_gpu.py."""

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from rldx_b200.decoder import B200TextDecoder  # noqa: E402
import test_decoder_gpu as T  # noqa: E402
from test_decoder_gpu import make  # noqa: E402


@torch.no_grad()
def test_a_sequence_of_nan_is_reported(cuda):
    dec = make(cuda)[-1]
    bad = dec.embed[:6].clone()
    bad[3] = float("nan")
    u = torch.rand(4, 2, generator=torch.Generator().manual_seed(1))
    with pytest.raises(RuntimeError, match="sequence 1 has no logit that is a number at its token 0"):
        dec.generate([[1, 2, 3], bad], 4, u=u)
    assert ops.device_error() == 0
    assert len(dec.generate([[1, 2, 3], bad[:3]], 4, u=u)[1]) == 4


@torch.no_grad()
def test_generate_with_positions(cuda):
    """The same tokens where the tables hold the same rows elsewhere, and those of single steps with the same positions."""
    stack, embed, head, cos, sin, dec = make(cuda)
    prompts = [[1, 5, 9, 200, 31], list(range(40, 140))]
    u = torch.rand(8, 2, generator=torch.Generator().manual_seed(2))
    want = dec.generate(prompts, 8, u=u, temperature=0.8, top_p=0.95)
    moved = B200TextDecoder(stack.layers, stack.norm, embed, head, *(torch.cat([torch.full_like(t[:50], 7.0), t]) for t in (cos, sin)),
                            device=cuda)
    at = [torch.arange(len(p)) + 50 for p in prompts]
    assert moved.generate(prompts, 8, u=u, temperature=0.8, top_p=0.95, positions=at) == want
    assert moved.generate(prompts, 8, u=u, temperature=0.8, top_p=0.95) != want
    # as vision tokens stand: several in one place, the text after them one past the largest
    rows = dec.embed[torch.tensor(prompts[1][:40], device=cuda)]
    place = torch.cat([torch.arange(10), 10 + torch.arange(20) // 5 % 4, torch.arange(14, 24)])
    got = dec.generate([rows], 6, u=u[:6, :1], temperature=0.0, positions=[place])[0]
    cache, hidden, new, pos, ids = dec.new_cache(1, 60), rows, [40], place, []
    for i in range(6):
        ids.append(int(dec.forward(hidden, cache, new, pos).float().argmax()))
        hidden, new, pos = dec.embed[ids[-1]][None], [1], torch.tensor([24 + i])
    assert got == ids
    assert ops.device_error() == 0


def plain_deepstack(stack, head, h, cos, sin, features, rows):
    """Logits of every row of one sequence of embeddings h, features[i] added after layer i to `rows`."""
    n, c, s = len(h), cos[: len(h), None], sin[: len(h), None]
    for i, m in enumerate(stack.layers):
        a = m.self_attn
        x = T.rms(h, m.input_layernorm.weight)
        q, k, v = (T.r(p(x)).unflatten(-1, (-1, T.CFG.head_dim)) for p in (a.q_proj, a.k_proj, a.v_proj))
        q, k = T.normed(q, a.q_norm.weight), T.normed(k, a.k_norm.weight)
        q, k = T.r(q * c + T.oq.rotate_half(q) * s), k * c + T.oq.rotate_half(k) * s
        k, v = (T.quantised(t).repeat_interleave(T.CFG.q_heads // T.CFG.kv_heads, 1) for t in (k, v))
        w = torch.einsum("qhd,khd->hqk", q, k) * T.CFG.head_dim ** -0.5
        w = w.masked_fill(torch.ones(n, n, dtype=torch.bool, device=h.device).triu(1), float("-inf")).softmax(-1)
        h = T.r(T.r(a.o_proj(T.r(torch.einsum("hqk,khd->qhd", w, v).flatten(1)))) + h)
        x = T.rms(h, m.post_attention_layernorm.weight)
        gate, up = T.r(m.mlp.gate_proj(x)), T.r(m.mlp.up_proj(x))
        h = T.r(T.r(m.mlp.down_proj(T.r(T.r(torch.nn.functional.silu(gate)) * up))) + h)
        if i < len(features):
            h = h.index_copy(0, rows, T.r(h[rows] + features[i]))
    return T.r(T.rms(h, stack.norm.weight) @ head.t())


@torch.no_grad()
def test_deepstack_features_join_their_rows(cuda):
    stack, _, head, cos, sin, dec = make(cuda)
    g = torch.Generator(device=cuda).manual_seed(3)
    seqs = [dec.embed[torch.randint(T.VOCAB, (n,), device=cuda, generator=g)] for n in (60, 25)]
    rows = [torch.arange(8, 40), torch.tensor([24, 3])]  # of each sequence; the second's last among them
    feats = [[(3.0 * torch.randn(len(r), T.CFG.hidden, device=cuda, generator=g)).to(T.BF) for _ in range(2)] for r in rows]
    want = torch.stack([plain_deepstack(stack, head, s.float(), cos, sin, [f.float() for f in fs], r.to(cuda))[-1]
                        for s, fs, r in zip(seqs, feats, rows)])
    both = dict(deepstack_features=[torch.cat(f) for f in zip(*feats)], deepstack_rows=torch.cat([rows[0], rows[1] + 60]))
    cache = dec.new_cache(2, 200)
    got = dec.forward(torch.cat(seqs), cache, [60, 25], **both)
    T.close(got, want)
    # generate() hands them to the prompts' pass only
    u = torch.zeros(4, 2)
    ids = dec.generate(seqs, 4, u=u, temperature=0.0, **both)
    step = [got.float().argmax(-1)]
    for _ in range(3):
        step.append(dec.forward(dec.embed[step[-1]], cache, [1, 1]).float().argmax(-1))
    assert ids == torch.stack(step, 1).tolist()
    assert ids != dec.generate(seqs, 4, u=u, temperature=0.0)
    assert ops.device_error() == 0
