"""B200TextDecoder's rotation from positions, layers with norms behind their blocks, and scores, run together and against
plain layers.  Plain forms, their roundings and the tolerance of logits: test_decoder_gpu.py.  Scores are compared with 64-bit
ones of the decoder's own logits: 2^-24 (180 + 3 ln vocab) of their size, as derived for ops.token_logprobs."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from rldx_b200.decoder import B200TextDecoder  # noqa: E402
from rldx_b200.rope import B200Rope  # noqa: E402
import test_decoder_gpu as T  # noqa: E402
from test_decoder_gpu import BF, CFG, VOCAB, r  # noqa: E402
from types import SimpleNamespace as NS  # noqa: E402

SECTIONS = (12, 10, 10)


def axis_of(pair):  # interleaved
    a = pair % 3
    return a if pair < 3 * SECTIONS[a] else 0


def plain_rows(freqs, places, factor=1.0):
    """cos, sin [n, d] of positions [3, n] in 64 bits."""
    angle = torch.stack([places[axis_of(i)].double() * freqs[i] for i in range(freqs.numel())], 1).repeat(1, 2)
    return (angle.cos() * factor).float(), (angle.sin() * factor).float()


def plain_logits(layers, norm, embed, head, ids, cos, sin, scale):
    """Logits of every position, with norms behind the blocks; block_norms rounds the sum and the norm once each."""
    h, n = embed[ids], len(ids)
    pos = torch.arange(n, device=h.device)
    seen = pos <= pos[:, None]
    c, s = cos[:, None], sin[:, None]

    def rms(x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w

    x = T.rms(h, layers[0].input_layernorm.weight)  # (the first norm stands alone)
    for i, m in enumerate(layers):
        a = m.self_attn
        q, k, v = (r(x @ p.weight.t()).unflatten(-1, (-1, CFG.head_dim)) for p in (a.q_proj, a.k_proj, a.v_proj))
        q, k = T.normed(q, a.q_norm.weight), T.normed(k, a.k_norm.weight)
        q, k = r(q * c + T.oq.rotate_half(q) * s), k * c + T.oq.rotate_half(k) * s
        k, v = (T.quantised(t).repeat_interleave(CFG.q_heads // CFG.kv_heads, 1) for t in (k, v))
        w = torch.einsum("qhd,khd->hqk", q, k) * CFG.head_dim ** -0.5
        w = w.masked_fill(~seen, float("-inf")).softmax(-1)
        y = r(r(torch.einsum("hqk,khd->qhd", w, v).flatten(1)) @ a.o_proj.weight.t())
        g = h + scale * rms(y, m.post_attention_layernorm.weight)
        h, x = r(g), r(rms(g, m.pre_feedforward_layernorm.weight))
        y = r(x @ m.mlp.gate_proj.weight.t()), r(x @ m.mlp.up_proj.weight.t())
        y = r(r(r(torch.nn.functional.silu(y[0])) * y[1]) @ m.mlp.down_proj.weight.t())
        g = h + scale * rms(y, m.post_feedforward_layernorm.weight)
        h, x = r(g), r(rms(g, layers[i + 1].input_layernorm.weight if i + 1 < len(layers) else norm.weight))
    return r(x @ head.t())


def make(dev, scale=0.7, scaling=None, **kw):
    stack, embed, head, _, _, _ = T.make(dev)
    g = torch.Generator(device=dev).manual_seed(9)
    layers = []
    for m in stack.layers:
        new = [NS(weight=(1.0 + 0.2 * torch.randn(CFG.hidden, device=dev, generator=g)).to(BF).float()) for _ in range(2)]
        layers.append(NS(input_layernorm=m.input_layernorm, self_attn=m.self_attn, mlp=m.mlp, pre_feedforward_layernorm=m.post_attention_layernorm,
                         post_attention_layernorm=new[0], post_feedforward_layernorm=new[1]))
    rope = B200Rope(CFG.head_dim, theta=1e6, sections=SECTIONS, interleaved_sections=True, scaling=scaling, device=dev)
    dec = B200TextDecoder(layers, stack.norm, embed, head, rope=rope, residual_scale=scale, device=dev, **kw)
    return layers, stack.norm, embed, head, rope, dec


def close(got, want, factor=1.0):
    """T.close's 0.999 for a rotation of size one.  One that multiplies q and k by `factor` multiplies the scores, and what a moved code of
    k changes in them, by factor^2: to first order so do the weights and the attention's error, and 1 - cosine is of second order."""
    cos = torch.nn.functional.cosine_similarity(got.double(), want.double(), dim=-1)
    assert bool((1 - cos <= 0.001 * factor ** 4).all()), cos.min().item()


def a_vision_prompt(n):
    """Positions [3, n]: text, a grid of patches, text, far out."""
    at = torch.arange(n).expand(3, -1).clone() + 300000
    grid = torch.arange(24)
    at[0, 10:34] = at[0, 10]
    at[1, 10:34] = at[0, 10] + grid // 6
    at[2, 10:34] = at[0, 10] + grid % 6
    at[:, 34:] = at[:, 34:] - 34 + int(at[:, :34].max()) + 1 - 300000
    return at


@pytest.mark.parametrize("scaling", [None, {"type": "yarn", "factor": 16.0, "original": 32768}])
@torch.no_grad()
def test_norms_on_both_sides_and_positions_of_three_axes(cuda, scaling):
    layers, norm, embed, head, rope, dec = make(cuda, scaling=scaling)
    g = torch.Generator().manual_seed(7)
    seqs = [torch.randint(VOCAB, (n,), generator=g).to(cuda) for n in (97, 41)]
    places = [a_vision_prompt(97), torch.arange(41).expand(3, -1)]
    want = [plain_logits(layers, norm, embed, head, s, *plain_rows(rope.freqs, p.to(cuda), rope.factor), 0.7) for s, p in zip(seqs, places)]
    cache = dec.new_cache(2, 300)
    cut = [90, 40]
    got = dec.forward(dec.embed[torch.cat([s[:c] for s, c in zip(seqs, cut)])], cache, cut,
                      torch.cat([p[:, :c] for p, c in zip(places, cut)], 1))
    close(got, torch.stack([w[c - 1] for w, c in zip(want, cut)]), rope.factor)
    got = dec.forward(dec.embed[torch.cat([s[c:] for s, c in zip(seqs, cut)])], cache, [7, 1],
                      torch.cat([p[:, c:] for p, c in zip(places, cut)], 1))
    close(got, torch.stack([w[-1] for w in want]), rope.factor)
    assert ops.device_error() == 0


@torch.no_grad()
def test_scores_are_those_of_the_logits(cuda):
    layers, norm, embed, head, rope, dec = make(cuda)
    prompts = [torch.randint(VOCAB, (n,), generator=torch.Generator().manual_seed(n)) for n in (50, 1, 17)]
    got = dec.score([p.tolist() for p in prompts], top=4)
    at = dec.score([p.tolist() for p in prompts], top=4, positions=[torch.arange(len(p)) for p in prompts])
    ids = torch.cat(prompts).to(cuda)
    normed = dec._run(dec.embed[ids], dec.new_cache(3, 100), [50, 1, 17])
    logits = ops.linear(normed(slice(0, 68)).contiguous(), dec.lm_head)
    room = 2.0 ** -24 * (180 + 3 * math.log(VOCAB))
    for prompt, x, s, t in zip(prompts, logits.split([50, 1, 17]), got, at):
        n = len(prompt)
        assert all(torch.equal(a, b) for a, b in zip(s, t))
        assert s.logprob.shape == s.entropy.shape == s.rank.shape == (n,) and s.top_ids.shape == s.top_logprobs.shape == (n, 4)
        assert float(s.logprob[-1]) == 0 and int(s.rank[-1]) == -1
        logs = torch.log_softmax(x.double(), -1)
        given = prompt[1:].to(cuda)
        scale = room * (1 + logs.abs().max())
        assert bool(((s.logprob[:-1].double() - logs[:-1].gather(1, given[:, None])[:, 0]).abs() <= scale).all())
        assert bool(((s.entropy.double() + (logs.exp() * logs).sum(-1)).abs() <= scale * (1 + math.log(VOCAB))).all())
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices
        assert torch.equal(s.top_ids, order[:, :4]) and bool(((s.top_logprobs.double() - logs.gather(1, s.top_ids)).abs() <= scale).all())
        assert torch.equal(s.rank[:-1].long(), (order[:-1] == given[:, None]).int().argmax(-1))
        T.close(x, plain_logits(layers, norm, embed, head, prompt.to(cuda), *plain_rows(rope.freqs, torch.arange(n, device=cuda).expand(3, -1)), 0.7))


@torch.no_grad()
def test_scores_of_rows_with_targets_and_of_generated_tokens(cuda):
    dec = T.make(cuda)[-1]
    prompts = [[1, 5, 9, 200], list(range(40, 140)), [700]]
    u = torch.rand(6, 3, generator=torch.Generator().manual_seed(1))
    plain = dec.generate(prompts, 6, u=u, temperature=0.9, top_p=0.95)
    stop = plain[1][2]
    forward, seen = dec.forward, []

    def recorded(*a, **kw):
        seen.append(forward(*a, **kw))
        return seen[-1]

    dec.forward = recorded
    ids, scores = dec.generate(prompts, 6, u=u, temperature=0.9, top_p=0.95, logprobs=3, stop_ids=[stop])
    dec.forward = forward
    assert ids[0] == plain[0] and ids[1] == plain[1][: plain[1].index(stop) + 1] and len(seen) == 6
    for i, logits in enumerate(seen):  # (a row's sums depend on where its 16-byte vectors begin: the same rows of the same logits)
        want = ops.token_logprobs(logits, torch.tensor([p[i] for p in plain], device=cuda), top=3)
        for q, (new, s) in enumerate(zip(ids, scores)):
            assert s.logprob.shape == (len(new),) and s.top_ids.shape == (len(new), 3)
            if i < len(new):
                assert new[i] == plain[q][i] and all(torch.equal(a[i], b[q]) for a, b in zip(s, want))
    rows = [dec.embed[torch.tensor(p, device=cuda)] for p in prompts]
    a = dec.score(prompts, top=2)
    b = dec.score(rows, top=2, targets=[p[1:] + [-1] for p in prompts])
    assert all(torch.equal(x, y) for s, t in zip(a, b) for x, y in zip(s, t))
    c = dec.score(rows, top=2)
    assert all(bool((s.logprob == 0).all()) and torch.equal(s.top_ids, t.top_ids) for s, t in zip(c, a))
    ids, scores = dec.generate(prompts, 0, u=u[:0], logprobs=2)
    assert ids == [[], [], []] and scores[1].top_ids.shape == (0, 2)
    assert ops.device_error() == 0


@torch.no_grad()
def test_deepstack_features_join_before_the_next_norm(cuda):
    """Features of zero change nothing but the path that adds them, up to one more rounding of the norm's input."""
    dec = make(cuda)[-1]
    rows = dec.embed[torch.randint(VOCAB, (30,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(2))]
    zero = [torch.zeros(5, CFG.hidden, dtype=BF, device=cuda)] * 3
    a = dec.forward(rows, dec.new_cache(1, 40), [30])
    b = dec.forward(rows, dec.new_cache(1, 40), [30], deepstack_features=zero, deepstack_rows=torch.arange(3, 8))
    T.close(b, a)
    ones = [torch.ones(5, CFG.hidden, dtype=BF, device=cuda)] * 3
    c = dec.forward(rows, dec.new_cache(1, 40), [30], deepstack_features=ones, deepstack_rows=torch.arange(25, 30))
    assert torch.nn.functional.cosine_similarity(c.float(), a.float(), dim=-1).max() < 0.999


@torch.no_grad()
def test_a_rope_gives_the_tables_logits(cuda):
    stack, embed, head, cos, sin, dec = T.make(cuda)
    rope = B200Rope(CFG.head_dim, theta=CFG.rope_theta, device=cuda)
    table = rope.rows(torch.arange(600, device=cuda))
    one = B200TextDecoder(stack.layers, stack.norm, embed, head, *table, device=cuda)
    two = B200TextDecoder(stack.layers, stack.norm, embed, head, rope=rope, device=cuda)
    prompts = [[1, 5, 9, 200], list(range(40, 140))]
    u = torch.rand(8, 2, generator=torch.Generator().manual_seed(4))
    assert one.generate(prompts, 8, u=u, temperature=0.8) == two.generate(prompts, 8, u=u, temperature=0.8)
    at = [torch.arange(4) + 5, torch.arange(100) + 9]
    assert one.generate(prompts, 8, u=u, temperature=0.8, positions=at) == two.generate(prompts, 8, u=u, temperature=0.8, positions=at)
