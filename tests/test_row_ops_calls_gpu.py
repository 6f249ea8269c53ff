"""The operators around a decoder's products as torch ops, at far positions, and their path through B200TextDecoder where layers
have no norms behind their blocks and where logits come in pieces.  Plain forms and their tolerances: test_decoder_gpu.py and
test_rope_gpu.py.

Far positions: the angle's two products and the constant 1 / (2 pi) are rounded to doubles, 2^-53 of the angle each and 0.6 of that for
the constant: 2^-51 |p f| covers them.  The angles wanted are made in 80-bit numbers, 2^11 finer."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

import rldx_b200  # noqa: E402,F401
import rldx_b200.torch_ops  # noqa: E402,F401
from rldx_b200 import ops  # noqa: E402
from rldx_b200.decoder import B200TextDecoder  # noqa: E402
from rldx_b200.rope import B200Rope  # noqa: E402
import test_decoder_gpu as T  # noqa: E402
from test_decoder_gpu import BF, CFG, VOCAB, r  # noqa: E402
from test_decoder_score_gpu import plain_rows  # noqa: E402

F16, F32, F64 = torch.float16, torch.float32, torch.float64


def test_torch_ops_are_the_functions(cuda):
    g = torch.Generator(device=cuda).manual_seed(2)

    def randn(*shape, dtype=BF):
        return torch.randn(*shape, device=cuda, generator=g).to(dtype)

    def same(a, b):
        assert len(a) == len(b) and all(x.dtype == y.dtype and x.is_contiguous() and torch.equal(x, y) for x, y in zip(a, b))

    op = torch.ops.b200msat
    q, k, freqs = randn(37, 6, 64), randn(37, 2, 64), 1e4 ** (-torch.arange(32, dtype=F64, device=cuda) / 32)
    one, three = torch.arange(37, device=cuda) + 900, torch.randint(900, (3, 37), device=cuda, generator=g)
    same(op.rope(q, k, one, freqs), ops.rope(q, k, one, freqs))
    same(op.rope(q, k, three, freqs, [12, 10, 10], True, True, 1.5, True),
         ops.rope(q, k, three, freqs, sections=[12, 10, 10], interleaved_sections=True, interleaved=True, factor=1.5, inverse=True))
    same(op.rope_rows(one, freqs), ops.rope_rows(one, freqs))
    same(op.rope_rows(three, freqs, [12, 10, 10], True, 1.5, True, F16),
         ops.rope_rows(three, freqs, sections=[12, 10, 10], interleaved_sections=True, factor=1.5, inverse=True, dtype=F16))
    y, h, w, v = randn(37, 72), randn(37, 72, dtype=F32), randn(5, 72), randn(4, 72)
    same(op.block_norms(y, h), ops.block_norms(y, h))
    vectors = dict(post_weight=w[0], post_bias=w[1], gate=v, pre_weight=w[2], pre_bias=w[3], mod_scale=randn(4, 72), mod_shift=w[4])
    same(op.block_norms(y, h, "layer", w[0], w[1], v, 0.3, "layer", w[2], w[3], vectors["mod_scale"], w[4], 10, True, 1e-5),
         ops.block_norms(y, h, post="layer", scale=0.3, pre="layer", rows_per_group=10, weight_plus_one=True, eps=1e-5, **vectors))
    with pytest.raises(ValueError, match="without a pre norm"):
        op.block_norms(y, h, pre="none")
    x, t = randn(37, 501), torch.randint(501, (37,), device=cuda, generator=g)
    same(op.token_logprobs(x, t), ops.token_logprobs(x, t))
    same(op.token_logprobs(x, t, 7), ops.token_logprobs(x, t, top=7))
    assert ops.device_error() == 0


@pytest.mark.parametrize("most", [2 ** 27, 2 ** 31, 2 ** 40])
def test_angles_of_far_positions(cuda, most):
    """As exact as fp32 up to 2^27 radians, and off by 2^-51 of the angle past it."""
    rng = np.random.default_rng(7)
    at = np.concatenate([rng.integers(-most, most, 500), [most - 1, 1 - most]])
    freqs = np.concatenate([[1.0], 1e6 ** (-np.arange(1, 32) / 32)])
    wide = at.astype(np.longdouble)[:, None] * freqs.astype(np.longdouble)
    cos, sin = ops.rope_rows(torch.from_numpy(at).to(cuda), torch.from_numpy(freqs).to(cuda))
    room = torch.from_numpy((np.abs(wide) * 2.0 ** -51).astype(np.float64)) + 2.0 ** -21
    assert most > 2 ** 27 or float(room.max()) <= 2.0 ** -24 + 2.0 ** -21
    for got, want in ((cos, np.cos(wide)), (sin, np.sin(wide))):
        want = torch.from_numpy(want.astype(np.float64))
        for part in got.cpu().double().chunk(2, 1):
            assert bool(((part - want).abs() <= room).all()), ((part - want).abs() / room).max()


def plain_scaled(stack, embed, head, ids, cos, sin, scale):
    """Logits of every position of plain layers whose blocks join the stream times `scale`: one rounding of the sum, and the norm of the
    unrounded one."""
    h, n = embed[ids], len(ids)
    pos = torch.arange(n, device=h.device)
    seen = pos <= pos[:, None]
    c, s = cos[:, None], sin[:, None]
    x = T.rms(h, stack.layers[0].input_layernorm.weight)
    for i, m in enumerate(stack.layers):
        a = m.self_attn
        q, k, v = (r(p(x)).unflatten(-1, (-1, CFG.head_dim)) for p in (a.q_proj, a.k_proj, a.v_proj))
        q, k = T.normed(q, a.q_norm.weight), T.normed(k, a.k_norm.weight)
        q, k = r(q * c + T.oq.rotate_half(q) * s), k * c + T.oq.rotate_half(k) * s
        k, v = (T.quantised(t).repeat_interleave(CFG.q_heads // CFG.kv_heads, 1) for t in (k, v))
        w = torch.einsum("qhd,khd->hqk", q, k) * CFG.head_dim ** -0.5
        w = w.masked_fill(~seen, float("-inf")).softmax(-1)
        sum_ = h + scale * r(a.o_proj(r(torch.einsum("hqk,khd->qhd", w, v).flatten(1))))
        h, x = r(sum_), r(T.normed(sum_, m.post_attention_layernorm.weight))
        gate, up = r(m.mlp.gate_proj(x)), r(m.mlp.up_proj(x))
        sum_ = h + scale * r(m.mlp.down_proj(r(r(torch.nn.functional.silu(gate)) * up)))
        after = stack.layers[i + 1].input_layernorm if i + 1 < len(stack.layers) else stack.norm
        h, x = r(sum_), r(T.normed(sum_, after.weight))
    return r(x @ head.t())


@pytest.mark.parametrize("scale", [0.5, 0.22])
@torch.no_grad()
def test_a_residual_scale_without_norms_behind_the_blocks(cuda, scale):
    stack, embed, head, _, _, plain = T.make(cuda)
    rope = B200Rope(CFG.head_dim, theta=CFG.rope_theta, device=cuda)
    dec = B200TextDecoder(stack.layers, stack.norm, embed, head, rope=rope, residual_scale=scale, device=cuda)
    assert dec.fused and not dec.after and not plain.fused
    g = torch.Generator().manual_seed(7)
    seqs = [torch.randint(VOCAB, (n,), generator=g).to(cuda) for n in (97, 5, 130)]
    want = [plain_scaled(stack, embed, head, s, *plain_rows_of_one_axis(rope, len(s), cuda), scale) for s in seqs]
    cache = dec.new_cache(3, 400)
    got = dec.forward(dec.embed[torch.cat([s[:-1] for s in seqs])], cache, [len(s) - 1 for s in seqs])
    T.close(got, torch.stack([w[-2] for w in want]))
    got = dec.forward(dec.embed[torch.stack([s[-1] for s in seqs])], cache, [1, 1, 1])
    T.close(got, torch.stack([w[-1] for w in want]))
    other = plain_scaled(stack, embed, head, seqs[2], *plain_rows_of_one_axis(rope, 130, cuda), 1.0)
    assert torch.nn.functional.cosine_similarity(got[2:].double(), other[-1:].double()).item() < 0.999  # (that the scale matters here)
    assert ops.device_error() == 0


def plain_rows_of_one_axis(rope, n, dev):
    """cos, sin of the places 0 .. n - 1 (the same on every axis)."""
    return plain_rows(rope.freqs, torch.arange(n, device=dev).expand(3, -1), rope.factor)


@torch.no_grad()
def test_scores_of_pieces_are_those_of_one(cuda):
    """Pieces of 1, 7 and 50 rows, which end inside prompts.  The rows of a product and of the log probabilities are each summed the
    same way wherever they stand, up to where a row's 16-byte vectors begin: 777 logits make that differ, so values are compared
    within the roundings of test_decoder_score_gpu.py and the numbers of tokens exactly."""
    dec = T.make(cuda)[-1]
    prompts = [torch.randint(VOCAB, (n,), generator=torch.Generator().manual_seed(n)).tolist() for n in (50, 1, 17, 33)]
    whole = dec.score(prompts, top=3)
    for rows in (1, 7, 50):
        dec.score_logits = rows * VOCAB
        for a, b in zip(whole, dec.score(prompts, top=3)):
            assert torch.equal(a.rank, b.rank) and torch.equal(a.top_ids, b.top_ids)
            for x, y in ((a.logprob, b.logprob), (a.entropy, b.entropy), (a.top_logprobs, b.top_logprobs)):
                assert x.shape == y.shape and bool(((x - y).abs() <= 2 * 2.0 ** -24 * (180 + 3 * 7) * (1 + x.abs()) * (1 + 7)).all())


@torch.no_grad()
def test_rows_of_any_layout(cuda):
    """Columns first, off 16 bytes or in wider rows: the same logits."""
    for kw in ({}, dict(residual_scale=0.5)):
        dec = T.make(cuda, **kw)[-1]
        rows = dec.embed[torch.arange(30, device=cuda)]
        want = dec.forward(rows, dec.new_cache(1, 64), [30])
        off = torch.zeros(30 * CFG.hidden + 1, dtype=BF, device=cuda)[1:].view(30, CFG.hidden)
        wide = torch.zeros(30, CFG.hidden + 3, dtype=BF, device=cuda)[:, 1: 1 + CFG.hidden]
        for x in (rows.t().contiguous().t(), off.copy_(rows), wide.copy_(rows)):
            assert torch.equal(dec.forward(x, dec.new_cache(1, 64), [30]), want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_logprobs_are_as_good_as_stated(cuda, dtype):
    """e = 2^-24 (140 + vocab / 680 + 3 D): 35 units of a weight and of the sums' fixed steps, 6 a chunk of a thread (a sum, and the move of
    its reference), at most vocab / 4096 + 1 chunks or 16; rows that rise slowly move the reference with every chunk."""
    vocab = 151680
    g = torch.Generator(device=cuda).manual_seed(4)
    rise = torch.linspace(-3, 0, vocab, device=cuda)
    x = torch.stack([rise, 20 * rise, rise.flip(0), torch.zeros(vocab, device=cuda), 0.01 * torch.randn(vocab, device=cuda, generator=g),
                     3 * torch.randn(vocab, device=cuda, generator=g), 2000 * rise]).to(dtype)
    for rows in (x, x.repeat(100, 1)):  # a cluster a row, and one CTA
        t = torch.randint(vocab, (len(rows),), device=cuda, generator=g)
        logprob, entropy, _, _, _ = ops.token_logprobs(rows, t)
        for a in range(0, len(rows), 70):
            at = slice(a, a + 70)
            y = rows[at].double()
            d = y - y.amax(1, keepdim=True)
            logs = torch.log_softmax(y, 1)
            p = logs.exp()
            mean, square = (p * d.abs()).sum(1), (p * d * d).sum(1)
            e = 2.0 ** -24 * (140 + vocab / 680 + 3 * mean)
            want = logs.gather(1, t[at, None])[:, 0]
            few = 4 * 2.0 ** -24
            assert bool(((logprob[at] - want).abs() <= e + few * (want.abs() + d.gather(1, t[at, None])[:, 0].abs())).all())
            want = -(p * logs).sum(1)
            assert bool(((entropy[at] - want).abs() <= e * (1 + mean) + 3 * 2.0 ** -24 * square + few * want).all())
