"""Rotary positions, block norms and log probabilities, the parts that need no GPU: refusals before any device work,
frequencies, the ctypes mirrors."""

import ctypes as C
import math

import pytest
import torch

import rldx_b200  # noqa: F401
from rldx_b200 import _lib, ops
from rldx_b200.rope import B200Rope, frequencies

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def test_struct_sizes():
    assert C.sizeof(_lib.RopePlan) == 3 * 8 + 11 * 4 + 4
    assert C.sizeof(_lib.RopeHeads) == 6 * 8 + 8
    assert C.sizeof(_lib.BlockNormsDesc) == 20 * 8 + 9 * 4 + 4


def test_frequencies():
    f, m = frequencies(64, 1e4)
    assert m == 1.0 and f.dtype == F64 and torch.equal(f, 1e4 ** (-torch.arange(0, 64, 2, dtype=F64) / 64))
    assert torch.equal(frequencies(64, 1e4, {"type": "linear", "factor": 4.0})[0], f / 4)
    g, _ = frequencies(64, 1e4, {"type": "ntk", "factor": 4.0})
    assert g[0] == 1 and abs(float(g[-1] / f[-1]) - 0.25) < 1e-12  # the fastest stays, the slowest is divided
    y, m = frequencies(128, 1e6, {"type": "yarn", "factor": 8.0, "original": 32768})
    f, _ = frequencies(128, 1e6)
    turns = 32768 * f / (2 * math.pi)
    assert torch.equal(y[turns > 40], f[turns > 40]) and torch.allclose(y[turns < 0.8], f[turns < 0.8] / 8, rtol=1e-15)
    assert bool((y[1:] < y[:-1]).all()) and m == 0.1 * math.log(8.0) + 1.0
    assert frequencies(128, 1e6, {"type": "yarn", "factor": 8.0, "original": 32768, "attention_factor": 1.0})[1] == 1.0


@pytest.mark.parametrize("scaling", [{"type": "other", "factor": 2.0}, {"type": "linear", "factor": 0.0}, {"type": "linear", "factor": -1.0},
                                     {"type": "yarn", "factor": 2.0}, {"type": "linear", "factor": 2.0, "orignal": 5},
                                     {"type": "yarn", "factor": 2.0, "original": 0}, {"type": "linear", "factor": math.nan},
                                     {"type": "yarn", "factor": 2.0, "original": 10, "beta_fast": 1.0, "beta_slow": 2.0}])
def test_scalings_that_are_refused(scaling):
    with pytest.raises(ValueError):
        frequencies(64, 1e4, scaling)


def test_plans_that_are_refused():
    for kw in (dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=0), dict(sections=(10, 10)), dict(sections=()),
               dict(sections=(40, -8)), dict(sections=(8, 8, 8, 4, 4)), dict(freqs=torch.ones(31)),
               dict(freqs=torch.ones(32), scaling={"type": "linear", "factor": 2.0}), dict(theta=-1.0)):
        with pytest.raises(ValueError):
            B200Rope(64, device="cpu", **kw)
    rope = B200Rope(64, sections=(16, 8, 8), device="cpu")
    assert rope.axes == 3 and rope.freqs.shape == (32,)
    with pytest.raises(ValueError, match="64"):
        rope(torch.zeros(1, 1, 32), None, torch.zeros(3, 1, dtype=torch.int64))
    with pytest.raises(ValueError, match="halves"):
        B200Rope(64, interleaved=True, device="cpu").rows(torch.zeros(1, dtype=torch.int64))


def test_rope_refusals():
    q, k = torch.zeros(6, 4, 64, dtype=BF), torch.zeros(6, 2, 64, dtype=BF)
    at, f = torch.arange(6), torch.ones(32, dtype=F64)

    def refused(kind, match, q=q, k=k, at=at, f=f, **kw):
        with pytest.raises(kind, match=match):
            ops.rope(q, k, at, f, **kw)

    refused(ValueError, "CUDA")  # everything else is right
    refused(TypeError, "tensor", q=None)
    refused(TypeError, "bfloat16", q=q.double(), k=k.double())
    refused(TypeError, "one type", k=k.float())
    refused(TypeError, "int32 or int64", at=at.float())
    refused(TypeError, "float64", f=f.float())
    refused(ValueError, "tokens, heads", q=q[:5])
    refused(ValueError, "tokens, heads", k=k[..., :32])
    refused(ValueError, "side by side", q=torch.zeros(6, 4, 128, dtype=BF)[..., ::2])
    refused(ValueError, "no heads", k=k[:, :0])
    refused(ValueError, "pairs", f=torch.ones(33, dtype=F64))
    refused(ValueError, "512", f=torch.ones(513, dtype=F64))
    refused(ValueError, "freqs", f=torch.ones(64, dtype=F64)[::2])
    refused(ValueError, "freqs", f=torch.ones(0, dtype=F64))
    refused(ValueError, "axes", at=torch.zeros(3, 6, dtype=torch.int64))
    refused(ValueError, "axes", sections=(16, 16))
    refused(ValueError, "add up", at=torch.zeros(2, 6, dtype=torch.int64), sections=(16, 15))
    refused(ValueError, "counts", at=torch.zeros(2, 6, dtype=torch.int64), sections=(33, -1))
    refused(ValueError, "1 to 4", at=torch.zeros(5, 6, dtype=torch.int64), sections=(32, 0, 0, 0, 0))
    refused(TypeError, "", sections=5)
    refused(ValueError, "side by side", at=torch.zeros(12, dtype=torch.int64)[::2])
    refused(TypeError, "", factor="two")
    refused(ValueError, "out_k", k=None, out_k=k)
    refused(TypeError, "type", out_q=q.float())
    refused(ValueError, "shape", out_q=torch.zeros(6, 3, 64, dtype=BF))
    wide = torch.zeros(6, 6 * 64, dtype=BF)
    refused(ValueError, "shares memory", q=wide[:, : 4 * 64].unflatten(1, (4, 64)), k=None, out_q=wide[:, 64: 5 * 64].unflatten(1, (4, 64)))
    refused(ValueError, "shares memory", q=wide[:, : 4 * 64].unflatten(1, (4, 64)), k=wide[:, 4 * 64:].unflatten(1, (2, 64)),
            out_q=wide[:, 64: 5 * 64].unflatten(1, (4, 64)))
    one = torch.zeros(6, 4, 64, dtype=BF)
    refused(ValueError, "share", q=q, k=k, out_q=one, out_k=one[:, :2])
    refused(ValueError, "share", q=q, k=q[:, 1:3], out_q=q)
    both = wide.unflatten(1, (6, 64))
    refused(ValueError, "CUDA", q=both[:, :4], k=both[:, 4:], out_q=both[:, :4], out_k=both[:, 4:])  # columns of one buffer are apart
    refused(ValueError, "CUDA", q=both[:, :4], k=None, out_q=torch.zeros(4, 6, 64, dtype=BF).transpose(0, 1))
    with pytest.raises(TypeError, match="dtype"):
        ops.rope_rows(at, f, dtype=F64)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_rows(at, f)


def test_block_norms_refusals():
    y, h = torch.zeros(6, 40, dtype=BF), torch.zeros(6, 40, dtype=BF)
    v, groups = torch.zeros(40, dtype=BF), torch.zeros(3, 40, dtype=BF)

    def refused(kind, match, y=y, h=h, **kw):
        with pytest.raises(kind, match=match):
            ops.block_norms(y, h, **kw)

    refused(ValueError, "CUDA", post="rms", post_weight=v, gate=groups, rows_per_group=2, mod_scale=v, mod_shift=groups.float()[:, :40].to(BF))
    refused(TypeError, "tensor", h=None)
    refused(ValueError, "post and pre", post="batch")
    refused(ValueError, "post and pre", pre="group")
    refused(TypeError, "bfloat16", y=y.double())
    refused(TypeError, "residual", h=h.half())
    refused(ValueError, "residual", h=h[:5])
    refused(ValueError, "row-major", y=torch.zeros(40, 6, dtype=BF).t())
    refused(ValueError, "row-major", y=torch.zeros(2, 6, 40, dtype=BF))
    refused(ValueError, "14336", y=torch.zeros(1, 14337), h=torch.zeros(1, 14337))
    refused(ValueError, "14336", y=torch.zeros(1, 0), h=torch.zeros(1, 0))
    refused(TypeError, "all", gate=v, pre_weight=v.float())
    refused(TypeError, "all", gate=v.half())
    refused(ValueError, "pre_weight", pre_weight=v[:39])
    refused(ValueError, "pre_weight", pre_weight=groups, rows_per_group=2)
    refused(ValueError, "gate", gate=torch.zeros(80, dtype=BF)[::2])
    refused(ValueError, "rows_per_group", gate=groups)
    refused(ValueError, "each group", gate=groups, rows_per_group=3)
    refused(ValueError, "negative", rows_per_group=-1)
    refused(TypeError, "type", out=torch.zeros(6, 40))
    refused(ValueError, "shape", out=torch.zeros(5, 40, dtype=BF))
    refused(ValueError, "shape", out_residual=torch.zeros(1, 40, dtype=BF).expand(6, -1))
    refused(ValueError, "no out", pre=None, out=torch.zeros(6, 40, dtype=BF))
    one = torch.zeros(7, 40, dtype=BF)
    refused(ValueError, "shares memory", y=one[:6], out=one[1:])
    refused(ValueError, "share memory", out=one[:6], out_residual=one[:6])
    refused(ValueError, "shares memory", gate=one[3], out=one[:6])
    refused(ValueError, "CUDA", y=y, h=h, out=y, out_residual=h)
    wide = torch.zeros(6, 160, dtype=BF)
    refused(ValueError, "CUDA", y=wide[:, :40], h=wide[:, 40:80], out=wide[:, 80:120], out_residual=wide[:, 120:])


def test_logprobs_refusals():
    x, t = torch.zeros(3, 50), torch.zeros(3, dtype=torch.int64)
    for kind, args, kw in ((TypeError, (None, t), {}), (TypeError, (x.double(), t), {}), (ValueError, (x[0], t), {}), (ValueError, (x.t(), t), {}),
                           (ValueError, (x, t[:2]), {}), (ValueError, (x, t.int()), {}), (ValueError, (x[:, :0], t), {}), (ValueError, (x, t), dict(top=33)),
                           (ValueError, (x, t), dict(top=-1)), (ValueError, (x[:, :4], t), dict(top=5)), (TypeError, (x, t), dict(top=1.5)),
                           (ValueError, (x, t), dict(top=2 ** 40)), (ValueError, (x, t), {})):
        with pytest.raises(kind):
            ops.token_logprobs(*args, **kw)
    with pytest.raises(ValueError, match="CUDA"):
        ops.token_logprobs(x, t, top=32)


def test_library_refuses_before_any_device_work(lib):
    p = _lib.RopePlan(256, 0, 256, 1, 1, (C.c_int * 4)(), 0, 32, 0, 0, 1.0)
    h = _lib.RopeHeads(256, 512, 128, 64, 128, 64, 2)
    arg, no = _lib.RLDX_ERR_ARG, _lib.RLDX_ERR_UNSUPPORTED

    def rope(p=p, h=h, n=1, tokens=4, d=64, dtype=0):
        return lib.rldx_rope(C.byref(p) if p else None, C.byref(h) if h else None, n, tokens, d, dtype, None)

    def but(struct, **kw):
        s = type(struct).from_buffer_copy(struct)
        for k, v in kw.items():
            setattr(s, k, v)
        return s

    assert rope(tokens=0) == _lib.RLDX_OK
    assert rope(p=None) == arg and rope(h=None) == arg and rope(n=3) == arg and rope(tokens=-1) == arg and rope(d=62) == arg
    assert rope(dtype=7) == no and rope(p=but(p, pairs=0)) == no and rope(p=but(p, pairs=513)) == no and rope(p=but(p, axes=5)) == no
    assert rope(p=but(p, axes=2)) == arg and rope(p=but(p, freqs=None)) == arg and rope(p=but(p, freqs=260)) == arg
    assert rope(p=but(p, positions=260)) == arg
    for field, value in (("inp", None), ("out", None), ("heads", 0), ("out_head", 32), ("out_tok", 64), ("in_tok", -1), ("inp", 257)):
        assert rope(h=but(h, **{field: value})) == arg, field
    assert lib.rldx_rope_rows(C.byref(p), 4, None, 256, 0, None) == arg and lib.rldx_rope_rows(None, 4, 256, 256, 0, None) == arg
    assert lib.rldx_rope_rows(C.byref(p), 0, 256, 256, 2, None) == _lib.RLDX_OK

    d = _lib.BlockNormsDesc(branch=256, residual=256, residual_out=256, out=256, ld_branch=40, ld_residual=40, ld_residual_out=40, ld_out=40, rows=0,
                            width=40, post=0, pre=1, dtype=0, residual_dtype=2, vector_dtype=0, scale=1.0, eps=1e-6)
    assert lib.rldx_block_norms(C.byref(d), None) == _lib.RLDX_OK and lib.rldx_block_norms(None, None) == arg
    for kw, rc in ((dict(width=0), no), (dict(width=20000), no), (dict(rows=-1), arg), (dict(post=3), arg), (dict(out=None), arg), (dict(ld_out=39), arg),
                   (dict(residual_dtype=1), no), (dict(vector_dtype=1), no), (dict(dtype=5), no), (dict(post_weight=256), arg), (dict(ld_branch=-1), arg),
                   (dict(pre=0), arg), (dict(ld_gate=40), arg), (dict(ld_gate=8, rows_per_group=1), arg), (dict(gate=257), arg), (dict(branch=257), arg),
                   (dict(weight_plus_one=1), arg), (dict(rows_per_group=-1), arg)):
        assert lib.rldx_block_norms(C.byref(but(d, **kw)), None) == rc, kw

    def lp(logits=256, ld=50, rows=3, vocab=50, dtype=2, tokens=256, top=2, out=256):
        return lib.rldx_token_logprobs(logits, ld, rows, vocab, dtype, tokens, top, out, out, out, out, out, None)

    assert lp(rows=0) == _lib.RLDX_OK
    assert lp(logits=None) == arg and lp(logits=258) == arg and lp(tokens=None) == arg and lp(out=None) == arg and lp(rows=-1) == arg
    assert lp(vocab=0) == arg and lp(ld=-1) == arg and lp(dtype=3) == no and lp(top=33) == no and lp(top=-1) == no and lp(vocab=1, top=2) == no
    assert lp(vocab=2 ** 28 + 1) == no and lp(rows=2 ** 29) == no


def test_fake_shapes():
    import rldx_b200.torch_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        q, k = torch.ops.b200msat.rope(torch.empty(7, 8, 64, dtype=BF), torch.empty(7, 2, 64, dtype=BF), torch.empty(3, 7, dtype=torch.int64),
                                       torch.empty(32, dtype=F64), [16, 8, 8])
        assert q.shape == (7, 8, 64) and k.shape == (7, 2, 64) and q.dtype == BF
        cos, sin = torch.ops.b200msat.rope_rows(torch.empty(3, 7, dtype=torch.int64), torch.empty(32, dtype=F64), [16, 8, 8], dtype=BF)
        assert cos.shape == sin.shape == (7, 64) and cos.dtype == BF
        h, n = torch.ops.b200msat.block_norms(torch.empty(5, 40, dtype=BF), torch.empty(5, 40))
        assert h.dtype == F32 and n.dtype == BF and h.shape == n.shape == (5, 40)
        out = torch.ops.b200msat.token_logprobs(torch.empty(5, 99, dtype=BF), torch.empty(5, dtype=torch.int64), 3)
        assert [t.dtype for t in out] == [F32, F32, torch.int32, torch.int64, F32] and out[3].shape == out[4].shape == (5, 3)


def test_decoder_refusals():
    from test_decoder_host import FFN, HEAD, HIDDEN, VOCAB, layer, make, weight
    from rldx_b200.decoder import B200TextDecoder

    def sandwich():
        m = layer()
        m.pre_feedforward_layernorm, m.post_feedforward_layernorm = weight(HIDDEN), weight(HIDDEN)
        return m

    def build(layers=None, **kw):
        kw.setdefault("rope", B200Rope(HEAD, device="cpu"))
        return B200TextDecoder(layers or [layer(), layer()], weight(HIDDEN), torch.zeros(VOCAB, HIDDEN), torch.zeros(VOCAB, HIDDEN), device="cpu", **kw)

    assert not make().fused and not build().fused and build(residual_scale=0.5).fused and build([sandwich(), sandwich()]).after
    with pytest.raises(NotImplementedError, match="every layer"):
        build([sandwich(), layer()])
    half = sandwich()
    half.post_feedforward_layernorm = None
    with pytest.raises(NotImplementedError, match="every layer"):
        build([half, half])
    with pytest.raises(ValueError, match="cos and sin, or a rope"):
        build(rope=None)
    with pytest.raises(ValueError, match="cos and sin, or a rope"):
        build(cos=torch.zeros(4, HEAD), sin=torch.zeros(4, HEAD))
    with pytest.raises(ValueError, match="cos and sin, or a rope"):
        build(rope=None, cos=torch.zeros(4, HEAD))
    for bad in (B200Rope(HEAD, rotary_dim=32, device="cpu"), B200Rope(HEAD, interleaved=True, device="cpu"), B200Rope(2 * HEAD, device="cpu")):
        with pytest.raises(ValueError, match="halves of whole heads"):
            build(rope=bad)
    dec = build(rope=B200Rope(HEAD, sections=(16, 8, 8), device="cpu"))
    cache = dec.new_cache(2, 256)
    rows = torch.zeros(3, HIDDEN, dtype=BF)
    for at in (torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, dtype=torch.int64), torch.zeros(3)):
        with pytest.raises(ValueError, match="positions must"):
            dec.forward(rows, cache, [1, 2], at)
    u = torch.zeros(2, 2)
    with pytest.raises(ValueError, match="positions must give"):
        dec.generate([[1], [2, 3]], 2, u=u, positions=[torch.zeros(3, 1), torch.zeros(2, 2)])
    with pytest.raises(ValueError, match="logprobs must be"):
        dec.generate([[1], [2, 3]], 2, u=u, logprobs=33)
    for kw, match in ((dict(top=33), "top must be"), (dict(top=-1), "top must be"), (dict(targets=[[1], [2]]), "targets must give"),
                      (dict(targets=[[1], [VOCAB, 2]]), "targets must be below"), (dict(positions=[torch.zeros(4, 1), torch.zeros(3, 2)]), "positions must give"),
                      (dict(cache=dec.new_cache(3, 256)), "the cache has 3 sequences")):
        with pytest.raises(ValueError, match=match):
            dec.score([[1], [2, 3]], **kw)
    with pytest.raises(ValueError, match="no token"):
        dec.score([[1], []])
    with pytest.raises(ValueError, match="no token"):
        dec.score([])
    for ids in ([VOCAB], [-1], torch.tensor([0, VOCAB])):
        with pytest.raises(ValueError, match="ids must be among"):
            dec.score([[1], ids])
        with pytest.raises(ValueError, match="ids must be among"):
            dec.generate([[1], ids], 2, u=u)
    with pytest.raises(RuntimeError, match="free pages"):
        dec.score([[1], [2] * 200], cache=dec.new_cache(2, 1))
    assert cache.tokens == [0, 0] and FFN
