"""Text decoding with the VLM backbone's layers over a 4-bit key / value cache.

The backbone chains (`rldx_b200.llm`) prefill a fixed sequence; this module keeps the keys and values
and produces tokens, one path through the decoding operators of `rldx_b200.ops`:

    n = rmsnorm(h); qkv = n Wqkv^T
    q = qkv_rope_append(qkv, ...)      per-head norms, rotation, 4-bit write into the cache
    a = kv4_attention(q, cache, ...)   over the whole sequence, or a sliding window and sinks
    h = h + a Wo^T; h = h + swiglu(rmsnorm(h) [Wg; Wu]^T) Wd^T
    token = sample(logits of the last rows, u, temperature, top_k, top_p, min_p)

    cache = B200KV4Cache(layers, kv_heads, head_dim, seqs=4, max_tokens=4096)
    decoder = B200TextDecoder(decoder_layers, norm, embed, lm_head, cos, sin)
    out = decoder.generate(prompts, 64, cache=cache, u=torch.rand(64, 4), temperature=0.7, top_p=0.9)
    scores = decoder.score(prompts, top=5)   # log probabilities of the prompts' tokens, alternatives

`decoder_layers` are Qwen3 text decoder layers (the attribute names that B200LLMChain takes), `cos` and
`sin` their RoPE tables [positions, head_dim]; with a B200Rope in their place (rope=) there is no table, positions may be of
several axes and far ones (as exact as fp32 up to 2^27).  Layers with norms behind their blocks too (pre_feedforward_layernorm and
post_feedforward_layernorm beside the other two), or a residual_scale, run through block_norms, which makes the sum
and both norms in one pass.  Prompts of a vision tower bring positions and deepstack
features of their own; everything that cannot be run is refused before the cache changes.  `python -m rldx_b200.decoder` decodes with random
weights.
"""

from __future__ import annotations

import argparse
import ctypes as C
import operator
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib, ops
from .llm import _raw_layer
from .rope import B200Rope

BF = torch.bfloat16


class Scores(NamedTuple):
    """What ops.token_logprobs gives of one sequence's tokens: logprob, entropy [n] fp32, rank [n] int32, top_ids [n, top] int64,
    top_logprobs [n, top] fp32."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    rank: torch.Tensor
    top_ids: torch.Tensor
    top_logprobs: torch.Tensor


class B200KV4Cache:
    """Pages of the 4-bit cache of `layers` layers for `seqs` sequences: a pool per layer, one page
    table, the lengths, and the list of free pages (on the host).  `max_tokens` bounds all
    sequences together, rounded up to pages."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, seqs: int, max_tokens: int, page_size: int = 64,
                 device="cuda"):
        if layers <= 0 or seqs <= 0 or max_tokens <= 0:
            raise ValueError("layers, seqs and max_tokens must be positive")
        self.page_size, self.seqs = int(page_size), int(seqs)
        self.pages = -(-int(max_tokens) // self.page_size) + seqs  # a sequence's last page may be part empty
        self.device = torch.device(device)
        self.pools = [ops.kv4_cache(self.pages, kv_heads, head_dim, page_size, device=self.device) for _ in range(layers)]
        self.table = torch.full((seqs, self.pages), -1, dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device=self.device)
        self.tokens = [0] * seqs  # host copies
        self._held = [[] for _ in range(seqs)]
        self._free = list(range(self.pages - 1, -1, -1))

    @property
    def free_tokens(self) -> int:
        return len(self._free) * self.page_size

    def room(self, new: Sequence[int]) -> list:
        """Pages that new[s] more tokens of each sequence need; raises where the cache has not so many."""
        if len(new) != self.seqs or any(n < 0 for n in new):
            raise ValueError(f"new must give a count for each of the {self.seqs} sequences")
        need = [-(-(t + n) // self.page_size) - len(h) for t, n, h in zip(self.tokens, new, self._held)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache has {len(self._free)} free pages, {sum(need)} are needed")
        return need

    def extend(self, new: Sequence[int]) -> None:
        """Makes room for new[s] more tokens of each sequence: lengths and pages cover them after."""
        need = self.room(new)
        seq, col, page = [], [], []
        for s, n in enumerate(need):
            for _ in range(n):
                seq.append(s)
                col.append(len(self._held[s]))
                page.append(self._free.pop())
                self._held[s].append(page[-1])
        if page:
            at = torch.tensor([seq, col, page], device=self.device)
            self.table[at[0], at[1]] = at[2].to(torch.int32)
        self.tokens = [t + n for t, n in zip(self.tokens, new)]
        self.lengths.copy_(torch.tensor(self.tokens, dtype=torch.int32))

    def release(self, seq: int) -> None:
        """Forgets a sequence; its pages are free again."""
        self._free.extend(reversed(self._held[seq]))
        self._held[seq] = []
        self.tokens[seq] = 0
        self.table[seq] = -1
        self.lengths[seq] = 0


def _whole(given, name: str, as_values: bool = False) -> torch.Tensor:
    """Whole numbers as int64 on the host.  Others are refused, not cut: floats (as_values: those that are not whole) and bools."""
    t = torch.as_tensor(given)
    if t.numel():  # (an empty list comes as floats)
        ok = t.dtype != torch.bool and not t.is_complex()
        if ok and t.is_floating_point():
            ok = as_values and bool(((t == t.trunc()) & (t.abs() < 2.0 ** 53)).all())
        if not ok:
            raise ValueError(f"{name} must be whole numbers, got {t.dtype}")
    return t.to("cpu", torch.int64)


def _refuse_other_norm(norm, name: str) -> None:
    """Raises for a norm that is not x / rms(x) * weight.  The weights alone do not say (some count from one), so a module that can
    be called is asked: a weight taken from the other of the two is off by all of x / rms(x), roundings by a few 2^-8 of the result."""
    if norm is None:
        return
    if getattr(norm, "bias", None) is not None:
        raise NotImplementedError(f"{name} has a bias, which an RMSNorm has not")
    if not callable(norm):
        return
    w = norm.weight.detach()
    n = w.shape[0]
    x = torch.linspace(-1.0, 2.0, n, device=w.device, dtype=torch.float32).to(w.dtype)
    with torch.no_grad():
        got = norm(x.repeat(2, 1))[0].float()
    x = x.float()
    hat = x * torch.rsqrt((x * x).mean())
    want = hat * w.float()
    if not bool(((got - want).abs() <= 2.0 ** -6 * (want.abs() + hat.abs())).all()):
        raise NotImplementedError(f"{name} is not x / rms(x) * weight (1 + weight, a mean taken off, or another norm)")


def _refuse_other_mlp(layer, i: int) -> None:
    """Raises for an activation other than SiLU, where the layer has one to ask."""
    act = getattr(layer.mlp, "act_fn", None)
    if act is None:
        return
    name = act.lower() if isinstance(act, str) else None
    x = torch.linspace(-8.0, 8.0, 65, device=layer.mlp.gate_proj.weight.device)
    if name is None:
        with torch.no_grad():
            silu = bool(((act(x) - torch.nn.functional.silu(x)).abs() <= 2.0 ** -8 * (1 + x.abs())).all())
    else:
        silu = name in ("silu", "swish")
    if not silu:
        raise NotImplementedError(f"layer {i}'s MLP does not gate with SiLU")


def _refuse_other_attention(layer, i: int) -> None:
    """Raises for scores other than q k / sqrt(head_dim), where the layer says how it makes them."""
    a = layer.self_attn
    scale, d = getattr(a, "scaling", None), a.q_norm.weight.shape[0]
    if scale is not None and abs(float(scale) * d ** 0.5 - 1) > 1e-5:
        raise NotImplementedError(f"layer {i}'s attention scales by {float(scale)}, not by head_dim ** -0.5 = {d ** -0.5}")
    if getattr(a, "attn_logit_softcapping", None) is not None:
        raise NotImplementedError(f"layer {i}'s attention caps its scores")


class B200TextDecoder:
    """Qwen3 decoder layers, embedding and output projection over a B200KV4Cache.

    Layers in a LayerWrapper that compresses video tokens (B200LLMChain's compress_info) would have to drop tokens from
    the cache of the layers after it, which no page table here can say: they are refused unless
    ignore_compression says that no prompt has what the wrapper compresses (it leaves one frame, and text, as
    they are).  The norms are x / rms(x) * weight, the MLP's activation SiLU, the scores q k / sqrt(head_dim): layers whose modules
    say otherwise are refused (norms of 1 + weight among them; their weights alone cannot tell)."""

    score_logits = 2 ** 29  # that score() makes at a time: a gibibyte

    def __init__(self, layers, norm, embed: torch.Tensor, lm_head: torch.Tensor, cos: Optional[torch.Tensor] = None,
                 sin: Optional[torch.Tensor] = None, *, window: int = 0, sinks: int = 0, device=None, ignore_compression: bool = False,
                 rope: Optional[B200Rope] = None, residual_scale: float = 1.0):
        layers = list(layers)
        if (rope is None) == (cos is None) or (cos is None) != (sin is None):
            raise ValueError("the decoder takes cos and sin, or a rope")
        for i, wrap in enumerate(layers):
            if _raw_layer(wrap) is not wrap and wrap.layer_idx == wrap.internal_projection and not ignore_compression:
                raise NotImplementedError(f"layer {i} compresses video tokens, which the decoder does not; ignore_compression=True "
                                          "where no prompt has more than one frame")
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        layers = [_raw_layer(layer) for layer in layers]
        a0 = layers[0].self_attn
        for m in layers:
            a = m.self_attn
            if getattr(a, "q_norm", None) is None or getattr(a, "k_norm", None) is None:
                raise NotImplementedError("a layer without q_norm and k_norm is not bound")
            if any(getattr(p, "bias", None) is not None for p in (a.q_proj, a.k_proj, a.v_proj, a.o_proj, m.mlp.gate_proj,
                                                                  m.mlp.up_proj, m.mlp.down_proj)):
                raise NotImplementedError("Qwen3 projections have no bias; a biased layer is not bound")
        norms = ("input_layernorm", "post_attention_layernorm", "pre_feedforward_layernorm", "post_feedforward_layernorm")
        for i, m in enumerate(layers):
            for at, name in [(m, n) for n in norms] + [(m.self_attn, "q_norm"), (m.self_attn, "k_norm")]:
                _refuse_other_norm(getattr(at, name, None), f"layer {i}'s {name}")
            _refuse_other_mlp(m, i)
            _refuse_other_attention(m, i)
        _refuse_other_norm(norm, "the final norm")
        self.head_dim = a0.q_norm.weight.shape[0]
        self.q_heads = a0.q_proj.weight.shape[0] // self.head_dim
        self.kv_heads = a0.k_proj.weight.shape[0] // self.head_dim
        self.hidden = embed.shape[1]
        self.window, self.sinks = int(window), int(sinks)
        # without a window= here a layer's own is kept to by refusing sequences that are longer than it
        own = [getattr(m.self_attn, "sliding_window", None) for m in layers]
        self.reach = min((int(w) for w in own if w is not None and not self.window), default=None)
        self._refuse_other_shapes(layers, norm, embed, lm_head)
        ln = layers[0].input_layernorm
        self.eps = float(getattr(ln, "variance_epsilon", getattr(ln, "eps", 1e-6)))

        # norms behind the blocks as well: then the one behind the attention has the name that else is the MLP's before it
        after = [getattr(m, "post_feedforward_layernorm", None) is not None for m in layers]
        if any((getattr(m, "pre_feedforward_layernorm", None) is not None) != b for m, b in zip(layers, after)) or len(set(after)) > 1:
            raise NotImplementedError("every layer has pre_feedforward_layernorm and post_feedforward_layernorm, or none has")
        self.after, self.residual_scale = after[0], float(residual_scale)
        # the sum and the norms around it in one pass; layers without either keep their roundings (a sum in the product)
        self.fused = self.after or self.residual_scale != 1.0

        def put(*w):
            return torch.cat([t.detach() for t in w]).to(self.device, BF).contiguous()

        def behind(m):
            if not self.after:
                return {}
            return dict(post1=put(m.post_attention_layernorm.weight), post2=put(m.post_feedforward_layernorm.weight))

        self.layers = [dict(behind(m), norm1=put(m.input_layernorm.weight),
                            norm2=put((m.pre_feedforward_layernorm if self.after else m.post_attention_layernorm).weight),
                            qkv=put(m.self_attn.q_proj.weight, m.self_attn.k_proj.weight, m.self_attn.v_proj.weight),
                            q_norm=put(m.self_attn.q_norm.weight), k_norm=put(m.self_attn.k_norm.weight),
                            o=put(m.self_attn.o_proj.weight), gate_up=put(m.mlp.gate_proj.weight, m.mlp.up_proj.weight),
                            down=put(m.mlp.down_proj.weight)) for m in layers]
        self.norm, self.embed, self.lm_head = put(norm.weight), put(embed), put(lm_head)
        self.rope = rope
        if rope is not None:
            if rope.head_dim != self.head_dim or rope.rotary_dim != self.head_dim or rope.interleaved:
                raise ValueError(f"the rope must turn halves of whole heads of {self.head_dim}")
            if rope.freqs.device != self.embed.device:
                raise ValueError(f"the rope is on {rope.freqs.device}, the decoder on {self.embed.device}")
            self.cos = self.sin = None
            return
        self.cos, self.sin = (t.detach().to(self.device).contiguous() for t in (cos, sin))
        if (cos.dim() != 2 or cos.shape[1] != self.head_dim or sin.shape != cos.shape or sin.dtype != cos.dtype or
                cos.dtype not in (torch.float32, BF)):
            raise ValueError(f"cos and sin must be [rows, {self.head_dim}], both float32 or both bfloat16")

    def _refuse_other_shapes(self, layers, norm, embed, lm_head) -> None:
        """Raises for a model that a step would refuse at one of its kernels, when the cache has changed."""
        d, hidden, q, kv = self.head_dim, self.hidden, self.q_heads * self.head_dim, self.kv_heads * self.head_dim
        if d not in (64, 128) or self.kv_heads < 1 or self.q_heads % self.kv_heads:
            raise NotImplementedError(f"heads of 64 or 128 values are run, each key / value head's with as many query heads; got {self.q_heads} "
                                      f"query and {self.kv_heads} key / value heads of {d}")
        if hidden % 8 or not 8 <= hidden <= 4096:
            raise NotImplementedError(f"hidden must be a multiple of 8, 4096 at most (the norms' rows), got {hidden}")
        if self.window < 0 or self.sinks < 0:
            raise ValueError(f"window and sinks must not be negative, got {self.window} and {self.sinks}")

        def has(t, name, *shape):
            if tuple(t.shape) != shape:
                raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")

        for i, m in enumerate(layers):
            a, ffn = m.self_attn, m.mlp.gate_proj.weight.shape[0]
            if ffn % 8 or ffn < 8:
                raise NotImplementedError(f"layer {i}'s MLP must have a multiple of 8 values, got {ffn}")
            for at, name, *shape in ((a, "q_proj", q, hidden), (a, "k_proj", kv, hidden), (a, "v_proj", kv, hidden), (a, "o_proj", hidden, q),
                                     (a, "q_norm", d), (a, "k_norm", d), (m.mlp, "gate_proj", ffn, hidden), (m.mlp, "up_proj", ffn, hidden),
                                     (m.mlp, "down_proj", hidden, ffn), (m, "input_layernorm", hidden), (m, "post_attention_layernorm", hidden),
                                     (m, "pre_feedforward_layernorm", hidden), (m, "post_feedforward_layernorm", hidden)):
                part = getattr(at, name, None)
                if part is not None:
                    has(part.weight, f"layer {i}'s {name}", *shape)
        has(norm.weight, "the final norm", hidden)
        for t, name in ((embed, "embed"), (lm_head, "lm_head")):
            has(t, name, t.shape[0], hidden)
            if t.shape[0] < 1:
                raise ValueError(f"{name} has no tokens")

    def new_cache(self, seqs: int, max_tokens: int, page_size: int = 64) -> B200KV4Cache:
        return B200KV4Cache(len(self.layers), self.kv_heads, self.head_dim, seqs, max_tokens, page_size, self.device)

    def _here(self, cache: B200KV4Cache, **tensors: Optional[torch.Tensor]) -> None:
        """Refuses tensors that are not the decoder's device's, or another current device, to whose stream the launches go."""
        at = self.embed.device
        for name, t in dict(tensors, cache=cache.table).items():
            if t is not None and t.device != at:
                raise ValueError(f"{name} is on {t.device}, the decoder on {at}")
        if at.type != "cuda" or at.index != torch.cuda.current_device():
            raise ValueError(f"the decoder is on {at}, which is not the current CUDA device (no CPU path exists)")

    def _rmsnorm(self, x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
        x = x.contiguous()  # one row stride serves input and output
        out = torch.empty_like(x)
        seg = _lib.ResLnSegment(x.data_ptr(), None, None, None, None, out.data_ptr(), x.shape[0], x.shape[1], x.shape[1],
                                weight.data_ptr())
        _lib.check(_lib.load().rldx_res_rmsnorm(C.byref(seg), 1, self.eps, C.c_void_p(torch.cuda.current_stream().cuda_stream)))
        return out

    def _refuse_longer(self, longest: int, tables: bool) -> None:
        """Raises for a sequence longer than the RoPE tables, or than a window that its layers have and the decoder was not given."""
        if tables and longest > self.cos.shape[0]:
            raise ValueError(f"a sequence of {longest} tokens is longer than the RoPE tables ({self.cos.shape[0]})")
        if self.reach is not None and longest > self.reach:
            raise ValueError(f"a sequence of {longest} tokens is longer than a layer's sliding window ({self.reach}): give the decoder its window")

    def _places(self, start: Sequence[int], new: Sequence[int], positions: Optional[torch.Tensor]) -> torch.Tensor:
        """The rows of the tables, or the rope's positions [axes, rows], that the new tokens take; refuses others."""
        rows, tables = sum(new), self.rope is None
        self._refuse_longer(max(s + n for s, n in zip(start, new)), tables and positions is None)
        if positions is None:
            positions = torch.cat([torch.arange(s, s + n, dtype=torch.int32) for s, n in zip(start, new)])
        elif tuple(positions.shape) != (rows,) and (tables or tuple(positions.shape) != (self.rope.axes, rows)):
            raise ValueError(f"positions must be [{rows}]" + ("" if tables else f" or [{self.rope.axes}, {rows}]") + f", got {tuple(positions.shape)}")
        elif tables and positions.device.type == "cpu":
            positions = _whole(positions, "positions", True)
            if not 0 <= int(positions.min()) <= int(positions.max()) < self.cos.shape[0]:
                raise ValueError(f"positions must be rows of the RoPE tables ({self.cos.shape[0]})")  # (on the device: device error 0x501)
        elif not tables and (positions.dtype.is_floating_point or positions.dtype == torch.bool):
            raise ValueError("positions must be whole numbers")
        return positions

    def _run(self, hidden: torch.Tensor, cache: B200KV4Cache, new: Sequence[int], positions: Optional[torch.Tensor] = None,
             deepstack_features: Optional[Sequence[torch.Tensor]] = None, deepstack_rows: Optional[torch.Tensor] = None):
        """The rows through the layers; returns f(rows) that gives the final norm of some of them."""
        new = [int(n) for n in new]
        if hidden.shape != (sum(new), self.hidden) or hidden.dtype != BF:
            raise ValueError(f"hidden must be bfloat16 [{sum(new)}, {self.hidden}], got {hidden.dtype} {tuple(hidden.shape)}")
        if len(new) != len(cache.tokens) or min(new) < 0 or max(new) == 0:
            raise ValueError(f"new must give a count for each of the {len(cache.tokens)} sequences, one of them positive")
        positions = self._places(list(cache.tokens), new, positions)
        if len(cache.pools) != len(self.layers) or any(p.shape[1] != self.kv_heads or p.shape[3] != 40 * self.head_dim
                                                       for p in cache.pools):
            raise ValueError(f"the cache is not one of {len(self.layers)} layers of {self.kv_heads} key / value heads of {self.head_dim}")
        features, at = list(deepstack_features or ()), None
        if features:
            if deepstack_rows is None:
                raise ValueError("deepstack_features need deepstack_rows")
            at = _whole(deepstack_rows, "deepstack_rows", True)  # (looked at on the host: rows outside would fault)
            if at.dim() != 1 or at.unique().numel() != at.numel() or (at.numel() and not 0 <= int(at.min()) <= int(at.max()) < sum(new)):
                raise ValueError(f"deepstack_rows must be different rows of the {sum(new)} of hidden")
            if len(features) > len(self.layers) or any(tuple(f.shape) != (at.numel(), self.hidden) for f in features):
                raise ValueError(f"deepstack_features must be at most {len(self.layers)} of [{at.numel()}, {self.hidden}]")
        elif deepstack_rows is not None:
            raise ValueError("deepstack_rows go with deepstack_features")
        self._here(cache, hidden=hidden)
        hidden = hidden.contiguous()  # (what a product adds, and the first norm reads, begins at 16 bytes)
        if hidden.data_ptr() % 16:
            hidden = hidden.clone()
        if features:
            at, features = at.to(self.device), [f.to(self.device, BF) for f in features]
        if self.rope is None:
            cos, sin, positions = self.cos, self.sin, positions.to(torch.int32).to(self.device)
        else:  # rows for these tokens alone
            positions = positions.to(self.device, torch.int64).contiguous()  # (an axis' positions side by side)
            if self.rope.sections is not None:
                positions = positions.expand(self.rope.axes, -1)
            elif positions.dim() == 2:
                positions = positions[0]
            cos, sin = self.rope.rows(positions)
            positions = torch.arange(sum(new), dtype=torch.int32, device=self.device)
        cache.extend(new)  # from here on nothing refuses
        cu = torch.tensor([0, *new], dtype=torch.int32).cumsum(0).to(torch.int32).to(self.device)
        max_new, max_len = max(new), max(cache.tokens)

        def attention(n, w, pool):
            qkv = ops.linear(n, w["qkv"])
            q = ops.qkv_rope_append(qkv, w["q_norm"], w["k_norm"], cos, sin, positions, pool, cache.table, cache.lengths, cu,
                                    q_heads=self.q_heads, eps=self.eps)
            return ops.kv4_attention(q, pool, cache.table, cache.lengths, cu, max_new=max_new, max_len=max_len, window=self.window,
                                     sinks=self.sinks).flatten(1)

        def mlp(n, w):
            gate, up = ops.linear(n, w["gate_up"]).chunk(2, 1)
            return ops.swiglu(gate, up)

        h = hidden
        if not self.fused:
            for i, (w, pool) in enumerate(zip(self.layers, cache.pools)):
                h = ops.linear(attention(self._rmsnorm(h, w["norm1"]), w, pool), w["o"], add=h)
                h = ops.linear(mlp(self._rmsnorm(h, w["norm2"]), w), w["down"], add=h)
                if i < len(features):
                    h[at] += features[i]
            return lambda rows: self._rmsnorm(h[rows].contiguous(), self.norm)

        def between(y, h, weight, post):
            """h + residual_scale * post(y), and the norm with `weight` of it."""
            return ops.block_norms(y, h, post="rms" if self.after else None, post_weight=post, scale=self.residual_scale,
                                   pre=None if weight is None else "rms", pre_weight=weight, eps=self.eps)

        n = self._rmsnorm(h, self.layers[0]["norm1"])
        for i, (w, pool) in enumerate(zip(self.layers, cache.pools)):
            h, n = between(ops.linear(attention(n, w, pool), w["o"]), h, w["norm2"], w.get("post1"))
            after = self.layers[i + 1]["norm1"] if i + 1 < len(self.layers) else self.norm
            joins = i < len(features)  # before the next norm
            h, n = between(ops.linear(mlp(n, w), w["down"]), h, None if joins else after, w.get("post2"))
            if joins:
                h[at] += features[i]
                n = self._rmsnorm(h, after)
        return lambda rows: n[rows]

    def forward(self, hidden: torch.Tensor, cache: B200KV4Cache, new: Sequence[int],
                positions: Optional[torch.Tensor] = None, deepstack_features: Optional[Sequence[torch.Tensor]] = None,
                deepstack_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Runs the rows `hidden` [sum(new), hidden] (the new tokens of every sequence, in order)
        through the layers; keys and values join the cache.  positions [sum(new)]: RoPE rows, the
        tokens' places in their sequences by default; with a rope any whole numbers, of one axis for all or [axes, sum(new)].
        deepstack_features[i] [n, hidden] are added after
        layer i to the rows deepstack_rows [n] of hidden (a vision tower's, as B200LLMChain takes them), with one
        rounding to bf16.  Returns logits [seqs with new tokens, vocab]
        of each sequence's last new token."""
        new = [int(n) for n in new]
        normed = self._run(hidden, cache, new, positions, deepstack_features, deepstack_rows)
        last = torch.tensor([e - 1 for n, e in zip(new, torch.tensor(new).cumsum(0).tolist()) if n], device=self.device)
        return ops.linear(normed(last).contiguous(), self.lm_head)

    def score(self, prompts, *, targets: Optional[Sequence] = None, top: int = 0, cache: Optional[B200KV4Cache] = None,
              positions: Optional[Sequence] = None, deepstack_features: Optional[Sequence[torch.Tensor]] = None,
              deepstack_rows: Optional[torch.Tensor] = None) -> list:
        """How likely the prompts' own tokens are: for each prompt (ids, or rows of embeddings) Scores whose entry i is about the
        token that follows its row i: targets[prompt][i], by default the prompt's next id, and none (-1: logprob 0, rank -1)
        behind the last one or where the prompt is rows.  Its entropy and `top` (0 to 32) alternatives are there either way.  Logits
        are made for a few thousand rows at a time.  positions, deepstack_features and deepstack_rows are generate()'s.  An error that a
        kernel has recorded on the device raises RldxError."""
        ids, rows = zip(*(self._rows(p) for p in prompts)) if len(prompts) else ((), ())
        new = [r.shape[0] for r in rows]
        if not new or min(new) == 0:
            raise ValueError("a prompt has no token")
        top = self._alternatives(top, "top")
        if targets is None:
            follow = [torch.full((n,), -1) if i is None else torch.cat([i[1:], torch.tensor([-1])]) for i, n in zip(ids, new)]
        else:
            follow = [_whole(t, "targets") for t in targets]
            if [tuple(t.shape) for t in follow] != [(n,) for n in new]:
                raise ValueError(f"targets must give {new} tokens, got {[tuple(t.shape) for t in follow]}")
        follow = torch.cat(follow)
        if int(follow.max()) >= self.lm_head.shape[0]:
            raise ValueError(f"targets must be below the {self.lm_head.shape[0]} tokens of lm_head")
        cache = cache or self.new_cache(len(prompts), sum(new))
        if cache.seqs != len(prompts):
            raise ValueError(f"the cache has {cache.seqs} sequences, {len(prompts)} prompts were given")
        cache.room(new)
        places = None if positions is None else self._prompt_places(positions, new)[0]
        normed = self._run(torch.cat(rows), cache, new, places, deepstack_features, deepstack_rows)
        follow, total, parts = follow.to(self.device), sum(new), []
        step = max(1, self.score_logits // self.lm_head.shape[0])
        for a in range(0, total, step):
            at = slice(a, min(a + step, total))
            parts.append(ops.token_logprobs(ops.linear(normed(at).contiguous(), self.lm_head), follow[at], top=top))
        self._report("tokens were scored")
        return [Scores(*part) for part in zip(*(torch.cat(t).split(list(new)) for t in zip(*parts)))]

    def _report(self, what: str) -> None:
        """Raises a device error that a kernel has recorded: what came out is not of all the data."""
        code = ops.device_error()
        if code:
            raise _lib.RldxError(_lib.RLDX_ERR_DEVICE, f"device error 0x{code:x} recorded while {what}, or left by earlier work")

    def _alternatives(self, n, name: str) -> int:
        """A number of alternatives that token_logprobs takes; refuses others, fractions with a TypeError."""
        n, most = operator.index(n), min(32, self.lm_head.shape[0])
        if not 0 <= n <= most:
            raise ValueError(f"{name} must be 0 to {most}, got {n}")
        return n

    def _rows(self, prompt):
        """A prompt's ids (None where it is rows of embeddings) and its rows; refuses ids that the embedding does not have."""
        if torch.is_tensor(prompt) and prompt.dim() == 2:
            return None, prompt.to(self.device, BF)
        ids = _whole(prompt, "a prompt's ids")
        if ids.dim() != 1:
            raise ValueError(f"a prompt is ids [n] or rows of embeddings [n, {self.hidden}], got {tuple(ids.shape)}")
        if ids.numel() and not 0 <= int(ids.min()) <= int(ids.max()) < self.embed.shape[0]:  # (looked at on the host: others would fault)
            raise ValueError(f"a prompt's ids must be among the {self.embed.shape[0]} of the embedding")
        return ids, self.embed[ids.to(self.device)]

    def _prompt_places(self, positions: Sequence, new: Sequence[int]):
        """The prompts' positions, one after the other, and one past each one's largest; refuses other shapes."""
        given = [torch.as_tensor(p) for p in positions]
        wanted = [(n,) for n in new]
        if self.rope is not None:  # one position for all axes, or each
            given = [p.expand(self.rope.axes, -1) if p.dim() == 1 else p for p in given]
            wanted = [(self.rope.axes, n) for n in new]
        if [tuple(p.shape) for p in given] != wanted:
            raise ValueError(f"positions must give {list(new)} rows, got {[tuple(p.shape) for p in given]}")
        given = [_whole(p, "positions", self.rope is None) for p in given]
        return torch.cat(given, -1), [int(p.max()) + 1 for p in given]

    def generate(self, prompts, max_new_tokens: int, *, u: torch.Tensor, cache: Optional[B200KV4Cache] = None,
                 temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, stop_ids: Sequence[int] = (),
                 positions: Optional[Sequence] = None, next_positions: Optional[Sequence[int]] = None,
                 deepstack_features: Optional[Sequence[torch.Tensor]] = None, deepstack_rows: Optional[torch.Tensor] = None,
                 logprobs: Optional[int] = None):
        """Appends max_new_tokens tokens to each of the prompts (lists of ids, or rows [n, hidden] of
        embeddings that a vision tower has filled in).  positions gives each prompt's RoPE rows [n], of
        tables whose rows stand for whatever the prompt's tokens have (vision tokens do not count up one by one);
        the new tokens go on at next_positions, by default one past a prompt's largest.  Without it the rows are
        the tokens' places in their sequences.  deepstack_features and deepstack_rows are forward()'s, of the
        prompts' rows one after the other.  u [max_new_tokens, prompts] are the draws'
        numbers in [0, 1).  Returns a list of id lists; a sequence ends after one of stop_ids.  With logprobs (0 to 32) it is
        (ids, scores): of each sequence Scores of its new tokens under the unfiltered logits, with so many alternatives.  A sequence whose logits
        have no number to draw from (all NaN or -inf) before its end raises RuntimeError, an error that a kernel
        has recorded on the device RldxError."""
        n = len(prompts)
        if tuple(u.shape) != (max_new_tokens, n):
            raise ValueError(f"u must be [{max_new_tokens}, {n}], got {tuple(u.shape)}")
        rows = [self._rows(p)[1] for p in prompts]
        cache = cache or self.new_cache(n, sum(r.shape[0] for r in rows) + n * max_new_tokens)
        if cache.seqs != n:
            raise ValueError(f"the cache has {cache.seqs} sequences, {n} prompts were given")
        if min(r.shape[0] for r in rows) == 0:
            raise ValueError("a prompt has no token")
        if max_new_tokens > 0:  # what would end the run in its middle: all but the last token drawn are run
            ends = [t + r.shape[0] + max_new_tokens - 1 for t, r in zip(cache.tokens, rows)]
            self._refuse_longer(max(ends), positions is None and self.rope is None)
            cache.room([e - t for e, t in zip(ends, cache.tokens)])
        places = follow = None
        if positions is not None:
            places, past = self._prompt_places(positions, [r.shape[0] for r in rows])
            follow = torch.tensor(past) if next_positions is None else \
                _whole(next_positions if torch.is_tensor(next_positions) else list(next_positions), "next_positions", True)
            if follow.shape != (n,):
                raise ValueError(f"next_positions must be {n} rows")
            if self.rope is None and not (0 <= int(places.min()) and int(places.max()) < self.cos.shape[0] and
                    (max_new_tokens <= 1 or (int(follow.min()) >= 0 and int(follow.max()) + max_new_tokens - 2 < self.cos.shape[0]))):
                raise ValueError(f"the positions of the prompts and the new tokens must be rows of the RoPE tables ({self.cos.shape[0]})")
        elif next_positions is not None:
            raise ValueError("next_positions go with positions")
        u = u.to(self.device, torch.float32).contiguous()

        def full(v, dtype):
            return torch.full((n,), v, dtype=dtype, device=self.device)

        limits = dict(temperature=full(temperature, torch.float32), top_k=full(top_k, torch.int32),
                      top_p=full(top_p, torch.float32), min_p=full(min_p, torch.float32))
        deep = {} if deepstack_features is None else dict(deepstack_features=deepstack_features, deepstack_rows=deepstack_rows)
        if not deep and deepstack_rows is not None:
            raise ValueError("deepstack_rows go with deepstack_features")
        if logprobs is not None:
            logprobs = self._alternatives(logprobs, "logprobs")
        hidden, new, tokens, scores = torch.cat(rows), [r.shape[0] for r in rows], [], []
        for i in range(max_new_tokens):
            logits = self.forward(hidden, cache, new, places, **deep)
            token, _, _ = ops.sample(logits, u[i], **limits)
            tokens.append(token)
            if logprobs is not None:
                scores.append(ops.token_logprobs(logits, token, top=logprobs))
            deep = {}
            hidden, new, places = self.embed[token], [1] * n, None if follow is None else follow + i
        out = torch.stack(tokens, 1).tolist() if tokens else [[] for _ in prompts]
        self._report("tokens were generated")
        for s, ids in enumerate(out):
            end = next((k for k, t in enumerate(ids) if t in stop_ids), None)
            if end is not None:
                del ids[end + 1:]
            if -1 in ids:  # (what was run after it began with the last row of the embedding)
                raise RuntimeError(f"sequence {s} has no logit that is a number at its token {ids.index(-1)}")
        if logprobs is None:
            return out
        if not scores:
            empty = Scores(*ops.token_logprobs(self.embed.new_empty(0, self.lm_head.shape[0]), torch.empty(0, dtype=torch.int64, device=self.device), top=logprobs))
            return out, [empty for _ in prompts]
        steps = [torch.stack(t, 1) for t in zip(*scores)]  # [sequences, tokens, ...]
        return out, [Scores(*(t[s, : len(ids)] for t in steps)) for s, ids in enumerate(out)]


def main() -> None:
    from types import SimpleNamespace as NS

    ap = argparse.ArgumentParser(description="Decodes tokens with random weights of a Qwen3-shaped decoder.")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--prompt", type=int, default=1104)
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--rope", action="store_true", help="angles from positions in place of tables")
    ap.add_argument("--score", action="store_true", help="log probabilities of the prompts' own tokens as well")
    a = ap.parse_args()
    g = torch.Generator(device="cuda").manual_seed(0)

    def w(*shape):
        return NS(weight=torch.randn(*shape, device="cuda", generator=g) * 0.02)

    d, hq, hkv, ffn = 128, 16, 2, 11008
    one = NS(weight=torch.ones(a.hidden, device="cuda"))
    head = NS(weight=torch.ones(d, device="cuda"))
    layers = [NS(input_layernorm=one, post_attention_layernorm=one,
                 self_attn=NS(q_proj=w(hq * d, a.hidden), k_proj=w(hkv * d, a.hidden), v_proj=w(hkv * d, a.hidden),
                              o_proj=w(a.hidden, hq * d), q_norm=head, k_norm=head),
                 mlp=NS(gate_proj=w(ffn, a.hidden), up_proj=w(ffn, a.hidden), down_proj=w(a.hidden, ffn)))
              for _ in range(a.layers)]
    if a.rope:
        angles = dict(rope=B200Rope(d, theta=1e6))
    else:
        inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device="cuda").float() / d))
        ang = torch.outer(torch.arange(a.prompt + a.tokens, device="cuda").float(), inv).repeat(1, 2)
        angles = dict(cos=ang.cos(), sin=ang.sin())
    dec = B200TextDecoder(layers, one, w(a.vocab, a.hidden).weight * 50, w(a.vocab, a.hidden).weight, **angles,
                          window=a.window, sinks=a.sinks)
    prompts = [torch.randint(a.vocab, (a.prompt - 7 * s,), device="cuda", generator=g).tolist() for s in range(a.seqs)]
    u = torch.rand(a.tokens, a.seqs, generator=torch.Generator().manual_seed(0))
    dec.generate(prompts, 2, u=u[:2], temperature=0.8, top_p=0.95)  # loads the kernels
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    out = dec.generate(prompts, a.tokens, u=u, temperature=0.8, top_k=50, top_p=0.95)
    e1.record()
    torch.cuda.synchronize()
    print(f"{a.seqs} sequences, prompts of {a.prompt}: {a.tokens} tokens each in {e0.elapsed_time(e1):.1f} ms; first ids "
          f"{[ids[:6] for ids in out]}")
    if a.score:
        dec.score(prompts, top=5)
        e0.record()
        scores = dec.score(prompts, top=5)
        e1.record()
        torch.cuda.synchronize()
        print(f"scored in {e0.elapsed_time(e1):.1f} ms; mean log probability {[round(float(x.logprob.mean()), 3) for x in scores]}")


if __name__ == "__main__":
    main()
