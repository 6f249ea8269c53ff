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

`decoder_layers` are Qwen3 text decoder layers (the attribute names that B200LLMChain takes), `cos` and
`sin` their RoPE tables [positions, head_dim].  Prompts of a vision tower bring positions and deepstack
features of their own; everything that cannot be run is refused before the cache changes.  `python -m rldx_b200.decoder` decodes with random
weights.
"""

from __future__ import annotations

import argparse
import ctypes as C
from typing import Optional, Sequence

import torch

from . import _lib, ops
from .llm import _raw_layer

BF = torch.bfloat16


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


class B200TextDecoder:
    """Qwen3 decoder layers, embedding and output projection over a B200KV4Cache.

    Layers in a LayerWrapper that compresses video tokens (B200LLMChain's compress_info) would have to drop tokens from
    the cache of the layers after it, which no page table here can say: they are refused unless
    ignore_compression says that no prompt has what the wrapper compresses (it leaves one frame, and text, as
    they are)."""

    def __init__(self, layers, norm, embed: torch.Tensor, lm_head: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                 window: int = 0, sinks: int = 0, device=None, ignore_compression: bool = False):
        layers = list(layers)
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
        self.head_dim = a0.q_norm.weight.shape[0]
        self.q_heads = a0.q_proj.weight.shape[0] // self.head_dim
        self.kv_heads = a0.k_proj.weight.shape[0] // self.head_dim
        self.hidden = embed.shape[1]
        self.window, self.sinks = int(window), int(sinks)
        ln = layers[0].input_layernorm
        self.eps = float(getattr(ln, "variance_epsilon", getattr(ln, "eps", 1e-6)))

        def put(*w):
            return torch.cat([t.detach() for t in w]).to(self.device, BF).contiguous()

        self.layers = [dict(norm1=put(m.input_layernorm.weight), norm2=put(m.post_attention_layernorm.weight),
                            qkv=put(m.self_attn.q_proj.weight, m.self_attn.k_proj.weight, m.self_attn.v_proj.weight),
                            q_norm=put(m.self_attn.q_norm.weight), k_norm=put(m.self_attn.k_norm.weight),
                            o=put(m.self_attn.o_proj.weight), gate_up=put(m.mlp.gate_proj.weight, m.mlp.up_proj.weight),
                            down=put(m.mlp.down_proj.weight)) for m in layers]
        self.norm, self.embed, self.lm_head = put(norm.weight), put(embed), put(lm_head)
        self.cos, self.sin = (t.detach().to(self.device).contiguous() for t in (cos, sin))
        if (cos.dim() != 2 or cos.shape[1] != self.head_dim or sin.shape != cos.shape or sin.dtype != cos.dtype or
                cos.dtype not in (torch.float32, BF)):
            raise ValueError(f"cos and sin must be [rows, {self.head_dim}], both float32 or both bfloat16")

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

    def forward(self, hidden: torch.Tensor, cache: B200KV4Cache, new: Sequence[int],
                positions: Optional[torch.Tensor] = None, deepstack_features: Optional[Sequence[torch.Tensor]] = None,
                deepstack_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Runs the rows `hidden` [sum(new), hidden] (the new tokens of every sequence, in order)
        through the layers; keys and values join the cache.  positions [sum(new)]: RoPE rows, the
        tokens' places in their sequences by default.  deepstack_features[i] [n, hidden] are added after
        layer i to the rows deepstack_rows [n] of hidden (a vision tower's, as B200LLMChain takes them), with one
        rounding to bf16.  Returns logits [seqs with new tokens, vocab]
        of each sequence's last new token."""
        new = [int(n) for n in new]
        if hidden.shape != (sum(new), self.hidden) or hidden.dtype != BF:
            raise ValueError(f"hidden must be bfloat16 [{sum(new)}, {self.hidden}], got {hidden.dtype} {tuple(hidden.shape)}")
        if len(new) != len(cache.tokens) or min(new) < 0 or max(new) == 0:
            raise ValueError(f"new must give a count for each of the {len(cache.tokens)} sequences, one of them positive")
        start = list(cache.tokens)
        if positions is None:
            longest = max(s + n for s, n in zip(start, new))
            if longest > self.cos.shape[0]:
                raise ValueError(f"a sequence of {longest} tokens is longer than the RoPE tables ({self.cos.shape[0]})")
            positions = torch.cat([torch.arange(s, s + n, dtype=torch.int32) for s, n in zip(start, new)])
        elif tuple(positions.shape) != (sum(new),):
            raise ValueError(f"positions must be [{sum(new)}], got {tuple(positions.shape)}")
        elif positions.device.type == "cpu" and not 0 <= int(positions.min()) <= int(positions.max()) < self.cos.shape[0]:
            raise ValueError(f"positions must be rows of the RoPE tables ({self.cos.shape[0]})")  # (else device error 0x501)
        if len(cache.pools) != len(self.layers) or any(p.shape[1] != self.kv_heads or p.shape[3] != 40 * self.head_dim
                                                       for p in cache.pools):
            raise ValueError(f"the cache is not one of {len(self.layers)} layers of {self.kv_heads} key / value heads of {self.head_dim}")
        features, at = list(deepstack_features or ()), None
        if features:
            if deepstack_rows is None:
                raise ValueError("deepstack_features need deepstack_rows")
            at = torch.as_tensor(deepstack_rows).to("cpu", torch.int64)  # (looked at on the host: rows outside would fault)
            if at.dim() != 1 or at.unique().numel() != at.numel() or (at.numel() and not 0 <= int(at.min()) <= int(at.max()) < sum(new)):
                raise ValueError(f"deepstack_rows must be different rows of the {sum(new)} of hidden")
            if len(features) > len(self.layers) or any(tuple(f.shape) != (at.numel(), self.hidden) for f in features):
                raise ValueError(f"deepstack_features must be at most {len(self.layers)} of [{at.numel()}, {self.hidden}]")
        elif deepstack_rows is not None:
            raise ValueError("deepstack_rows go with deepstack_features")
        self._here(cache, hidden=hidden)
        if features:
            at, features = at.to(self.device), [f.to(self.device, BF) for f in features]
        positions = positions.to(self.device, torch.int32)
        cache.extend(new)  # from here on nothing refuses
        cu = torch.tensor([0, *new], dtype=torch.int32).cumsum(0).to(torch.int32).to(self.device)
        max_new, max_len = max(new), max(cache.tokens)
        h = hidden
        for i, (w, pool) in enumerate(zip(self.layers, cache.pools)):
            qkv = ops.linear(self._rmsnorm(h, w["norm1"]), w["qkv"])
            q = ops.qkv_rope_append(qkv, w["q_norm"], w["k_norm"], self.cos, self.sin, positions, pool, cache.table,
                                    cache.lengths, cu, q_heads=self.q_heads, eps=self.eps)
            a = ops.kv4_attention(q, pool, cache.table, cache.lengths, cu, max_new=max_new, max_len=max_len,
                                  window=self.window, sinks=self.sinks)
            h = ops.linear(a.flatten(1), w["o"], add=h)
            gate, up = ops.linear(self._rmsnorm(h, w["norm2"]), w["gate_up"]).chunk(2, 1)
            h = ops.linear(ops.swiglu(gate, up), w["down"], add=h)
            if i < len(features):
                h[at] += features[i]
        last = torch.tensor([e - 1 for n, e in zip(new, torch.tensor(new).cumsum(0).tolist()) if n], device=self.device)
        return ops.linear(self._rmsnorm(h[last].contiguous(), self.norm), self.lm_head)

    def generate(self, prompts, max_new_tokens: int, *, u: torch.Tensor, cache: Optional[B200KV4Cache] = None,
                 temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0, stop_ids: Sequence[int] = (),
                 positions: Optional[Sequence] = None, next_positions: Optional[Sequence[int]] = None,
                 deepstack_features: Optional[Sequence[torch.Tensor]] = None, deepstack_rows: Optional[torch.Tensor] = None):
        """Appends max_new_tokens tokens to each of the prompts (lists of ids, or rows [n, hidden] of
        embeddings that a vision tower has filled in).  positions gives each prompt's RoPE rows [n], of
        tables whose rows stand for whatever the prompt's tokens have (vision tokens do not count up one by one);
        the new tokens go on at next_positions, by default one past a prompt's largest.  Without it the rows are
        the tokens' places in their sequences.  deepstack_features and deepstack_rows are forward()'s, of the
        prompts' rows one after the other.  u [max_new_tokens, prompts] are the draws'
        numbers in [0, 1).  Returns a list of id lists; a sequence ends after one of stop_ids.  A sequence whose logits
        have no number to draw from (all NaN or -inf) before its end raises RuntimeError, an error that a kernel
        has recorded on the device RldxError."""
        n = len(prompts)
        if tuple(u.shape) != (max_new_tokens, n):
            raise ValueError(f"u must be [{max_new_tokens}, {n}], got {tuple(u.shape)}")
        rows = [self.embed[torch.as_tensor(p, device=self.device)] if not torch.is_tensor(p) or p.dim() == 1 else
                p.to(self.device, BF) for p in prompts]
        cache = cache or self.new_cache(n, sum(r.shape[0] for r in rows) + n * max_new_tokens)
        if cache.seqs != n:
            raise ValueError(f"the cache has {cache.seqs} sequences, {n} prompts were given")
        if min(r.shape[0] for r in rows) == 0:
            raise ValueError("a prompt has no token")
        if max_new_tokens > 0:  # what would end the run in its middle: all but the last token drawn are run
            ends = [t + r.shape[0] + max_new_tokens - 1 for t, r in zip(cache.tokens, rows)]
            if positions is None and max(ends) > self.cos.shape[0]:
                raise ValueError(f"a sequence of {max(ends)} tokens is longer than the RoPE tables ({self.cos.shape[0]})")
            cache.room([e - t for e, t in zip(ends, cache.tokens)])
        places = follow = None
        if positions is not None:
            given = [torch.as_tensor(p).to("cpu", torch.int32) for p in positions]
            if [tuple(p.shape) for p in given] != [(r.shape[0],) for r in rows]:
                raise ValueError(f"positions must give {[r.shape[0] for r in rows]} rows, got {[tuple(p.shape) for p in given]}")
            places = torch.cat(given)
            follow = torch.tensor([int(p.max()) + 1 for p in given] if next_positions is None else [int(p) for p in next_positions],
                                  dtype=torch.int32)
            if follow.shape != (n,):
                raise ValueError(f"next_positions must be {n} rows")
            if not (0 <= int(places.min()) and int(places.max()) < self.cos.shape[0] and
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
        hidden, new, tokens = torch.cat(rows), [r.shape[0] for r in rows], []
        for i in range(max_new_tokens):
            token, _, _ = ops.sample(self.forward(hidden, cache, new, places, **deep), u[i], **limits)
            tokens.append(token)
            deep = {}
            hidden, new, places = self.embed[token], [1] * n, None if follow is None else follow + i
        out = torch.stack(tokens, 1).tolist() if tokens else [[] for _ in prompts]
        code = ops.device_error()
        if code:
            raise _lib.RldxError(_lib.RLDX_ERR_DEVICE, f"device error 0x{code:x} recorded while tokens were generated, or left by earlier work")
        for s, ids in enumerate(out):
            end = next((k for k, t in enumerate(ids) if t in stop_ids), None)
            if end is not None:
                del ids[end + 1:]
            if -1 in ids:  # (what was run after it began with the last row of the embedding)
                raise RuntimeError(f"sequence {s} has no logit that is a number at its token {ids.index(-1)}")
        return out


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
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device="cuda").float() / d))
    ang = torch.outer(torch.arange(a.prompt + a.tokens, device="cuda").float(), inv).repeat(1, 2)
    dec = B200TextDecoder(layers, one, w(a.vocab, a.hidden).weight * 50, w(a.vocab, a.hidden).weight, ang.cos(), ang.sin(),
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


if __name__ == "__main__":
    main()
