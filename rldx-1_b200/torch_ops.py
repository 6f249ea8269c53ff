"""torch.ops.b200msat: the reference's op-level surface on librldx_b200.

The reference registers torch.library custom ops for the Triton / SDPA pieces of its compiled
action-head chains (rldx/inference/action_model/double_stream/engine/ops/*.py as ds::*,
rldx/inference/action_model/single_stream/engine/ops/*.py as ss::*).  Importing this module
registers B200 counterparts under the namespace b200msat with the same argument lists, return
shapes and fake (meta) implementations, so a chain that calls torch.ops.ds.X can call
torch.ops.b200msat.ds_X instead (or rebind the name):

    ds::fused_attention_2way / _3way   -> b200msat::ds_fused_attention_2way / _3way
    ss::fused_attention_2way / _3way   -> b200msat::ss_fused_attention_2way / _3way
    ds::grouped_res_ln                 -> b200msat::ds_grouped_res_ln
    ds::grouped_swiglu                 -> b200msat::ds_grouped_swiglu
    ds::vl_epilogue_ln                 -> b200msat::ds_vl_epilogue_ln
    ss::fused_epilogue_ln              -> b200msat::ss_fused_epilogue_ln
    ss::fused_mlp_swiglu               -> b200msat::ss_fused_mlp_swiglu

plus the kernels themselves (b200msat::linear, ::joint_attention, ::layernorm,
::qk_rmsnorm_rope, ::swiglu) and the token-decoding operators (::qkv_rope_append, ::kv4_read,
::kv4_attention, ::sample), which the reference has no counterpart of.  Unlike the reference ops (which hard-code 24 heads x 64 and
batch 1), the head count comes from the shapes.  Every op runs the sm_100a kernels of
librldx_b200.so on the current stream; there is no CPU implementation.

Numerics: the fused-attention ops follow the reference's eager path (per-head RMSNorm with the
weight applied before the bf16 cast, norms.py:18-22; fp32 pair rotation, ops.py:48-67), the
epilogue ops the rounding order of the reference's kernels (sequential bf16 adds for
vl_epilogue_ln / fused_epilogue_ln, one fp32 sum for grouped_res_ln, fp32 bias + SwiGLU for
grouped_swiglu).  ss_fused_mlp_swiglu rounds the un-biased projection to bf16 before the fp32
bias + SwiGLU, where the reference's single Triton kernel keeps it in fp32.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from . import ops

BF = torch.bfloat16


def _attention(segments, H: int, L: int, device) -> Tensor:
    Lp = (L + 7) // 8 * 8
    q = torch.empty(1, H, L, 64, dtype=BF, device=device)
    k = torch.empty(1, H, L, 64, dtype=BF, device=device)
    vt = torch.empty(1, H, 64, Lp, dtype=BF, device=device)
    ops.qkv_prep(segments, q, k, vt)
    out = torch.empty(1, L, H * 64, dtype=BF, device=device)
    ops.joint_attention(q, k, vt, [L], outs=[out.view(L, H * 64)])
    return out


def _heads(qkv: Tensor) -> int:
    if qkv.shape[-1] % 192:
        raise ValueError("qkv rows must be 3 * heads * 64 wide")
    return qkv.shape[-1] // 192


# ---------------------------------------------------------------------------------------------
# fused QK-RMSNorm + RoPE + joint attention
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("b200msat::ds_fused_attention_2way", mutates_args=())
def ds_fused_attention_2way(sa_qkv: Tensor, vl_qkv: Tensor, q_norm_sa_weight: Tensor,
                            k_norm_sa_weight: Tensor, q_norm_vl_weight: Tensor,
                            k_norm_vl_weight: Tensor, rope_cos: Tensor, rope_sin: Tensor, n_sa: int,
                            n_vl: int) -> Tensor:
    """ds::fused_attention_2way (double_stream/engine/ops/op_fused_attention.py:12-92): [VL | SA],
    RoPE on the SA rows only (tables (n_sa, 32) fp32)."""
    segs = [{"qkv": vl_qkv[:n_vl], "q_norm": q_norm_vl_weight, "k_norm": k_norm_vl_weight},
            {"qkv": sa_qkv[:n_sa], "q_norm": q_norm_sa_weight, "k_norm": k_norm_sa_weight,
             "rope_cos": rope_cos, "rope_sin": rope_sin}]
    return _attention(segs, _heads(sa_qkv), n_vl + n_sa, sa_qkv.device)


@ds_fused_attention_2way.register_fake
def _(sa_qkv, vl_qkv, q_norm_sa_weight, k_norm_sa_weight, q_norm_vl_weight, k_norm_vl_weight,
      rope_cos, rope_sin, n_sa, n_vl):
    return sa_qkv.new_empty((1, n_sa + n_vl, sa_qkv.shape[-1] // 3))


@torch.library.custom_op("b200msat::ds_fused_attention_3way", mutates_args=())
def ds_fused_attention_3way(sa_qkv: Tensor, vl_qkv: Tensor, p_qkv: Tensor, q_norm_sa_weight: Tensor,
                            k_norm_sa_weight: Tensor, q_norm_vl_weight: Tensor,
                            k_norm_vl_weight: Tensor, q_norm_p_weight: Tensor,
                            k_norm_p_weight: Tensor, sa_rope_cos: Tensor, sa_rope_sin: Tensor,
                            p_rope_cos: Tensor, p_rope_sin: Tensor, n_sa: int, n_vl: int,
                            n_p: int) -> Tensor:
    """ds::fused_attention_3way (double_stream/engine/ops/op_fused_attention_3way.py:13-116):
    [VL | SA | P], RoPE on SA and P rows with their own tables."""
    segs = [{"qkv": vl_qkv[:n_vl], "q_norm": q_norm_vl_weight, "k_norm": k_norm_vl_weight},
            {"qkv": sa_qkv[:n_sa], "q_norm": q_norm_sa_weight, "k_norm": k_norm_sa_weight,
             "rope_cos": sa_rope_cos, "rope_sin": sa_rope_sin},
            {"qkv": p_qkv[:n_p], "q_norm": q_norm_p_weight, "k_norm": k_norm_p_weight,
             "rope_cos": p_rope_cos, "rope_sin": p_rope_sin}]
    return _attention(segs, _heads(sa_qkv), n_vl + n_sa + n_p, sa_qkv.device)


@ds_fused_attention_3way.register_fake
def _(sa_qkv, vl_qkv, p_qkv, q_norm_sa_weight, k_norm_sa_weight, q_norm_vl_weight,
      k_norm_vl_weight, q_norm_p_weight, k_norm_p_weight, sa_rope_cos, sa_rope_sin, p_rope_cos,
      p_rope_sin, n_sa, n_vl, n_p):
    return sa_qkv.new_empty((1, n_sa + n_vl + n_p, sa_qkv.shape[-1] // 3))


@torch.library.custom_op("b200msat::ss_fused_attention_2way", mutates_args=())
def ss_fused_attention_2way(qkv: Tensor, q_norm_weight: Tensor, k_norm_weight: Tensor,
                            rope_cos: Tensor, rope_sin: Tensor, n_sa: int) -> Tensor:
    """ss::fused_attention_2way (single_stream/engine/ops/op_fused_attention.py:12-80): one
    [VL_proj | time | S/A] stream, RoPE on its last n_sa rows."""
    M = qkv.shape[0]
    segs = [{"qkv": qkv, "q_norm": q_norm_weight, "k_norm": k_norm_weight, "rope_cos": rope_cos,
             "rope_sin": rope_sin, "rope_from": M - n_sa}]
    return _attention(segs, _heads(qkv), M, qkv.device)


@ss_fused_attention_2way.register_fake
def _(qkv, q_norm_weight, k_norm_weight, rope_cos, rope_sin, n_sa):
    return qkv.new_empty((1, qkv.shape[0], qkv.shape[-1] // 3))


@torch.library.custom_op("b200msat::ss_fused_attention_3way", mutates_args=())
def ss_fused_attention_3way(x_qkv: Tensor, p_qkv: Tensor, x_q_norm_weight: Tensor,
                            x_k_norm_weight: Tensor, p_q_norm_weight: Tensor,
                            p_k_norm_weight: Tensor, sa_rope_cos: Tensor, sa_rope_sin: Tensor,
                            p_rope_cos: Tensor, p_rope_sin: Tensor, n_x: int, n_sa: int,
                            n_p: int) -> Tensor:
    """ss::fused_attention_3way (single_stream/engine/ops/op_fused_attention_3way.py:13-110):
    [VL_proj + SA | P], RoPE on the last n_sa rows of x and on the P rows."""
    segs = [{"qkv": x_qkv[:n_x], "q_norm": x_q_norm_weight, "k_norm": x_k_norm_weight,
             "rope_cos": sa_rope_cos, "rope_sin": sa_rope_sin, "rope_from": n_x - n_sa},
            {"qkv": p_qkv[:n_p], "q_norm": p_q_norm_weight, "k_norm": p_k_norm_weight,
             "rope_cos": p_rope_cos, "rope_sin": p_rope_sin}]
    return _attention(segs, _heads(x_qkv), n_x + n_p, x_qkv.device)


@ss_fused_attention_3way.register_fake
def _(x_qkv, p_qkv, x_q_norm_weight, x_k_norm_weight, p_q_norm_weight, p_k_norm_weight,
      sa_rope_cos, sa_rope_sin, p_rope_cos, p_rope_sin, n_x, n_sa, n_p):
    return x_qkv.new_empty((1, n_x + n_p, x_qkv.shape[-1] // 3))


# ---------------------------------------------------------------------------------------------
# epilogue ops
# ---------------------------------------------------------------------------------------------
def _rows(t: Tensor, m: int, dim: int) -> Tensor:
    return t.reshape(-1, dim)[:m]


@torch.library.custom_op("b200msat::ds_grouped_res_ln", mutates_args=())
def ds_grouped_res_ln(sa_res: Tensor, sa_bias: Tensor, sa_proj: Tensor, vl_res: Tensor,
                      vl_bias: Tensor, vl_proj: Tensor, m_sa: int, m_vl: int, sa_dim: int,
                      vl_dim: int) -> Tuple[Tensor, Tensor]:
    """ds::grouped_res_ln (double_stream/engine/ops/op_grouped_res_ln.py:12-45):
    LN(res + proj + bias) per stream, summed in fp32."""
    sa_out = torch.empty(1, m_sa, sa_dim, dtype=BF, device=sa_res.device)
    vl_out = torch.empty(1, m_vl, vl_dim, dtype=BF, device=vl_res.device)
    ops.res_layernorm([
        {"x": _rows(sa_res, m_sa, sa_dim), "y": _rows(sa_proj, m_sa, sa_dim), "v1": sa_bias,
         "ln_out": sa_out.view(m_sa, sa_dim)},
        {"x": _rows(vl_res, m_vl, vl_dim), "y": _rows(vl_proj, m_vl, vl_dim), "v1": vl_bias,
         "ln_out": vl_out.view(m_vl, vl_dim)}], fp32_sum=True)
    return sa_out, vl_out


@ds_grouped_res_ln.register_fake
def _(sa_res, sa_bias, sa_proj, vl_res, vl_bias, vl_proj, m_sa, m_vl, sa_dim, vl_dim):
    return sa_res.new_empty((1, m_sa, sa_dim)), vl_res.new_empty((1, m_vl, vl_dim))


@torch.library.custom_op("b200msat::ds_grouped_swiglu", mutates_args=())
def ds_grouped_swiglu(sa_w12: Tensor, sa_bias: Tensor, vl_w12: Tensor, vl_bias: Tensor, m_sa: int,
                      m_vl: int, n_half_sa: int, n_half_vl: int) -> Tuple[Tensor, Tensor]:
    """ds::grouped_swiglu (double_stream/engine/ops/op_grouped_swiglu.py:12-41):
    silu(x[:, :h] + b[:h]) * (x[:, h:] + b[h:]) in fp32 per stream."""
    sa_out = torch.empty(m_sa, n_half_sa, dtype=BF, device=sa_w12.device)
    vl_out = torch.empty(m_vl, n_half_vl, dtype=BF, device=vl_w12.device)
    sa, vl = _rows(sa_w12, m_sa, 2 * n_half_sa), _rows(vl_w12, m_vl, 2 * n_half_vl)
    ops.swiglu_bias([
        {"gate": sa[:, :n_half_sa], "up": sa[:, n_half_sa:], "bias_gate": sa_bias[:n_half_sa],
         "bias_up": sa_bias[n_half_sa:], "out": sa_out},
        {"gate": vl[:, :n_half_vl], "up": vl[:, n_half_vl:], "bias_gate": vl_bias[:n_half_vl],
         "bias_up": vl_bias[n_half_vl:], "out": vl_out}])
    return sa_out, vl_out


@ds_grouped_swiglu.register_fake
def _(sa_w12, sa_bias, vl_w12, vl_bias, m_sa, m_vl, n_half_sa, n_half_vl):
    return sa_w12.new_empty((m_sa, n_half_sa)), vl_w12.new_empty((m_vl, n_half_vl))


@torch.library.custom_op("b200msat::ds_vl_epilogue_ln", mutates_args=())
def ds_vl_epilogue_ln(vl_res: Tensor, proj_bias: Tensor, w3_bias: Tensor, w3_out: Tensor, m: int,
                      dim: int) -> Tuple[Tensor, Tensor]:
    """ds::vl_epilogue_ln (double_stream/engine/ops/op_vl_epilogue_ln.py:13-38):
    new = res + proj_bias + w3_bias + w3_out (bf16 after each add), ln = LN(new)."""
    new = torch.empty(1, m, dim, dtype=BF, device=vl_res.device)
    ln = torch.empty(1, m, dim, dtype=BF, device=vl_res.device)
    ops.res_layernorm([{"x": _rows(vl_res, m, dim), "v1": proj_bias, "v2": w3_bias,
                        "y": _rows(w3_out, m, dim), "sum_out": new.view(m, dim), "ln_out": ln.view(m, dim)}])
    return new, ln


@ds_vl_epilogue_ln.register_fake
def _(vl_res, proj_bias, w3_bias, w3_out, m, dim):
    return vl_res.new_empty((1, m, dim)), vl_res.new_empty((1, m, dim))


@torch.library.custom_op("b200msat::ss_fused_epilogue_ln", mutates_args=())
def ss_fused_epilogue_ln(hidden: Tensor, residual: Tensor) -> Tuple[Tensor, Tensor]:
    """ss::fused_epilogue_ln (single_stream/engine/ops/op_fused_epilogue_ln.py:11-30):
    new = hidden + residual (bf16), ln = LN(new)."""
    dim = hidden.shape[-1]
    h2, r2 = hidden.reshape(-1, dim), residual.reshape(-1, dim)
    new, ln = torch.empty_like(hidden), torch.empty_like(hidden)
    ops.res_layernorm([{"x": h2, "y": r2, "sum_out": new.view(-1, dim), "ln_out": ln.view(-1, dim)}])
    return new, ln


@ss_fused_epilogue_ln.register_fake
def _(hidden, residual):
    return torch.empty_like(hidden), torch.empty_like(hidden)


@torch.library.custom_op("b200msat::ss_fused_mlp_swiglu", mutates_args=())
def ss_fused_mlp_swiglu(x: Tensor, weight: Tensor, bias: Tensor, split_k: int = 1) -> Tensor:
    """ss::fused_mlp_swiglu (single_stream/engine/ops/op_fused_mlp_swiglu.py:13-37):
    silu(x W_gate^T + b_gate) * (x W_up^T + b_up), W = [W_gate; W_up].  The tcgen05 GEMM (which
    splits K on its own) writes the un-biased projection; bias + SwiGLU follow in fp32.
    split_k is accepted for signature compatibility."""
    del split_k
    n_half = weight.shape[0] // 2
    h = ops.linear(x, weight)
    out = torch.empty(x.shape[0], n_half, dtype=BF, device=x.device)
    ops.swiglu_bias([{"gate": h[:, :n_half], "up": h[:, n_half:], "bias_gate": bias[:n_half],
                      "bias_up": bias[n_half:], "out": out}])
    return out


@ss_fused_mlp_swiglu.register_fake
def _(x, weight, bias, split_k=1):
    return x.new_empty((x.shape[0], weight.shape[0] // 2))


# ---------------------------------------------------------------------------------------------
# the kernels themselves
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("b200msat::linear", mutates_args=())
def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: int = 0,
           add: Optional[Tensor] = None) -> Tensor:
    """bf16(act(x @ weight^T + bias)) (+ add): nn.Linear through the tcgen05 GEMM."""
    return ops.linear(x, weight, bias, act=act, add=add)


@linear.register_fake
def _(x, weight, bias=None, act=0, add=None):
    return x.new_empty((x.shape[0], weight.shape[0]))


@torch.library.custom_op("b200msat::joint_attention", mutates_args=())
def joint_attention(q: Tensor, k: Tensor, vt: Tensor, seg_lens: List[int],
                    key_mask: Optional[Tensor] = None) -> List[Tensor]:
    """Non-causal joint attention over concatenated segments (q, k [B, H, L, d], vt [B, H, d, Lp])."""
    return ops.joint_attention(q, k, vt, seg_lens, key_mask=key_mask)


@joint_attention.register_fake
def _(q, k, vt, seg_lens, key_mask=None):
    B, H, _, d = q.shape
    return [q.new_empty((B * n, H * d)) for n in seg_lens]


@torch.library.custom_op("b200msat::layernorm", mutates_args=())
def layernorm(x: Tensor, eps: float = 1e-6, scale1p: Optional[Tensor] = None,
              shift: Optional[Tensor] = None) -> Tensor:
    """LayerNorm without affine (optionally * scale1p + shift) over [rows, D]."""
    return ops.layernorm(x, eps, scale1p, shift)


@layernorm.register_fake
def _(x, eps=1e-6, scale1p=None, shift=None):
    return torch.empty_like(x)


@torch.library.custom_op("b200msat::qk_rmsnorm_rope", mutates_args=())
def qk_rmsnorm_rope(x: Tensor, weight: Tensor, pos: Tensor, cos: Tensor, sin: Tensor,
                    eps: float = 1e-6) -> Tensor:
    """Qwen3 per-head RMSNorm + rotate-half RoPE on [T, H, 128]."""
    return ops.qk_rmsnorm_rope(x, weight, pos, cos, sin, eps)


@qk_rmsnorm_rope.register_fake
def _(x, weight, pos, cos, sin, eps=1e-6):
    return torch.empty_like(x)


@torch.library.custom_op("b200msat::swiglu", mutates_args=())
def swiglu(gate: Tensor, up: Tensor) -> Tensor:
    """bf16(bf16(silu(gate)) * up)."""
    return ops.swiglu(gate, up)


@swiglu.register_fake
def _(gate, up):
    return gate.new_empty(gate.shape)


# ---------------------------------------------------------------------------------------------
# token decoding
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("b200msat::qkv_rope_append", mutates_args=("cache",))
def qkv_rope_append(qkv: Tensor, q_norm: Tensor, k_norm: Tensor, cos: Tensor, sin: Tensor, rope_pos: Tensor, cache: Tensor,
                    table: Tensor, lengths: Tensor, cu_seqlens: Tensor, q_heads: int, eps: float = 1e-6) -> Tensor:
    """Per-head norms and rotation of q and k, k and v into the 4-bit cache; q [tokens, q_heads, d]."""
    return ops.qkv_rope_append(qkv, q_norm, k_norm, cos, sin, rope_pos, cache, table, lengths, cu_seqlens, q_heads=q_heads,
                               eps=eps)


@qkv_rope_append.register_fake
def _(qkv, q_norm, k_norm, cos, sin, rope_pos, cache, table, lengths, cu_seqlens, q_heads, eps=1e-6):
    return qkv.new_empty((qkv.shape[0], q_heads, cache.shape[3] // 40))


@torch.library.custom_op("b200msat::kv4_read", mutates_args=())
def kv4_read(cache: Tensor, table: Tensor, lengths: Tensor, cu_seqlens: Tensor, tokens: int) -> Tuple[Tensor, Tensor]:
    """The values that the 4-bit cache holds for the new tokens: k, v [tokens, kv_heads, d]."""
    return ops.kv4_read(cache, table, lengths, cu_seqlens, tokens=tokens)


@kv4_read.register_fake
def _(cache, table, lengths, cu_seqlens, tokens):
    shape = (tokens, cache.shape[1], cache.shape[3] // 40)
    return cache.new_empty(shape, dtype=BF), cache.new_empty(shape, dtype=BF)


@torch.library.custom_op("b200msat::kv4_attention", mutates_args=())
def kv4_attention(q: Tensor, cache: Tensor, table: Tensor, lengths: Tensor, cu_seqlens: Tensor, max_new: int, max_len: int,
                  window: int = 0, sinks: int = 0, scale: Optional[float] = None) -> Tensor:
    """Attention of the new tokens over the 4-bit cache (causal, optional sliding window and sinks)."""
    return ops.kv4_attention(q, cache, table, lengths, cu_seqlens, max_new=max_new, max_len=max_len, window=window,
                             sinks=sinks, scale=scale)


@kv4_attention.register_fake
def _(q, cache, table, lengths, cu_seqlens, max_new, max_len, window=0, sinks=0, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("b200msat::sample", mutates_args=())
def sample(logits: Tensor, u: Tensor, temperature: Optional[Tensor] = None, top_k: Optional[Tensor] = None,
           top_p: Optional[Tensor] = None, min_p: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """One token per row from given numbers: token, logprob, kept."""
    return ops.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)


@sample.register_fake
def _(logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows = logits.shape[0]
    return (logits.new_empty((rows,), dtype=torch.int64), logits.new_empty((rows,), dtype=torch.float32),
            logits.new_empty((rows,), dtype=torch.int32))
