"""Cases of the token-decoding operators: query / key norm + rotation + append to the 4-bit cache,
attention over that cache, and sampling.

Every case names its operator in "op":

  append   q, k rows of a projected [q | k | v] are normed per head and rotated, k and v are
           quantised to 4 bits and written into the paged cache; the outputs are q and the values
           the cache then holds for the new tokens
  attend   softmax attention of the newest tokens' queries over the cache, causal, optionally with
           a sliding window and a few first tokens that stay visible
  sample   temperature, top-k, top-p and min-p, then one draw per row from a given number

Head layouts are the backbone's (16 query / 2 key-value heads of 128) and the action head's
(24 x 64), plus generic ones; 1104 is the backbone's prompt plus cognition tokens, 256 a set of
memory tokens.

The cache is a uint8 tensor [pages, kv_heads, page_size / 32, 40 d]: one unit of 40 d bytes holds K
and V of 32 consecutive tokens of one head.  unit_order() gives where each byte of it stands.
"""

import math

import torch

own = False

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = 32  # tokens of a unit, and channels of a quantisation group


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def append_case(name, seqs, new, ctx, hq, hkv, d, page, table):
    return {"name": name, "op": "append", "seqs": seqs, "new": new, "ctx": ctx, "q_heads": hq, "kv_heads": hkv,
            "head_dim": d, "page": page, "rope": table}


def attend_case(name, seqs, new, ctx, hq, hkv, d, page, window=0, sinks=0):
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "ctx": ctx, "q_heads": hq, "kv_heads": hkv,
            "head_dim": d, "page": page, "window": window, "sinks": sinks}


def sample_case(name, rows, vocab, dtype, filters, pad=0):
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "filters": filters, "pad": pad}


def listed():
    return [
        # one new token of one request: only latency counts
        append_case("append one token", 1, 1, 705, 16, 2, 128, 64, "bf16"),
        # one decode step of a full serving batch
        append_case("append 64 tokens", 64, 1, 4096, 16, 2, 128, 64, "bf16"),
        # prompts of several observations written at once
        append_case("append 8 prompts", 8, 1104, 2300, 16, 2, 128, 64, "f32"),
        # interactive decoding of a short prompt: latency
        attend_case("decode 1 x 705", 1, 1, 705, 16, 2, 128, 64),
        # a serving batch of unequal contexts: the cache's bandwidth
        attend_case("decode 64 x 8192", 64, 1, 8192, 16, 2, 128, 64),
        # few requests with very long histories: the split over the length
        attend_case("decode 3 x 131077", 3, 1, 131077, 16, 2, 128, 128),
        # long histories read through a window and sinks
        attend_case("decode windowed", 16, 1, 50000, 32, 8, 128, 64, window=4096, sinks=67),
        # several proposed tokens checked at once, one key-value head a query head, small heads
        attend_case("check 5 tokens 24 x 64", 12, 5, 2931, 24, 24, 64, 32),
        # new observations' prompts attend over themselves and the history
        attend_case("chunk 8 x 1104", 8, 1104, 2300, 16, 2, 128, 64),
        # one row of logits: latency
        sample_case("sample 1 row", 1, 151680, "bf16", "all"),
        # a serving batch, odd vocabulary, rows in a wider buffer
        sample_case("sample 64 odd rows", 64, 50257, "f32", "mixed", pad=7),
        # the largest batch over the vocabulary of the backbone's prompts
        sample_case("sample 256 rows", 256, 151680, "bf16", "mixed"),
    ]


HEADS = [(16, 2, 128), (16, 2, 128), (32, 8, 128), (24, 24, 64), (8, 1, 64), (12, 4, 128)]


def spread(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "chunk", "sample", "sample"])
    hq, hkv, d = rng.choice(HEADS)
    page = rng.choice([32, 64, 128])
    if kind == "append":
        seqs = spread(rng, 1, 64)
        new = spread(rng, 1, max(1, 8 * 1104 * 2560 // ((hq + 2 * hkv) * d) // seqs))
        c = append_case("", seqs, min(new, 2208), min(new, 2208) + spread(rng, 1, 4096), hq, hkv, d, page,
                        rng.choice(["bf16", "f32"]))
    elif kind == "sample":
        rows = spread(rng, 1, 256)
        vocab = spread(rng, 1000, 151680)
        c = sample_case("", rows, vocab, rng.choice(["bf16", "f32"]) if rows <= 128 else "bf16",
                        rng.choice(["all", "mixed", "temperature"]), rng.choice([0, 0, 5, 64]))
    else:
        new = spread(rng, 1, 8) if kind == "decode" else spread(rng, 16, 1104)
        seqs = spread(rng, 1, 64 if kind == "decode" else 8)
        room = 64 * 8192 * 256 // (hkv * d)
        if kind == "chunk":
            room = min(room, 8 * 2300)
        ctx = max(new, spread(rng, new, max(new, min(131072, room // seqs))))
        window = rng.choice([0, 0, spread(rng, 16, 8192)])
        c = attend_case("", seqs, new, ctx, hq, hkv, d, page, window, rng.choice([0, 4, 67]) if window else 0)
    del c["name"]
    return c


def shares(seqs):
    """A fixed spread of [0, 1) over the sequences, 1 for the first."""
    return [1.0 if b == 0 else (b * 2654435761 % (1 << 32)) / (1 << 32) for b in range(seqs)]


def new_and_lengths(case):
    """New tokens and whole lengths (new ones included) of the case's unequal sequences."""
    new = [case["new"] if case["new"] < 16 else max(1, int(case["new"] * (0.5 + 0.5 * f))) for f in shares(case["seqs"])]
    lens = [max(n, int(case["ctx"] * (0.4 + 0.6 * f))) for n, f in zip(new, shares(case["seqs"]))]
    return new, lens


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + 32 * case["rows"], "flops": 4 * n}
    new, lens = new_and_lengths(case)
    hq, hkv, d, t = case["q_heads"], case["kv_heads"], case["head_dim"], sum(new)
    stored = 2 * hkv * (d // 2 + d // 8)  # bytes of K and V of one token
    if case["op"] == "append":
        rope = 2 * d * (2 if case["rope"] == "bf16" else 4)
        moved = t * ((hq + 2 * hkv) * d * 2 + rope + hq * d * 2 + stored + 2 * hkv * d * 2)
        return {"bytes": moved, "flops": t * (hq + 2 * hkv) * d * 10}
    w, s = case["window"], case["sinks"]
    seen, pairs = 0, 0
    for n, length in zip(new, lens):
        first = length - n  # position of the first new token
        seen += length if not w else min(length, min(s, max(0, first - w + 1)) + n + min(first, w - 1))
        if not w:
            pairs += n * first + n * (n + 1) // 2
        else:
            pairs += sum(min(p + 1, w + min(s, max(0, p + 1 - w))) for p in range(first, length))
    return {"bytes": seen * stored + 2 * t * hq * d * 2, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------
# the 4-bit cache in plain form
# ------------------------------------------------------------------------------------------------
def unit_order(d, device):
    """Place in the unit of each byte of the plain order: K codes [32, d/2], V codes [32, d/2] (byte m
    holds channel 2m in its low and 2m + 1 in its high half), K scales [32, G, 2], K minima, V scales,
    V minima (fp16, G = d / 32 groups)."""
    g_n = d // UNIT
    tok = torch.arange(UNIT, device=device).view(UNIT, 1)
    blk, half, pair, odd = tok // 16, tok // 8 % 2, tok // 2 % 4, tok % 2
    ch = 2 * torch.arange(d // 2, device=device).view(1, d // 2)
    grp, inside = ch // UNIT, ch % UNIT
    k_codes = tok * (d // 2) + inside // 8 * (4 * g_n) + grp * 4 + inside % 8 // 2
    v_codes = (16 * d + blk * 8 * d + half * 4 * d + (inside // 4 * 4 + pair) * 4 * g_n + odd * 2 * g_n + grp * 2
               + inside % 4 // 2)
    tok, blk, half, pair, odd = (x.view(UNIT, 1, 1) for x in (tok, blk, half, pair, odd))
    grp, byte = torch.arange(g_n, device=device).view(1, g_n, 1), torch.arange(2, device=device)
    k_scale = 32 * d + tok * 4 * g_n + grp * 2 + byte
    k_min = k_scale + 2 * g_n
    v_scale = 32 * d + 128 * g_n + blk * 32 * g_n + half * 16 * g_n + pair * 4 * g_n + grp * 4 + odd * 2 + byte
    v_min = v_scale + 64 * g_n
    return k_codes, v_codes, k_scale, k_min, v_scale, v_min


def quantise(x):
    """x [..., d] -> codes uint8 [..., d], scale and minimum fp16 [..., d / 32]."""
    x = x.float().unflatten(-1, (-1, UNIT))
    top, low = x.amax(-1).clamp(-65504, 65504), x.amin(-1).clamp(-65504, 65504)
    low, scale = low.to(F16), ((top - low) * (1.0 / 15.0)).to(F16)
    s = scale.float()
    inverse = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    codes = ((x - low.float().unsqueeze(-1)) * inverse.unsqueeze(-1)).round().clamp(0, 15)
    return codes.nan_to_num(0.0).to(torch.uint8).flatten(-2), scale, low


def dequantise(codes, scale, low):
    x = codes.float().unflatten(-1, (-1, UNIT))
    return (x * scale.float().unsqueeze(-1) + low.float().unsqueeze(-1)).flatten(-2)


def packed(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def unpacked(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def fp16_bytes(x):
    return x.contiguous().view(torch.uint8).unflatten(-1, (-1, 2))


def from_bytes(b):
    return b.flatten(-2).contiguous().view(F16)


def pack_units(k, v):
    """k, v [..., 32, d] fp32 -> units [..., 40 d]."""
    d = k.shape[-1]
    unit = torch.empty(*k.shape[:-2], 40 * d, dtype=torch.uint8, device=k.device)
    order = unit_order(d, k.device)
    (kc, ks, kl), (vc, vs, vl) = quantise(k), quantise(v)
    for where, what in zip(order, (packed(kc), packed(vc), fp16_bytes(ks), fp16_bytes(kl), fp16_bytes(vs), fp16_bytes(vl))):
        unit[..., where] = what
    return unit


def unpack_units(unit):
    """units [..., 40 d] -> k, v [..., 32, d] fp32."""
    kc, vc, ks, kl, vs, vl = (unit[..., where] for where in unit_order(unit.shape[-1] // 40, unit.device))
    return (dequantise(unpacked(kc), from_bytes(ks), from_bytes(kl)),
            dequantise(unpacked(vc), from_bytes(vs), from_bytes(vl)))


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def rope_tables(rows, d, dtype, device):
    inv = 1.0 / (1e6 ** (torch.arange(0, d, 2, device=device).float() / d))
    angle = torch.outer(torch.arange(rows, device=device).float(), inv)
    angle = torch.cat((angle, angle), -1)
    return angle.cos().to(dtype), angle.sin().to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        wide = torch.empty(rows, vocab + case["pad"], dtype=BF16 if case["dtype"] == "bf16" else F32, device=dev)
        logits = wide[:, :vocab]
        # a language model's rows: a bulk of unlikely tokens and a few that stand out
        logits.copy_(2.0 * randn(rows, vocab) - 4.0)
        logits.scatter_add_(1, torch.randint(vocab, (rows, 40), device=dev, generator=g), (6.0 + 3.0 * randn(rows, 40)).to(wide.dtype))
        logits[:, vocab - vocab // 50:] = -math.inf  # ids that are never to be produced

        def pick(values):
            return torch.tensor(values, device=dev)[torch.randint(len(values), (rows,), device=dev, generator=g)]

        u = torch.rand(rows, device=dev, generator=g)
        if case["filters"] == "temperature":
            p = {"temperature": pick([0.7, 1.0, 1.3]), "top_k": None, "top_p": None, "min_p": None}
        elif case["filters"] == "all":
            p = {"temperature": pick([0.8]), "top_k": pick([50]).int(), "top_p": pick([0.95]), "min_p": pick([0.02])}
        else:
            p = {"temperature": pick([0.0, 0.6, 0.9, 1.0, 1.5]), "top_k": pick([0, 1, 20, 1000]).int(),
                 "top_p": pick([0.5, 0.9, 0.95, 1.0]), "min_p": pick([0.0, 0.0, 0.05])}
        return {"case": case, "logits": logits, "u": u, **p}

    new, lens = new_and_lengths(case)
    hq, hkv, d, page, seqs = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    held = [-(-n // page) for n in lens]
    width, pages = max(held) + 1, sum(held) + 3
    # pages of a sequence lie anywhere in the pool; entries past its length name none
    shuffled = torch.randperm(pages, device=dev, generator=g).int()
    table = torch.full((seqs, width), -1, dtype=torch.int32, device=dev)
    used = torch.arange(width, device=dev) < torch.tensor(held, device=dev).unsqueeze(1)
    table[used] = shuffled[: sum(held)]
    cu = torch.tensor([0] + new, device=dev).cumsum(0).int()
    state = {"case": case, "table": table, "lengths": torch.tensor(lens, dtype=torch.int32, device=dev), "cu": cu,
             "max_new": max(new), "max_len": max(lens)}
    t = sum(new)
    if case["op"] == "append":
        state["cache"] = torch.zeros(pages, hkv, page // UNIT, 40 * d, dtype=torch.uint8, device=dev)
        # keys have channels that stand out from zero
        offset = torch.cat((torch.zeros(hq * d, device=dev), randn(hkv * d), torch.zeros(hkv * d, device=dev)))
        state["qkv"] = (randn(t, (hq + 2 * hkv) * d) + offset).to(BF16)
        state["q_norm"], state["k_norm"] = ((1.2 + 0.2 * randn(d)).to(BF16) for _ in range(2))
        state["cos"], state["sin"] = rope_tables(max(lens), d, BF16 if case["rope"] == "bf16" else F32, dev)
        state["rope_pos"] = torch.cat([torch.arange(n - m, n, dtype=torch.int32, device=dev) for m, n in zip(new, lens)])
    else:
        shape = (pages, hkv, page // UNIT, UNIT, d)
        state["cache"] = pack_units(1.2 * randn(*shape) + randn(hkv, 1, 1, d), randn(*shape))
        state["q"] = (1.5 * randn(t, hq, d)).to(BF16)
    return state


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def normed_and_rotated(x, weight, cos, sin):
    """x [T, H, d] -> rotate-half RoPE of its per-head RMS norm."""
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()
    a, b = x.chunk(2, -1)
    return x * cos.float().unsqueeze(1) + torch.cat((-b, a), -1) * sin.float().unsqueeze(1)


def token_places(s):
    """Sequence, position and place in the cache (page, unit, token of the unit) of every new token."""
    cu, lengths, page = s["cu"].long(), s["lengths"].long(), s["case"]["page"]
    rows = torch.arange(s["qkv"].shape[0], device=cu.device)
    seq = torch.searchsorted(cu, rows, right=True) - 1
    pos = lengths[seq] - cu[seq + 1] + rows
    return s["table"][seq, pos // page].long(), pos % page // UNIT, pos % UNIT


def plain_append(s):
    c = s["case"]
    hq, hkv, d = c["q_heads"], c["kv_heads"], c["head_dim"]
    q, k, v = s["qkv"].unflatten(1, (-1, d)).split((hq, hkv, hkv), 1)
    cos, sin = s["cos"][s["rope_pos"].long()], s["sin"][s["rope_pos"].long()]
    q = normed_and_rotated(q, s["q_norm"], cos, sin)
    k = normed_and_rotated(k, s["k_norm"], cos, sin)
    (kc, ks, kl), (vc, vs, vl) = quantise(k), quantise(v)
    page, unit, tok = token_places(s)
    head = torch.arange(hkv, device=page.device)
    for where, what in zip(unit_order(d, page.device),
                           (packed(kc), packed(vc), fp16_bytes(ks), fp16_bytes(kl), fp16_bytes(vs), fp16_bytes(vl))):
        where, what = where.flatten(1)[tok].unsqueeze(1), what.flatten(2)
        s["cache"][page.view(-1, 1, 1), head.view(1, -1, 1), unit.view(-1, 1, 1), where] = what
    return {"q": q.to(BF16), "k": dequantise(kc, ks, kl).to(BF16), "v": dequantise(vc, vs, vl).to(BF16)}


def plain_attend(s):
    c = s["case"]
    hq, hkv, d, dev = c["q_heads"], c["kv_heads"], c["head_dim"], s["q"].device
    cu, lengths = s["cu"].long(), s["lengths"].long()
    new = cu[1:] - cu[:-1]
    span = -(-s["max_len"] // c["page"])
    units = s["cache"][s["table"][:, :span].long().clamp_min(0)]  # [B, span, Hkv, units, 40 d]
    k, v = (x.permute(0, 2, 1, 3, 4, 5).flatten(2, 4) for x in unpack_units(units))  # [B, Hkv, L, d]
    row = torch.arange(s["max_new"], device=dev)
    real = row < new.unsqueeze(1)  # [B, Q]
    at = (cu[:-1].unsqueeze(1) + row).clamp_max(s["q"].shape[0] - 1)
    q = s["q"].float()[at].unflatten(2, (hkv, hq // hkv))  # [B, Q, Hkv, R, d]
    q = q.permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, Hkv, R Q, d]
    pos = (lengths - new).unsqueeze(1) + row  # [B, Q]
    key = torch.arange(k.shape[2], device=dev)
    seen = (key <= pos.unsqueeze(-1)) & (key < lengths.view(-1, 1, 1))
    if c["window"]:
        seen &= (pos.unsqueeze(-1) - key < c["window"]) | (key < c["sinks"])
    hidden = ~seen.repeat(1, hq // hkv, 1).unsqueeze(1)  # [B, 1, R Q, L]
    w = (q @ k.transpose(-1, -2) * d ** -0.5).masked_fill_(hidden, -math.inf)
    w = (w - w.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    o = w @ v / w.sum(-1, keepdim=True).clamp_min(1e-38)
    o = o.unflatten(2, (hq // hkv, -1)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, Q, Hq, d]
    return o[real].to(BF16)


def param(s, name, off):
    return s[name].unsqueeze(1) if s[name] is not None else torch.full_like(s["u"], off).unsqueeze(1)


def plain_sample(s):
    x = s["logits"].float() + 0.0
    t, k, p, m = (param(s, n, off) for n, off in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = x[:, :1]
    w = torch.where(x == top, torch.zeros_like(x), (x - top) / t.clamp_min(1e-30))
    w = (w.exp() * 4294967296.0).long()  # weights as whole numbers: their sums have no order
    rank = torch.arange(x.shape[1], device=x.device)
    w = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    before = w.cumsum(-1) - w
    total = w.sum(-1, keepdim=True)
    kept = (w > 0) & ((p >= 1) | (before.double() < p.double() * total.double()) | (rank == 0))
    kept &= w.double() >= m.double() * 4294967296.0
    kept = torch.where(t > 0, kept, rank == 0)
    w = torch.where(kept, w, torch.zeros_like(w))
    by_id = torch.zeros_like(w).scatter_(1, order, w)
    reach = by_id.cumsum(-1)
    total = reach[:, -1:]
    goal = (s["u"].unsqueeze(1).double() * total.double()).long().clamp_max(total - 1)
    token = (reach <= goal).sum(-1)
    chosen = by_id.gather(1, token.unsqueeze(1))
    return {"token": token, "logprob": (chosen.double() / total.double()).log().float().squeeze(1), "kept": kept.sum(-1).int()}


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": plain_append, "attend": plain_attend, "sample": plain_sample}[op](state)
    from rldx_b200 import ops

    s, c = state, state["case"]
    if op == "append":
        q = ops.qkv_rope_append(s["qkv"], s["q_norm"], s["k_norm"], s["cos"], s["sin"], s["rope_pos"], s["cache"],
                                s["table"], s["lengths"], s["cu"], q_heads=c["q_heads"])
        k, v = ops.kv4_read(s["cache"], s["table"], s["lengths"], s["cu"], tokens=q.shape[0])
        return {"q": q, "k": k, "v": v}
    if op == "attend":
        return ops.kv4_attention(s["q"], s["cache"], s["table"], s["lengths"], s["cu"], max_new=s["max_new"],
                                 max_len=s["max_len"], window=c["window"], sinks=c["sinks"])
    token, logprob, kept = ops.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"])
    return {"token": token, "logprob": logprob, "kept": kept}


# ------------------------------------------------------------------------------------------------
# values in 64 bits, one sequence or row at a time
# ------------------------------------------------------------------------------------------------
def stored_value(units, tok, d, which):
    """Values [H, n, d] in 64 bits that the cache holds for tokens `tok` of the units [n, H, 40 d]:
    which = 0 for K, 1 for V, byte by byte from the description of the unit."""
    groups, n = d // 32, tok.numel()
    rows, heads = torch.arange(n, device=tok.device).view(n, 1, 1), torch.arange(units.shape[1], device=tok.device).view(1, -1, 1)
    ch = torch.arange(d, device=tok.device).view(1, 1, d)
    tok = tok.view(n, 1, 1)
    group = ch // 32
    lane_pair = tok % 8 // 2
    if which == 0:
        code_at = tok * (d // 2) + (ch % 32 // 8) * 4 * groups + group * 4 + ch % 8 // 2
        scale_at = 32 * d + tok * 4 * groups + group * 2
        low_at = scale_at + 2 * groups
    else:
        code_at = 16 * d + (tok // 8) * 4 * d + ((ch % 32 // 4) * 4 + lane_pair) * 4 * groups + tok % 2 * 2 * groups + group * 2 + ch % 4 // 2
        scale_at = 32 * d + 128 * groups + (tok // 8) * 16 * groups + lane_pair * 4 * groups + group * 4 + tok % 2 * 2
        low_at = scale_at + 64 * groups
    byte = units[rows, heads, code_at].long()
    code = torch.where(ch % 2 == 0, byte % 16, byte // 16).double()

    def half(at):
        b = units[rows, heads, at].to(torch.int16) | (units[rows, heads, at + 1].to(torch.int16) << 8)
        return b.view(F16).double()

    return (half(scale_at) * code + half(low_at)).transpose(0, 1)


def exact_append(case, s):
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
    pos = s["rope_pos"].long()
    c, sn = s["cos"].double()[pos][:, None], s["sin"].double()[pos][:, None]
    weight = torch.cat((s["q_norm"].double().expand(hq, d), s["k_norm"].double().expand(hkv, d)))
    y = x[:, : hq + hkv]
    y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * weight
    h = d // 2
    y = torch.cat((y[..., :h] * c[..., :h] - y[..., h:] * sn[..., :h], y[..., h:] * c[..., h:] + y[..., :h] * sn[..., h:]), -1)

    def held(z):
        z = z.reshape(*z.shape[:2], d // 32, 32)
        low = z.min(-1, keepdim=True).values.half().double()
        step = ((z.max(-1, keepdim=True).values - z.min(-1, keepdim=True).values) / 15).half().double()
        code = ((z - low) / step.clamp_min(1e-30)).round().clamp(0, 15)
        return (low + step * code).reshape(*z.shape[:2], d)

    return {"q": y[:, :hq], "k": held(y[:, hq:]), "v": held(x[:, hq + hkv:])}


def exact_attend(case, s):
    hq, hkv, d, page = case["q_heads"], case["kv_heads"], case["head_dim"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    cu, lens = s["cu"].tolist(), s["lengths"].tolist()
    for b, length in enumerate(lens):
        j = torch.arange(length, device=out.device)
        units = s["cache"][s["table"][b, j // page].long(), :, j % page // 32]
        k, v = (stored_value(units, j % 32, d, which) for which in (0, 1))
        q = s["q"][cu[b]: cu[b + 1]].double().view(-1, hkv, hq // hkv, d)
        p = torch.arange(length - q.shape[0], length, device=out.device).view(-1, 1)
        ok = j <= p
        if case["window"]:
            ok = ok & ((j > p - case["window"]) | (j < case["sinks"]))
        for h in range(hkv):
            e = torch.einsum("qrd,kd->rqk", q[:, h], k[h]) / math.sqrt(d)
            e = torch.where(ok, e, torch.full_like(e, -math.inf)).softmax(-1)
            out[cu[b]: cu[b + 1], h * (hq // hkv): (h + 1) * (hq // hkv)] = torch.einsum("rqk,kd->qrd", e, v[h])
    return out


def exact_sample(case, s):
    """The weights are by definition whole numbers made of a 32-bit exponential; all else is in 64 bits."""
    logprob = []
    for r in range(case["rows"]):
        x = s["logits"][r].float()
        t, k, p, m = (None if s[n] is None else s[n][r].item() for n in ("temperature", "top_k", "top_p", "min_p"))
        if t is not None and not t > 0:
            logprob.append(0.0)
            continue
        w = torch.exp((x - x.max()) / torch.tensor(1.0 if t is None else t, device=x.device)).double().mul(2.0 ** 32).floor()
        keep = torch.zeros_like(x, dtype=torch.bool)
        ids = torch.argsort(x, descending=True, stable=True)
        ids = ids[: k] if k else ids
        run_w = w[ids].cumsum(0)
        if p is not None and p < 1:
            ids = ids[: int((run_w < s["top_p"][r].double() * run_w[-1]).sum()) + 1]
        keep[ids] = True
        if m is not None:
            keep &= w >= s["min_p"][r].double() * 2.0 ** 32
        w = w * keep
        goal = torch.floor(s["u"][r].double() * w.sum())
        token = int(torch.searchsorted(w.cumsum(0), goal, right=True))
        logprob.append(math.log(float(w[token]) / float(w.sum())))
    return {"token": None, "logprob": torch.tensor(logprob, dtype=torch.float64), "kept": None}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": exact_append, "attend": exact_attend, "sample": exact_sample}[case["op"]](case, s)
