"""Cases of the operators around a decoder's products: rotary positions, the norms after and before a
block, and the log probabilities of given tokens.

Every case names its operator in "op":

  rope      q and k heads are rotated by angles made from positions and frequencies: halves or neighbours
            as pairs, a part of the head, positions of one or three axes, frequencies scaled for long
            contexts, forwards or backwards
  rows      the same angles written as cos / sin rows for a kernel that rotates with a table
  norms     residual + scale * gate * norm(branch), and the norm of that sum for the next block, with its
            modulation
  logprobs  of given tokens under rows of logits, with the entropy, the token's rank and the top alternatives

Head layouts are the backbone's (16 query / 2 key-value heads of 128) and the action head's (24 x 64),
widths theirs (2048 and 1536) and generic ones; 1104 is the backbone's prompt plus cognition tokens, 562
the action head's joint sequence, 151680 the vocabulary of the backbone's prompts.
"""

import math

import torch

own = False

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
TYPES = {"bf16": BF16, "f16": F16, "f32": F32}


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def rope_case(name, op, tokens, hq, hk, d, rotary, dtype, pairs="halves", axes="one", scaling="none", reach=32768,
              inverse=False, where="rows of qkv"):
    return {"name": name, "op": op, "tokens": tokens, "q_heads": hq, "k_heads": hk, "head_dim": d, "rotary": rotary,
            "dtype": dtype, "pairs": pairs, "axes": axes, "scaling": scaling, "reach": reach, "inverse": inverse, "where": where}


def norms_case(name, rows, width, dtype, stream, post, pre, gate="none", modulation="none", group=0, plus_one=False, scale=1.0,
               pad=0):
    return {"name": name, "op": "norms", "rows": rows, "width": width, "dtype": dtype, "stream": stream, "post": post,
            "pre": pre, "gate": gate, "modulation": modulation, "group": group, "plus_one": plus_one, "scale": scale, "pad": pad}


def logprobs_case(name, rows, vocab, dtype, top, pad=0, unnamed=0):
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top, "pad": pad,
            "unnamed": unnamed}


def listed():
    return [
        # one new token of one request, positions of three axes as its vision prompt has them: only latency counts
        rope_case("rope one token", "rope", 1, 16, 2, 128, 128, "bf16", axes="interleaved"),
        # prompts of several observations, frequencies of three axes side by side
        rope_case("rope 8 prompts", "rope", 8 * 1104, 16, 2, 128, 128, "bf16", axes="sections"),
        # a part of the head, neighbours as pairs, far positions with frequencies ramped for them, odd count
        rope_case("rope far half heads", "rope", 20011, 24, 24, 64, 32, "f32", pairs="neighbours", scaling="ramp", reach=1 << 20,
                  where="own"),
        # the bound of memory: the largest head layout that the framework's norm and rotation is quoted on
        rope_case("rope 65536 x 32 heads", "rope", 65536, 16, 16, 128, 128, "bf16", scaling="stretch", reach=65536, where="own"),
        # cos and sin for the prompts of a serving batch, read by the kernel that fills the cache
        rope_case("rows 8 prompts", "rows", 8 * 1104, 0, 0, 128, 128, "f32", axes="interleaved"),
        # one decode step of one request between two blocks: latency
        norms_case("norms one row", 1, 2048, "bf16", "bf16", "rms", "rms"),
        # prompts of several observations through a block with norms on both sides
        norms_case("norms 8 prompts", 8 * 1104, 2048, "bf16", "bf16", "rms", "rms", gate="channels", plus_one=True, scale=0.5),
        # a batch of joint sequences, gate and modulation of each observation's time step
        norms_case("norms 64 x 562 modulated", 64 * 562, 1536, "bf16", "bf16", "none", "layer", gate="groups",
                   modulation="groups", group=562),
        # a stream kept in 32 bits, an odd width in wider rows, a norm with bias
        norms_case("norms odd f32 stream", 4999, 1001, "f16", "f32", "layer", "rms", gate="channels", pad=3),
        # one row of logits: latency
        logprobs_case("logprobs one row", 1, 151680, "bf16", 5),
        # a serving batch, odd vocabulary, rows in a wider buffer, rows without a token
        logprobs_case("logprobs 64 odd rows", 64, 50257, "f32", 20, pad=7, unnamed=5),
        # a scored prompt of the largest vocabulary
        logprobs_case("logprobs 2208 rows", 2208, 151680, "bf16", 20),
    ]


HEADS = [(16, 2, 128), (16, 2, 128), (16, 16, 128), (24, 24, 64), (32, 8, 128), (8, 1, 256), (12, 4, 96), (16, 16, 72)]
MOST_BYTES = 65536 * 32 * 128 * 2 * 2


def spread(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["rope", "rope", "rows", "norms", "norms", "logprobs", "logprobs"])
    if op in ("rope", "rows"):
        hq, hk, d = rng.choice(HEADS)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"]) if op == "rope" else rng.choice(["bf16", "f32"])
        size = 4 if dtype == "f32" else 2
        most = MOST_BYTES // ((hq + hk) * d * 2 * size) if op == "rope" else 65536
        rotary = d if op == "rows" else rng.choice([d, d, d // 2, d // 4])
        axes = rng.choice(["one", "one", "sections", "interleaved"])
        c = rope_case("", op, spread(rng, 1, min(65536, most)), hq if op == "rope" else 0, hk if op == "rope" else 0, d, rotary,
                      dtype, rng.choice(["halves", "neighbours"]) if op == "rope" else "halves", axes,
                      rng.choice(["none", "stretch", "ramp"]), spread(rng, 4096, 1 << 20),
                      op == "rope" and rng.random() < 0.25, rng.choice(["rows of qkv", "own"]))
    elif op == "norms":
        dtype, width = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([rng.randint(1, 700), 8 * rng.randint(8, 1024), spread(rng, 64, 8192)])
        stream = "f32" if dtype == "f32" else rng.choice([dtype, dtype, "f32"])
        per_row = width * (2 * (4 if dtype == "f32" else 2) + 2 * (4 if stream == "f32" else 2))
        rows = spread(rng, 1, max(1, 64 * 562 * 1536 * 8 // per_row))
        group = rng.choice([1, spread(rng, 1, rows), spread(rng, 1, rows)])
        group = max(group, -(-rows * width // (1 << 24)))  # gates and modulations stay a small part
        c = norms_case("", rows, width, dtype, stream, rng.choice(["none", "rms", "rms", "layer"]), rng.choice(["rms", "layer"]),
                       rng.choice(["none", "channels", "groups"]), rng.choice(["none", "none", "groups"]), group,
                       rng.random() < 0.3, rng.choice([1.0, 0.22, 0.5]), rng.choice([0, 0, 1, 8]))
    else:
        dtype, vocab = rng.choice(["bf16", "bf16", "f16", "f32"]), spread(rng, 1000, 151680)
        rows = spread(rng, 1, max(1, min(8192, 2208 * 151680 * 2 // (vocab * (4 if dtype == "f32" else 2)))))
        c = logprobs_case("", rows, vocab, dtype, rng.choice([0, 1, 5, 20, 32]), rng.choice([0, 0, 5, 64]),
                          rng.choice([0, 0, 7]))
    del c["name"]
    return c


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
        return {"bytes": 2 * n * TYPES[case["dtype"]].itemsize + 8 * case["tokens"] * (1 if case["axes"] == "one" else 3),
                "flops": 3 * n * case["rotary"] // case["head_dim"]}
    if case["op"] == "rows":
        n = case["tokens"] * case["head_dim"]
        return {"bytes": 2 * n * TYPES[case["dtype"]].itemsize + 8 * case["tokens"] * (1 if case["axes"] == "one" else 3), "flops": 10 * n}
    if case["op"] == "norms":
        n, p = case["rows"] * case["width"], TYPES[case["dtype"]].itemsize
        groups = -(-case["rows"] // case["group"]) if case["group"] else 1
        read = (case["post"] != "none") * (2 if case["post"] == "layer" else 1) + 1  # weights and biases
        read += {"none": 0, "channels": 1, "groups": groups}[case["gate"]] + {"none": 0, "groups": 2 * groups}[case["modulation"]]
        return {"bytes": n * 2 * (p + TYPES[case["stream"]].itemsize) + read * case["width"] * p, "flops": 14 * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * TYPES[case["dtype"]].itemsize + case["rows"] * (20 + 12 * case["top"]), "flops": 6 * n}


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def plan_of(case):
    """What makes the frequencies: theta 1e6, pairs of the rotated part, three axes in the backbone's shares."""
    half = case["rotary"] // 2
    a = half * 20 // 64
    sections = None if case["axes"] == "one" else (half - 2 * a, a, a)
    scaling = {"none": None, "stretch": {"type": "linear", "factor": 4.0},
               "ramp": {"type": "yarn", "factor": 32.0, "original": 32768}}[case["scaling"]]
    return sections, scaling


def frequencies(case, device):
    """float64 [rotary / 2] radians a position, and the factor on cos and sin."""
    r, theta = case["rotary"], 1e6
    i = torch.arange(0, r, 2, dtype=F64, device=device)
    f = theta ** (-i / r)
    if case["scaling"] == "stretch":
        return f / 4.0, 1.0
    if case["scaling"] == "ramp":
        # turns over the original length: above 32 kept, below 1 divided, between blended linearly in the pair's index
        def pair_at(turns):
            return r * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(math.floor(pair_at(32.0)), 0), min(math.ceil(pair_at(1.0)), r - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return f / 32.0 * ramp + f * (1 - ramp), 0.1 * math.log(32.0) + 1.0
    return f, 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    dtype = TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] in ("rope", "rows"):
        t, hq, hk, d = case["tokens"], case["q_heads"], case["k_heads"], case["head_dim"]
        start = torch.randint(max(1, case["reach"] - t), (1,), device=dev, generator=g)
        at = start + torch.arange(t, device=dev)
        if case["axes"] != "one":  # a grid of patches: the second and third axis go over its rows and columns
            at = torch.stack((at, start + at % 1104 // 14, start + at % 14))
        state["positions"] = at
        state["freqs"], state["factor"] = frequencies(case, dev)
        if case["op"] == "rope":
            if case["where"] == "own":
                state["q"], state["k"] = randn(t, hq, d).to(dtype), randn(t, hk, d).to(dtype)
            else:
                qkv = randn(t, (hq + 2 * hk) * d).to(dtype).unflatten(1, (-1, d))
                state["q"], state["k"] = qkv[:, :hq], qkv[:, hq: hq + hk]
        if own:
            from rldx_b200.rope import B200Rope

            sections, scaling = plan_of(case)
            state["rope"] = B200Rope(case["head_dim"], theta=1e6, rotary_dim=case["rotary"],
                                     interleaved=case["pairs"] == "neighbours", sections=sections,
                                     interleaved_sections=case["axes"] == "interleaved", scaling=scaling, device=dev)
        return state
    if case["op"] == "norms":
        n, w, stream = case["rows"], case["width"], TYPES[case["stream"]]
        groups = -(-n // case["group"]) if case["group"] else 1

        def rows(kind, size):
            return torch.empty(n, w + case["pad"], dtype=kind, device=dev)[:, :w].copy_(size * randn(n, w) + 0.3 * randn(w))

        state["branch"], state["residual"] = rows(dtype, 0.7), rows(stream, 3.0)
        one = 0.0 if case["plus_one"] else 1.0
        state["post_weight"] = (one + 0.2 * randn(w)).to(dtype) if case["post"] != "none" else None
        state["post_bias"] = (0.2 * randn(w)).to(dtype) if case["post"] == "layer" else None
        state["pre_weight"] = (one + 0.2 * randn(w)).to(dtype)
        state["gate"] = {"none": None, "channels": (0.8 * randn(w)).to(dtype), "groups": (0.8 * randn(groups, w)).to(dtype)}[case["gate"]]
        wide = (0.5 * randn(groups, 2 * w)).to(dtype) if case["modulation"] != "none" else None  # one product makes both
        state["mod_scale"], state["mod_shift"] = (None, None) if wide is None else (wide[:, :w], wide[:, w:])
        return state
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty(rows, vocab + case["pad"], dtype=dtype, device=dev)[:, :vocab]
    # a language model's rows: a bulk of unlikely tokens, a few that stand out, ids that are never to be produced
    logits.copy_(torch.randn(rows, vocab, device=dev, generator=g).mul_(2.0).sub_(4.0))
    hot = torch.randint(vocab, (rows, 1), device=dev, generator=g) + torch.arange(40, device=dev) * (vocab // 40)
    hot %= vocab  # different ones: sums in any order
    logits.scatter_add_(1, hot, (6.0 + 3.0 * randn(rows, 40)).to(dtype))
    logits[:, vocab - vocab // 50:] = -math.inf
    # half of the tokens are among those that stand out, the others any that can be
    token = torch.where(torch.rand(rows, device=dev, generator=g) < 0.5, hot[:, 0],
                        torch.randint(vocab, (rows,), device=dev, generator=g)).clamp_max(vocab - vocab // 50 - 1)
    if case["unnamed"]:
        token[::case["unnamed"]] = -1
    state["logits"], state["tokens"] = logits, token
    return state


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------
def axis_of(case, device):
    """The axis whose position each pair takes."""
    half = case["rotary"] // 2
    sections, _ = plan_of(case)
    i = torch.arange(half, device=device)
    if sections is None:
        return torch.zeros_like(i)
    bounds = torch.tensor(sections, device=device)
    if case["axes"] == "sections":
        return torch.searchsorted(bounds.cumsum(0), i, right=True)
    return torch.where(i < 3 * bounds[i % 3], i % 3, torch.zeros_like(i))


def plain_angles(s):
    """cos, sin [tokens, rotary / 2] in 32 bits; the angles in 64, as far positions need them."""
    at = s["positions"] if s["positions"].dim() == 2 else s["positions"].unsqueeze(0)
    angle = at[axis_of(s["case"], at.device)].t().double() * s["freqs"]
    return (angle.cos() * s["factor"]).float(), (angle.sin() * s["factor"]).float()


def plain_rope(s):
    c = s["case"]
    cos, sin = (x.unsqueeze(1) for x in plain_angles(s))
    if c["inverse"]:
        sin = -sin
    out = []
    for x in (s["q"], s["k"]):
        y = x.float()
        part, rest = y[..., : c["rotary"]], y[..., c["rotary"]:]
        if c["pairs"] == "halves":
            a, b = part.chunk(2, -1)
            part = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        out.append(torch.cat((part, rest), -1).to(x.dtype))
    return {"q": out[0], "k": out[1]}


def plain_rows(s):
    return {n: torch.cat((x, x), -1).to(TYPES[s["case"]["dtype"]]) for n, x in zip(("cos", "sin"), plain_angles(s))}


def plain_norm(x, kind, weight, bias, plus_one):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    if weight is not None:
        x = x * (weight.float() + (1.0 if plus_one else 0.0))
    return x if bias is None else x + bias.float()


def of_rows(x, case):
    """A vector for every row, or each group's."""
    if x is None or x.dim() == 1:
        return None if x is None else x.float()
    return x.float().repeat_interleave(case["group"], 0)[: case["rows"]]


def plain_norms(s):
    c = s["case"]
    y = plain_norm(s["branch"].float(), c["post"], s["post_weight"], s["post_bias"], c["plus_one"])
    if s["gate"] is not None:
        y = y * of_rows(s["gate"], c)
    h = s["residual"].float() + c["scale"] * y
    n = plain_norm(h, c["pre"], s["pre_weight"], None, c["plus_one"])
    if s["mod_scale"] is not None:
        n = n * (1.0 + of_rows(s["mod_scale"], c)) + of_rows(s["mod_shift"], c)
    return {"residual": h.to(s["residual"].dtype), "out": n.to(s["branch"].dtype)}


def plain_logprobs(s):
    x, token, top = s["logits"].float(), s["tokens"], s["case"]["top"]
    given = token >= 0
    mine = x.gather(1, token.clamp_min(0).unsqueeze(1))
    ids = torch.arange(x.shape[1], device=x.device)
    rank = ((x > mine) | ((x == mine) & (ids < token.unsqueeze(1)))).sum(-1)
    d = x - x.amax(-1, keepdim=True)
    w = d.exp()
    total = w.sum(-1, keepdim=True)
    log_total = total.log()
    entropy = log_total.squeeze(1) - torch.where(w > 0, w * d, torch.zeros_like(w)).sum(-1) / total.squeeze(1)
    logprob = (d.gather(1, token.clamp_min(0).unsqueeze(1)) - log_total).squeeze(1)
    out = {"logprob": torch.where(given, logprob, torch.zeros_like(logprob)), "entropy": entropy,
           "rank": torch.where(given, rank, torch.full_like(rank, -1)).int()}
    if top:
        del w
        d, order = torch.sort(d, dim=-1, descending=True, stable=True)  # of equal ones the lowest id first
        out["top_ids"], out["top_logprobs"] = order[:, :top].contiguous(), d[:, :top] - log_total
    return out


def run(state):
    s, c = state, state["case"]
    op = c["op"]
    if not own:
        return {"rope": plain_rope, "rows": plain_rows, "norms": plain_norms, "logprobs": plain_logprobs}[op](s)
    from rldx_b200 import ops

    if op == "rope":
        q, k = s["rope"](s["q"], s["k"], s["positions"], inverse=c["inverse"])
        return {"q": q, "k": k}
    if op == "rows":
        cos, sin = s["rope"].rows(s["positions"], dtype=TYPES[c["dtype"]])
        return {"cos": cos, "sin": sin}
    if op == "norms":
        residual, out = ops.block_norms(s["branch"], s["residual"], post=c["post"], post_weight=s["post_weight"],
                                        post_bias=s["post_bias"], gate=s["gate"], scale=c["scale"], pre=c["pre"],
                                        pre_weight=s["pre_weight"], mod_scale=s["mod_scale"], mod_shift=s["mod_shift"],
                                        rows_per_group=c["group"], weight_plus_one=c["plus_one"])
        return {"residual": residual, "out": out}
    logprob, entropy, rank, top_ids, top_logprobs = ops.token_logprobs(s["logits"], s["tokens"], top=c["top"])
    out = {"logprob": logprob, "entropy": entropy, "rank": rank}
    if c["top"]:
        out["top_ids"], out["top_logprobs"] = top_ids, top_logprobs
    return out


# ------------------------------------------------------------------------------------------------
# values in 64 bits, written apart from the plain forms
# ------------------------------------------------------------------------------------------------
def exact_turns(case, s):
    """Complex numbers [tokens, pairs] that the pairs are multiplied by."""
    half = case["rotary"] // 2
    at = s["positions"].reshape(-1, case["tokens"]).double()
    sections, _ = plan_of(case)
    columns = []
    for i in range(half):
        axis = 0
        if case["axes"] == "sections":
            axis = 0 if i < sections[0] else 1 if i < sections[0] + sections[1] else 2
        elif case["axes"] == "interleaved" and i < 3 * sections[i % 3]:
            axis = i % 3
        columns.append(at[axis] * s["freqs"][i])
    angle = torch.stack(columns, 1)
    return torch.polar(torch.full_like(angle, s["factor"]), angle)


def exact_rope(case, s):
    turn = exact_turns(case, s)
    if case["op"] == "rows":
        return {"cos": turn.real.repeat(1, 2), "sin": turn.imag.repeat(1, 2)}
    turn = (turn.conj() if case["inverse"] else turn).unsqueeze(1)
    half, out = case["rotary"] // 2, {}
    for name in ("q", "k"):
        x = s[name].double()
        y = x.clone()
        if case["pairs"] == "halves":
            z = torch.complex(x[..., :half], x[..., half: 2 * half]) * turn
            y[..., :half], y[..., half: 2 * half] = z.real, z.imag
        else:
            z = torch.view_as_complex(x[..., : 2 * half].unflatten(-1, (half, 2)).contiguous()) * turn
            y[..., : 2 * half] = torch.view_as_real(z).flatten(-2)
        out[name] = y
    return out


def exact_norms(case, s):
    def norm(x, kind, weight, bias):
        if kind == "none":
            return x
        middle = x.mean(1, keepdim=True) if kind == "layer" else 0.0
        spread_ = ((x - middle) ** 2).sum(1, keepdim=True) / x.shape[1]
        x = (x - middle) / (spread_ + 1e-6).sqrt() * (weight.double() + float(case["plus_one"]))
        return x + bias.double() if bias is not None else x

    def rows(x, first, last):
        if x.dim() == 1:
            return x.double()
        return x[torch.arange(first, last, device=x.device) // case["group"]].double()

    h_all, n_all = [], []
    step = max(1, (1 << 25) // case["width"])
    for first in range(0, case["rows"], step):
        last = min(first + step, case["rows"])
        y = norm(s["branch"][first:last].double(), case["post"], s["post_weight"], s["post_bias"])
        y = y * rows(s["gate"], first, last) if s["gate"] is not None else y
        h = s["residual"][first:last].double() + case["scale"] * y
        n = norm(h, case["pre"], s["pre_weight"], None)
        if s["mod_scale"] is not None:
            n = n + n * rows(s["mod_scale"], first, last) + rows(s["mod_shift"], first, last)
        h_all.append(h)
        n_all.append(n)
    return {"residual": torch.cat(h_all), "out": torch.cat(n_all)}


def exact_logprobs(case, s):
    parts = {"logprob": [], "entropy": [], "top_logprobs": []}
    for x, token in zip(s["logits"].split(64), s["tokens"].split(64)):
        lp = torch.log_softmax(x.double(), -1)
        parts["logprob"].append(torch.where(token < 0, 0.0, lp.gather(1, token.clamp_min(0)[:, None])[:, 0]))
        parts["entropy"].append(torch.special.entr(lp.exp()).sum(1))
        parts["top_logprobs"].append(lp.topk(max(1, case["top"]), 1).values)
    out = {n: torch.cat(v) for n, v in parts.items()}
    out["rank"] = None
    if case["top"]:
        out["top_ids"] = None
    else:
        del out["top_logprobs"]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": exact_rope, "rows": exact_rope, "norms": exact_norms, "logprobs": exact_logprobs}[case["op"]](case, s)
