"""The transformer operators on device tensors, as cases that can be timed and checked.

A case is one pass through one operator as a program around image or video tokens calls
it: the rotation of queries and keys by their positions on several axes, attention over
sequences (capped, with a distance bias, causal or with a prefix, packed or padded), and
the residual join with its gate, its scale and the norms before and after.

  listed()            the named cases
  draw(rng)           one more case of the same ranges
  prepare(case, seed) the tensors and the workspace that a program holds before the call
  run(state)          one pass: with `own` through the framework's entry points, without
                      it in elementary torch operations in 32 bits (angles in 64)
  work(case)          bytes and flops that a pass cannot do without
  exact(case, seed)   the result in 64 bits, from the operators' definitions
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5


def _hat():
    folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hat-rs_amd")
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import hat_amd
    return hat_amd


def listed():
    return [
        # one 16 x 16 window of the smallest network (six heads of 24): launch and latency
        dict(name="rotary_window_f32", op="rotary", type="f32", batch=1, grid="16x16", q_heads=6, k_heads=6, dim=24,
             sections="6,6", pairs="halves", joint=False, inverse=False),
        # two images of 64 x 64 tokens, shared key heads, the direction of the gradient
        dict(name="rotary_image_bf16", op="rotary", type="bf16", batch=2, grid="64x64", q_heads=16, k_heads=4, dim=128,
             sections="32,32", pairs="neighbours", joint=True, inverse=True),
        # sixteen frames of 45 x 80 tokens; the last eight dims of each head stay as they are
        dict(name="rotary_video_f16", op="rotary", type="f16", batch=1, grid="16x45x80", q_heads=12, k_heads=12, dim=72,
             sections="8,12,12", pairs="halves", joint=False, inverse=False),
        # a block's join on a 64 x 64 plane of the smallest network: one gate for the
        # plane, the CAB's scale, the next LayerNorm
        dict(name="norm_plane_f32", op="norm", type="f32", rows=4096, width=144, post="none", pre="layer", gates=1,
             scale=0.01),
        # the join of a few tokens of a wide model, a norm on either side: latency
        dict(name="norm_tokens_bf16", op="norm", type="bf16", rows=3, width=4096, post="rms", pre="rms", gates=0,
             scale=1.0),
        # a video's tokens with one gate a frame, the block's output normed and scaled
        dict(name="norm_video_bf16", op="norm", type="bf16", rows=57600, width=1536, post="rms", pre="layer", gates=16,
             scale=0.5),
        # the windows of a 256 x 256 plane, a bias by distance in the window, fp32
        dict(name="attn_windows_f32", op="attention", type="f32", batch=256, q_len=256, k_len=256, q_heads=6, kv_heads=6,
             dim=24, mask="full", cap=0.0, bias="grid", docs=0, ragged=0),
        # one query of one sequence against a short cache: latency
        dict(name="attn_one_query_f16", op="attention", type="f16", batch=1, q_len=1, k_len=1023, q_heads=8, kv_heads=2,
             dim=64, mask="full", cap=0.0, bias="none", docs=0, ragged=0),
        # one token each of sixteen sequences against padded caches of their own lengths
        dict(name="attn_tokens_bf16", op="attention", type="bf16", batch=16, q_len=1, k_len=16384, q_heads=32, kv_heads=8,
             dim=128, mask="causal", cap=30.0, bias="none", docs=0, ragged=5),
        # documents packed behind one another, causal, capped
        dict(name="attn_docs_bf16", op="attention", type="bf16", batch=1, q_len=8192, k_len=8192, q_heads=16, kv_heads=4,
             dim=128, mask="causal", cap=50.0, bias="none", docs=11, ragged=7),
        # two sequences with a prefix that sees itself whole, a bias by distance, odd length
        dict(name="attn_prefix_f16", op="attention", type="f16", batch=2, q_len=4099, k_len=4099, q_heads=12, kv_heads=12,
             dim=64, mask="prefix", cap=0.0, bias="index", docs=0, ragged=0),
        # all tokens of a 128 x 128 plane among themselves: the matrix cores
        dict(name="attn_image_bf16", op="attention", type="bf16", batch=1, q_len=16384, k_len=16384, q_heads=8, kv_heads=8,
             dim=128, mask="full", cap=0.0, bias="none", docs=0, ragged=0),
    ]


def _between(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "attention", "attention"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "rotary":
        axes = rng.choice([1, 2, 3])
        sides = [_between(rng, 1, 24)] * (axes == 3) + [_between(rng, 4, 64) for _ in range(min(axes, 2))]
        sections = [rng.randint(1, 48 // axes) for _ in range(axes)]
        dim = 2 * sum(sections) + rng.choice([0, 0, 1, 8])
        heads = rng.choice([1, 2, 4])
        return dict(op=op, type=kind, batch=rng.choice([1, 2, 3]), grid="x".join(map(str, sides)),
                    q_heads=heads * rng.choice([1, 2, 4]), k_heads=heads, dim=dim, sections=",".join(map(str, sections)),
                    pairs=rng.choice(["halves", "neighbours"]), joint=rng.random() < 0.5, inverse=rng.random() < 0.3)
    if op == "norm":
        width = _between(rng, 17, 8192)
        rows = _between(rng, 1, max(2, 60_000_000 // width // 4))
        gates = rng.choice([0, 1, rows] + [g for g in range(2, 17) if rows % g == 0])
        return dict(op=op, type=kind, rows=rows, width=width, post=rng.choice(["none", "layer", "rms"]),
                    pre=rng.choice(["layer", "rms"]), gates=gates, scale=rng.choice([1.0, 0.5, 0.01]))
    heads = rng.choice([1, 2, 4])
    case = dict(op=op, type=kind, q_heads=heads * rng.choice([1, 2, 3, 8]), kv_heads=heads,
                dim=rng.choice([24, 30, 33, 64, 72, 80, 96, 128]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]))
    if rng.random() < 0.4:  # a few queries against a long cache
        return dict(case, batch=rng.randint(1, 12), q_len=rng.choice([1, 1, 1, 2, 5]), k_len=_between(rng, 1, 16384),
                    mask=rng.choice(["full", "causal"]), bias=rng.choice(["none", "index"]), docs=0,
                    ragged=rng.randint(0, 99))
    if rng.random() < 0.4:  # packed documents
        tokens = _between(rng, 40, 4096)
        return dict(case, batch=1, q_len=tokens, k_len=tokens, mask=rng.choice(["full", "causal"]),
                    bias=rng.choice(["none", "index", "grid"]), docs=rng.randint(1, 12), ragged=rng.randint(1, 99))
    q_len = _between(rng, 7, 3000)
    mask = rng.choice(["full", "causal", "prefix"])
    return dict(case, batch=rng.randint(1, 3), q_len=q_len, k_len=max(1, q_len + rng.choice([0, 0, -5, 70])), mask=mask,
                bias=rng.choice(["none", "index", "grid"]), docs=0, ragged=0)


# ---- inputs --------------------------------------------------------------------------


def _normal(gen, kind, *shape, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * std).to(TYPES[kind])


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _doc_ends(case):
    """The offsets of a packed case's documents: lengths of a wide spread, some empty or one."""
    rng = random.Random(case["ragged"])
    weights = [rng.random() ** 3 for _ in range(case["docs"])]
    cuts = [0]
    for w in weights[:-1]:
        cuts.append(min(case["q_len"], cuts[-1] + int(case["q_len"] * w / sum(weights))))
    return cuts + [case["q_len"]]


def _cache_lengths(case):
    """The lengths in use of a padded case's caches."""
    rng = random.Random(1000 + case["ragged"])
    return [rng.randint(1 + case["k_len"] // 2, case["k_len"]) if case["k_len"] > 1 else 1
            for _ in range(case["batch"])]


def _padded(case):
    return case["ragged"] > 0 and case["docs"] == 0


def _grid(case):
    return [int(s) for s in case["grid"].split("x")]


def _grid_positions(sides, repeat=1):
    axes = torch.meshgrid(*[torch.arange(s, device="cuda", dtype=torch.int32) for s in sides], indexing="ij")
    return torch.stack([a.reshape(-1) for a in axes], dim=1).repeat(repeat, 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["type"]
    state = dict(case=case)
    if case["op"] == "rotary":
        sides = _grid(case)
        tokens = math.prod(sides)
        state["q"] = _normal(gen, kind, case["batch"], tokens, case["q_heads"], case["dim"])
        state["k"] = _normal(gen, kind, case["batch"], tokens, case["k_heads"], case["dim"])
        # a crop of a larger plane or a later part of a film: an offset per axis
        off = torch.randint(0, 2000, (len(sides),), generator=gen, device="cuda", dtype=torch.int32)
        state["pos"] = _grid_positions(sides) + off
        state["sections"] = [int(s) for s in case["sections"].split(",")]
        state["outs"] = torch.empty_like(state["q"]), torch.empty_like(state["k"])
        return state
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        state["x"] = _normal(gen, kind, rows, width, std=3.0) + _normal(gen, kind, 1, width)
        state["y"] = _normal(gen, kind, rows, width, std=2.0)
        state["gate"] = torch.sigmoid(_normal(gen, kind, case["gates"], width)) if case["gates"] else None
        for side in ("post", "pre"):
            state[side + "_w"] = 1 + _normal(gen, "f32", width, std=0.2)
            state[side + "_b"] = _normal(gen, "f32", width, std=0.2) if case[side] == "layer" else None
        state["outs"] = torch.empty_like(state["x"]), torch.empty_like(state["x"])
        return state
    lead = lambda n: (case["batch"], n) if not case["docs"] else (n,)  # noqa: E731
    # scores of a trained spread: a few units
    state["q"] = _normal(gen, kind, *lead(case["q_len"]), case["q_heads"], case["dim"], std=1.6)
    state["k"] = _normal(gen, kind, *lead(case["k_len"]), case["kv_heads"], case["dim"], std=1.2)
    state["v"] = _normal(gen, kind, *lead(case["k_len"]), case["kv_heads"], case["dim"])
    more = dict(causal=case["mask"] != "full", cap=case["cap"])
    if case["docs"]:
        more["cu_q"] = more["cu_k"] = _ints(_doc_ends(case))
    if _padded(case):
        more["k_lens"] = _ints(_cache_lengths(case))
    if case["mask"] == "prefix":
        more["prefix"] = torch.randint(0, case["k_len"] + 1, (case["batch"],), generator=gen, device="cuda",
                                       dtype=torch.int32)
    if case["bias"] != "none":
        more["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["q_heads"] + 1, device="cuda") / case["q_heads"])
    if case["bias"] == "grid":
        side = math.isqrt(case["q_len"] - 1) + 1  # the tokens in rows of a square plane
        at = torch.arange(max(case["q_len"], case["k_len"]), device="cuda", dtype=torch.int32)
        pos = torch.stack([at // side, at % side], dim=1).contiguous()
        more["pos_q"], more["pos_k"] = pos[: case["q_len"]], pos[: case["k_len"]]
    state["more"] = more
    state["out"] = torch.empty_like(state["q"])
    state["workspace"] = None
    if own:
        hat = _hat()
        need = hat.attention_workspace(state["q"], state["k"], state["v"], state["out"], **more)
        state["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
    return state


# ---- one pass ------------------------------------------------------------------------


def run(state):
    case = state["case"]
    if own:
        hat = _hat()
        if case["op"] == "rotary":
            q, k = state["outs"]
            hat.op_rotary(state["q"], state["k"], state["pos"], state["sections"], pairs=case["pairs"],
                          joint=case["joint"], inverse=case["inverse"], q_out=q, k_out=k)
            return q, k
        if case["op"] == "norm":
            x, h = state["outs"]
            hat.op_residual_norm(state["x"], state["y"], x, h, gate=state["gate"], scale=case["scale"], post=case["post"],
                                 post_weight=state["post_w"] if case["post"] != "none" else None,
                                 post_bias=state["post_b"], pre=case["pre"], pre_weight=state["pre_w"],
                                 pre_bias=state["pre_b"], eps=EPS)
            return x, h
        hat.op_attention(state["q"], state["k"], state["v"], state["out"], workspace=state["workspace"], **state["more"])
        return state["out"]
    if case["op"] == "rotary":
        cos, sin = _angles(state)
        return _rotate(case, state["q"], cos, sin), _rotate(case, state["k"], cos, sin)
    if case["op"] == "norm":
        return _join(state)
    return _attend(state)


def _angles(state):
    """cos and sin [tokens, 1, pairs] of each token's angles."""
    case = state["case"]
    sections = torch.tensor(state["sections"], device="cuda")
    n = sum(state["sections"])
    axis = torch.repeat_interleave(torch.arange(len(state["sections"]), device="cuda"), sections, output_size=n)
    step = torch.arange(n, device="cuda", dtype=torch.float64)
    if case["joint"]:
        ladder = step / n
    else:
        ladder = (step - (torch.cumsum(sections, 0) - sections)[axis]) / sections[axis]
    angle = state["pos"][:, axis].double() * torch.pow(10000.0, -ladder)
    if case["inverse"]:
        angle = -angle
    return torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]


def _rotate(case, x, cos, sin):
    n = cos.shape[-1]
    turned, rest = x[..., : 2 * n].float(), x[..., 2 * n:]
    if case["pairs"] == "halves":
        a, b = turned[..., :n], turned[..., n:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned.to(x.dtype), rest], dim=-1)


def _normed(x, kind, w, b):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(dim=-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w
    return x if b is None else x + b


def _join(state):
    case = state["case"]
    y = _normed(state["y"].float(), case["post"], state["post_w"], state["post_b"])
    if case["gates"]:
        g = state["gate"].float()
        y = (y.reshape(g.shape[0], -1, g.shape[1]) * g[:, None]).reshape(y.shape)
    x = state["x"].float() + case["scale"] * y
    h = _normed(x, case["pre"], state["pre_w"], state["pre_b"])
    return x.to(state["x"].dtype), h.to(state["x"].dtype)


def _attend(state):
    case, more = state["case"], state["more"]
    lq, lk, hk, d = case["q_len"], case["k_len"], case["kv_heads"], case["dim"]
    group = case["q_heads"] // hk
    # [batch, key head, group, token, dim]
    q = state["q"].float().reshape(-1, lq, hk, group, d).permute(0, 2, 3, 1, 4)
    k = state["k"].float().reshape(-1, lk, hk, d).permute(0, 2, 1, 3)
    v = state["v"].float().reshape(-1, lk, hk, d).permute(0, 2, 1, 3)
    n = q.shape[0]
    i = torch.arange(lq, device="cuda")[None, :, None]
    j = torch.arange(lk, device="cuda")[None, None, :]
    used_q, used_k, first_q, first_k = lq, lk, 0, 0
    seen = torch.ones((n, lq, lk), dtype=torch.bool, device="cuda")
    if case["docs"]:  # the document of each token and where it starts
        cu = more["cu_q"].long()
        doc = torch.searchsorted(cu[1:].contiguous(), torch.arange(lq, device="cuda"), right=True)
        seen &= doc[None, :, None] == doc[None, None, :]
    elif _padded(case):
        used_k = more["k_lens"].long()[:, None, None]
        seen &= j < used_k
    # within one document the offsets of both sides cancel
    row = i - first_q + used_k - used_q
    if case["mask"] != "full":
        earlier = (j - first_k) <= row
        if case["mask"] == "prefix":
            earlier = earlier | (j < more["prefix"].long()[:, None, None])
        seen = seen & earlier
    s = torch.matmul(q.reshape(n, hk, group * lq, d), k.transpose(2, 3).contiguous()).reshape(n, hk, group, lq, lk)
    s = s * (1.0 / math.sqrt(d))
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    if case["bias"] != "none":
        if case["bias"] == "grid":
            far = (more["pos_q"].float()[:, None] - more["pos_k"].float()[None]).abs().sum(dim=-1)[None]
        else:
            far = (row - j).abs().float()
        s = s - more["slopes"].reshape(1, hk, group, 1, 1) * far[:, None, None]
    seen = seen[:, None, None]
    s = torch.where(seen, s, -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(s - top)
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.reshape(n, hk, group * lq, lk), v).reshape(n, hk, group, lq, d)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(state["q"].shape).to(state["q"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------


def _seen_pairs(case):
    """Query and key pairs that the mask leaves (of one head), and the keys read."""
    def below(lq, lk):  # the causal pairs of one sequence
        first = max(0, lq - lk)
        n = lq - first
        return n * (lk - lq + first) + n * (n + 1) // 2
    if case["docs"]:
        ends = _doc_ends(case)
        lens = [b - a for a, b in zip(ends, ends[1:])]
        pairs = sum(below(n, n) if case["mask"] == "causal" else n * n for n in lens)
        return pairs, case["k_len"]
    lens = _cache_lengths(case) if _padded(case) else [case["k_len"]] * case["batch"]
    # a prefix of unknown length adds up to as many pairs again: the causal ones are certain
    return sum(case["q_len"] * n if case["mask"] == "full" else below(case["q_len"], n) for n in lens), sum(lens)


def work(case):
    size = BYTES[case["type"]]
    if case["op"] == "rotary":
        tokens = math.prod(_grid(case))
        values = case["batch"] * tokens * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return dict(bytes=2 * values * size + 4 * tokens * len(_grid(case)), flops=3 * values)
    if case["op"] == "norm":
        values = case["rows"] * case["width"]
        return dict(bytes=4 * values * size + case["gates"] * case["width"] * size + 16 * case["width"], flops=16 * values)
    pairs, keys = _seen_pairs(case)
    values = 2 * case["batch"] * case["q_len"] * case["q_heads"] * case["dim"] + 2 * keys * case["kv_heads"] * case["dim"]
    return dict(bytes=values * size, flops=4 * pairs * case["q_heads"] * case["dim"])


# ---- the result in 64 bits -----------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return dict(rotary=_exact_rotary, norm=_exact_norm, attention=_exact_attention)[case["op"]](case, state)


def _exact_rotary(case, state):
    """Each pair as a complex number times e^(i angle)."""
    columns = []
    total = sum(state["sections"])
    for axis, count in enumerate(state["sections"]):
        for i in range(count):
            exponent = len(columns) / total if case["joint"] else i / count
            columns.append(state["pos"][:, axis].double() / 10000.0 ** exponent)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.stack(columns, dim=1))
    turn = (turn.conj() if case["inverse"] else turn)[None, :, None, :]
    outs = []
    for x in (state["q"], state["k"]):
        y = x.double().clone()
        if case["pairs"] == "halves":
            first, second = slice(0, total), slice(total, 2 * total)
        else:
            first, second = slice(0, 2 * total, 2), slice(1, 2 * total, 2)
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        outs.append(y)
    return tuple(outs)


def _exact_norm(case, state):
    def norm(v, kind, w, b):
        if kind == "none":
            return v
        mean = v.mean(1, True) if kind == "layer" else 0.0
        power = v.var(1, unbiased=False, keepdim=True) if kind == "layer" else v.pow(2).mean(1, True)
        out = (v - mean) * (power + EPS).rsqrt() * w.double()
        return out + b.double() if b is not None else out
    add = norm(state["y"].double(), case["post"], state["post_w"], state["post_b"])
    if case["gates"]:
        add = add * state["gate"].double().repeat_interleave(case["rows"] // case["gates"], dim=0)
    x = state["x"].double() + case["scale"] * add
    return x, norm(x, case["pre"], state["pre_w"], state["pre_b"])


def _exact_attention(case, state):
    """Sequence by sequence, head by head."""
    more = state["more"]
    q, k, v = (state[n] for n in ("q", "k", "v"))
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    if case["docs"]:
        ends = _doc_ends(case)
        parts = [(out[a:b], q[a:b], k[a:b], v[a:b], a) for a, b in zip(ends, ends[1:])]
    else:
        lens = _cache_lengths(case) if _padded(case) else [case["k_len"]] * case["batch"]
        parts = [(out[b], q[b], k[b, :n], v[b, :n], 0) for b, n in enumerate(lens)]
    for number, (to, qs, ks, vs, start) in enumerate(parts):
        lq, lk = qs.shape[0], ks.shape[0]
        if lq == 0 or lk == 0:
            continue
        at_q = torch.arange(lk - lq, lk, device="cuda")
        at_k = torch.arange(lk, device="cuda")
        hidden = torch.zeros((lq, lk), dtype=torch.bool, device="cuda")
        if more["causal"]:
            hidden = at_k[None] > at_q[:, None]
            if "prefix" in more:
                hidden[:, : int(more["prefix"][number])] = False
        if "pos_q" in more:
            pq, pk = more["pos_q"][start:start + lq].double(), more["pos_k"][start:start + lk].double()
            distance = torch.cdist(pq, pk, p=1.0)
        else:
            distance = (at_q[:, None] - at_k[None]).abs().double()
        for h in range(case["q_heads"]):
            g = h // (case["q_heads"] // case["kv_heads"])
            s = qs[:, h].double() @ ks[:, g].double().t().contiguous() / math.sqrt(case["dim"])
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if "slopes" in more:
                s -= more["slopes"][h].double() * distance
            s.masked_fill_(hidden, -math.inf)
            p = torch.softmax(s, dim=1)
            p.masked_fill_(hidden, 0.0)  # a row that sees nothing adds nothing
            to[:, h] = p @ vs[:, g].double()
    return out
