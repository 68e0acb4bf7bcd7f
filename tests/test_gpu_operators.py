"""The operators on device tensors (hat_op_rotary, hat_op_attention,
hat_op_residual_norm) against their formulas in 64 bits.

Tolerances. A value stored in type t is off by half a step, U[t] = finfo(t).eps / 2, of
itself. Beside that, with u = 2^-24 (an fp32 rounding):
- rotary: cos and sin from an angle rounded to fp32 (in revolutions, so up to pi u) and
  the function itself (2 u), then two products and a sum (3 u): below 9 u of |a| + |b|.
- norms: sums of n values in fp32 are off by at most (n / threads + 10) u of the sum of
  magnitudes: with at most 32 values a thread 42 u; a mean and a square root of a mean
  then a product and a sum each: below 160 u of (|w| (1 + |z|) + |b|), z the normed value,
  times what the mean's error makes of the spread (the inputs' mean is below their
  spread here), and the same again through the second norm, whose input carries the first's.
- attention: a score is off by (D + 8) u of scale * sum |q_d k_d| + the bias's size (with a
  cap: 2^-21 of the cap from the fast tanh in the 16-bit types), which changes a probability by that much of itself
  and the output by at most twice that of sum p |v|; the sums over keys add (n / 16 + 16) u; in
  the 16-bit types the probabilities are rounded to the type before the product with v:
  U of sum p |v|, and in fp16 2^-25 of each at least (probabilities below 2^-14 of the
  largest are subnormal).
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
u = 2.0 ** -24


def U(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else u


@pytest.fixture(scope="module")
def hl():
    import hat_amd
    assert hat_amd.gpu_available(), "the HIP runtime or the GPU is missing"
    return hat_amd


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(gen, t, *shape, std=1.0):
    return (torch.randn(shape, generator=gen) * std).to(t)


def _strided(x, kind):
    """x on the device with other strides: packed behind gaps, or heads before tokens."""
    if kind == "plain":
        return x.cuda()
    if kind == "gaps":
        wide = torch.full((*x.shape[:-2], x.shape[-2] + 1, x.shape[-1] + 8), 7.0, dtype=x.dtype, device="cuda")
        view = wide[..., : x.shape[-2], : x.shape[-1]]
    elif kind == "odd":  # rows at odd element offsets
        wide = torch.full((*x.shape[:-1], x.shape[-1] + 1), 7.0, dtype=x.dtype, device="cuda")
        view = wide[..., 1:]
    else:  # heads first
        view = torch.empty_like(x.transpose(-3, -2).contiguous(), device="cuda").transpose(-3, -2)
    view.copy_(x)
    return view


# ---- rotary ------------------------------------------------------------------------


def _rotary_want(x, pos, sections, pairs, joint, inverse, base=10000.0):
    S = sum(sections)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    inner = [i for n in sections for i in range(n)]
    ladder = [n / S if joint else inner[n] / sections[axis[n]] for n in range(S)]
    freq = torch.tensor([base ** -e for e in ladder], dtype=torch.float64)
    angle = pos.double()[..., axis] * freq
    if inverse:
        angle = -angle
    if angle.dim() == 2:
        angle = angle[None]
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    y = x.double().clone()
    one, two = (slice(0, S), slice(S, 2 * S)) if pairs == "halves" else (slice(0, 2 * S, 2), slice(1, 2 * S, 2))
    a, b = x.double()[..., one], x.double()[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(y)
    size[..., one] = size[..., two] = a.abs() + b.abs()
    return y, size


ROTARY = [
    # batch, tokens, q heads, k heads, dim, sections, pairs, joint, inverse, stride
    (1, 1, 1, 1, 2, [1], "halves", False, False, "plain"),
    (1, 256, 6, 6, 24, [6, 6], "halves", False, False, "plain"),
    (1, 77, 6, 6, 30, [7, 8], "halves", True, False, "plain"),
    (2, 33, 8, 2, 128, [16, 24, 24], "neighbours", False, True, "plain"),
    (2, 19, 4, 4, 72, [8, 12, 12], "halves", False, False, "gaps"),
    (3, 11, 3, 1, 80, [0, 20, 8], "neighbours", True, False, "heads"),
    (1, 50, 5, 5, 33, [3, 4, 4, 4], "neighbours", False, False, "odd"),
    (1, 50, 5, 5, 33, [3, 4, 4, 4], "halves", True, True, "odd"),
    (1, 9, 2, 2, 256, [128], "halves", False, False, "plain"),
    (1, 2, 300, 2, 64, [16, 16], "neighbours", False, False, "plain"),
    (1, 5000, 1, 1, 8, [4], "halves", False, False, "plain"),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("case", ROTARY, ids=lambda c: f"{c[0]}x{c[1]}x{c[2]}x{c[4]}-{c[6]}-{c[9]}")
def test_rotary(hl, kind, case):
    B, T, hq, hk, D, sections, pairs, joint, inverse, stride = case
    t, g = TYPES[kind], _gen(T * D)
    print(f"rotary {kind} {case}", flush=True)
    q, k = _randn(g, t, B, T, hq, D), _randn(g, t, B, T, hk, D)
    pos = torch.randint(-3000, 5000, (T, len(sections)), generator=g, dtype=torch.int32)
    pos[-1] = 1 << 30  # far: an angle in fp32 would be anything
    qd, kd = _strided(q, stride), _strided(k, stride)
    qo, ko = torch.full_like(qd, 9.0), torch.full_like(kd, 9.0)
    hl.op_rotary(qd, kd, pos.cuda(), sections, pairs=pairs, joint=joint, inverse=inverse, q_out=qo, k_out=ko)
    torch.cuda.synchronize()
    for x, got in ((q, qo), (k, ko)):
        want, size = _rotary_want(x, pos, sections, pairs, joint, inverse)
        # the frequency's own rounding in 64 bits: 2^-52 of 2^30 radians
        tol = U(t) * want.abs() * 1.01 + (9 * u + 2.0 ** -21) * size
        assert ((got.cpu().double() - want).abs() <= tol).all(), ((got.cpu().double() - want).abs() / tol.clamp_min(1e-30)).max()
        S2 = 2 * sum(sections)
        assert torch.equal(got.cpu()[..., S2:], x[..., S2:])
    # in place: the same bits, the dims behind the rotated ones left alone
    hl.op_rotary(qd, kd, pos.cuda(), sections, pairs=pairs, joint=joint, inverse=inverse)
    torch.cuda.synchronize()
    assert torch.equal(qd, qo) and torch.equal(kd, ko)


def test_rotary_inverse_undoes_and_is_the_gradient(hl):
    """R is linear and orthogonal: R^-1 R x = x, and <w, R x> has the gradient R^-1 w."""
    g = _gen(5)
    x, w = _randn(g, torch.float32, 1, 40, 3, 48), _randn(g, torch.float32, 1, 40, 3, 48)
    pos = torch.randint(0, 500, (1, 40, 2), generator=g, dtype=torch.int32).cuda()
    xd, wd = x.cuda(), w.cuda()
    y, gx = torch.empty_like(xd), torch.empty_like(xd)
    hl.op_rotary(xd, None, pos, [12, 8], q_out=y)
    hl.op_rotary(wd, None, pos, [12, 8], inverse=True, q_out=gx)
    back = torch.empty_like(xd)
    hl.op_rotary(y, None, pos, [12, 8], inverse=True, q_out=back)
    torch.cuda.synchronize()
    assert (back.cpu() - x).abs().max() <= 2 * 11 * u * 2 * x.abs().max()
    # differences: the map is linear, so a step of any size serves; entry (token 7, head 1, dim d)
    for d in (0, 13, 45):
        e = torch.zeros_like(xd)
        e[0, 7, 1, d] = 1.0
        re = torch.empty_like(xd)
        hl.op_rotary(e, None, pos, [12, 8], q_out=re)
        torch.cuda.synchronize()
        by_difference = float((re.double() * wd.double()).sum())
        assert abs(by_difference - float(gx[0, 7, 1, d])) <= 2 * 12 * u * 2 * float(w.abs().max())


def test_rotary_far_positions_and_no_tokens(hl):
    x = torch.ones(1, 2, 1, 4)
    pos = torch.tensor([[2 ** 31 - 1], [-(2 ** 31)]], dtype=torch.int32)
    y = torch.empty_like(x, device="cuda")
    hl.op_rotary(x.cuda(), None, pos.cuda(), [2], base=3.0, q_out=y)
    torch.cuda.synchronize()
    want, size = _rotary_want(x, pos, [2], "halves", False, False, base=3.0)
    # 2^31 radians known to 2^-53 of themselves on both sides: 2^-21
    assert ((y.cpu().double() - want).abs() <= (9 * u + 2.0 ** -20) * size).all()
    empty = torch.empty(1, 0, 1, 4, device="cuda")
    hl.op_rotary(empty, None, torch.empty(0, 1, dtype=torch.int32, device="cuda"), [2])


# ---- the residual join -----------------------------------------------------------------


def _normed(v, kind, w, b, eps):
    if kind == "none":
        return v, 0.0, v.abs()
    z = v - v.mean(1, keepdim=True) if kind == "layer" else v
    z = z / torch.sqrt((z * z).mean(1, keepdim=True) + eps)
    w = torch.ones(v.shape[1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(v.shape[1], dtype=torch.float64) if b is None else b.double()
    return z * w + b, w.abs() * (1 + z.abs()) + b.abs(), z


NORMS = [
    # rows, width, post, pre, gates, weights, layout
    (1, 1, "none", "rms", 0, "both", "plain"),
    (5, 17, "layer", "layer", 1, "both", "plain"),
    (300, 144, "none", "layer", 1, "both", "plain"),
    (33, 180, "rms", "layer", 33, "weight", "plain"),
    (18, 192, "layer", "rms", 9, "none", "plain"),
    (7, 256, "rms", "rms", 0, "both", "gaps"),
    (70, 264, "rms", "none", 2, "weight", "plain"),
    (9, 1000, "layer", "layer", 3, "both", "odd"),
    (4, 1024, "none", "none", 1, "none", "plain"),
    (6, 1500, "rms", "layer", 6, "both", "odd"),
    (5, 2048, "layer", "rms", 5, "both", "plain"),
    (3, 4096, "rms", "rms", 0, "both", "plain"),
    (2, 5000, "rms", "layer", 1, "both", "gaps"),
    (2, 8192, "layer", "rms", 0, "weight", "plain"),
    (2, 16384, "layer", "layer", 1, "both", "plain"),
    (2, 16383, "rms", "rms", 2, "both", "plain"),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("case", NORMS, ids=lambda c: "-".join(map(str, c)))
def test_residual_norm(hl, kind, case):
    rows, width, post, pre, gates, weights, layout = case
    t, g, eps, scale = TYPES[kind], _gen(rows * width), 1e-5, 0.375
    print(f"residual_norm {kind} {case}", flush=True)
    x, y = _randn(g, t, rows, width, std=2.0) + 0.5, _randn(g, t, rows, width)
    gate = torch.sigmoid(_randn(g, t, gates, width).float()).to(t) if gates else None
    vec = lambda on: _randn(g, torch.float32, width, std=0.5) + 1.0 if on else None  # noqa: E731
    pw, pb = (vec(weights != "none"), vec(weights == "both")) if post != "none" else (None, None)
    nw, nb = (vec(weights != "none"), vec(weights == "both")) if pre != "none" else (None, None)

    def dev(v):
        if v is None or v.dim() == 1 or layout == "plain":
            return None if v is None else v.cuda()
        wide = torch.full((v.shape[0], v.shape[1] + (8 if layout == "gaps" else 1)), 5.0, dtype=v.dtype, device="cuda")
        view = wide[:, : v.shape[1]] if layout == "gaps" else wide[:, 1:]
        view.copy_(v)
        return view

    xd, yd = dev(x), dev(y)
    xo, h = torch.full_like(xd, 3.0), torch.full_like(xd, 3.0)
    kw = dict(gate=dev(gate), scale=scale, post=post, post_weight=dev(pw), post_bias=dev(pb), pre=pre,
              pre_weight=dev(nw), pre_bias=dev(nb), eps=eps)
    hl.op_residual_norm(xd, yd, xo, h, **kw)
    torch.cuda.synchronize()
    add, size, _ = _normed(y.double(), post, pw, pb, eps)
    gd = gate.double().repeat_interleave(rows // gates, 0) if gates else torch.ones(1, 1, dtype=torch.float64)
    want = x.double() + scale * gd * add
    err = 160 * u * scale * gd * size + 4 * u * (x.double().abs() + (scale * gd * add).abs())
    assert ((xo.cpu().double() - want).abs() <= err + U(t) * (want.abs() + err)).all()
    hw, hsize, z = _normed(want, pre, nw, nb, eps)
    if pre == "none":
        herr = err
    else:
        # an error e of x' moves z by at most (|e| + the row's rms of e (1 + |z|)) / spread
        c = want - want.mean(1, keepdim=True) if pre == "layer" else want
        spread = torch.sqrt((c * c).mean(1, keepdim=True) + eps)
        e = err + torch.zeros_like(want)
        w = torch.ones(width, dtype=torch.float64) if nw is None else nw.double().abs()
        herr = 160 * u * hsize + w * (e + 2 * (e * e).mean(1, keepdim=True).sqrt() * (1 + z.abs())) / spread
    assert ((h.cpu().double() - hw).abs() <= herr + U(t) * (hw.abs() + herr)).all()
    # either output alone, and in place of the inputs: the same bits
    only = torch.empty_like(xd)
    hl.op_residual_norm(xd, yd, None, only, **kw)
    assert torch.equal(only, h)
    hl.op_residual_norm(xd, yd, xd, yd, **kw)
    torch.cuda.synchronize()
    assert torch.equal(xd, xo) and torch.equal(yd, h)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("width", [16, 130, 264, 600, 1001, 1030, 1536, 2047, 4100, 6000, 9000, 9002])
def test_residual_norm_every_combination(hl, kind, width):
    """Each norm before with each norm behind, with and without a gate and weights, for
    every number of threads a row and vectors a thread."""
    t, g, rows = TYPES[kind], _gen(width), 6
    print(f"residual_norm {kind} {width}", flush=True)
    x, y = _randn(g, t, rows, width, std=2.0).cuda(), _randn(g, t, rows, width).cuda()
    gate = torch.sigmoid(_randn(g, t, 2, width).float()).to(t).cuda()
    w, b = (_randn(g, torch.float32, width, std=0.5).cuda() + 1.0 for _ in range(2))
    for post in ("none", "layer", "rms"):
        for pre in ("none", "layer", "rms"):
            for gated in (False, True):
                for weights in ((None, None), (w, None), (w, b)):
                    xo, h = torch.full_like(x, 3.0), torch.full_like(x, 3.0)
                    pw, pb = weights if post != "none" else (None, None)
                    nw, nb = weights if pre != "none" else (None, None)
                    hl.op_residual_norm(x, y, xo, h, gate=gate if gated else None, scale=0.375, post=post,
                                        post_weight=pw, post_bias=pb, pre=pre, pre_weight=nw, pre_bias=nb)
                    def norm(v, kind, w, b):
                        v = v - v.mean(1, keepdim=True) if kind == "layer" else v
                        v = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5) if kind != "none" else v
                        v = v * w.double() if w is not None else v
                        return v + b.double() if b is not None else v
                    add = norm(y.double(), post, pw, pb) * (gate.double().repeat_interleave(3, 0) if gated else 1.0)
                    want = x.double() + 0.375 * add
                    # values of up to ten units and sums in fp32 (see above): 400 u of ten
                    for got, true in ((xo, want), (h, norm(want, pre, nw, nb))):
                        off = (got.double() - true).abs() - U(t) * 1.01 * true.abs()
                        assert off.max() <= 4000 * u, (post, pre, gated, weights[0] is not None, weights[1] is not None)


def test_residual_norm_of_the_stream_alone(hl):
    """y left out: a norm of x, at the width the forward's own LayerNorm has."""
    g = _gen(3)
    x, w, b = _randn(g, torch.float32, 50, 144), _randn(g, torch.float32, 144), _randn(g, torch.float32, 144)
    h = torch.empty(50, 144, device="cuda")
    hl.op_residual_norm(x.cuda(), h=h, pre="layer", pre_weight=w.cuda(), pre_bias=b.cuda())
    want, size, _ = _normed(x.double(), "layer", w, b, 1e-5)
    torch.cuda.synchronize()
    assert ((h.cpu().double() - want).abs() <= 160 * u * size + u * want.abs()).all()


def test_residual_norm_rows_stay_apart(hl):
    """A row with NaN or infinities changes no other row; no rows is no work."""
    g = _gen(4)
    for width in (144, 1024, 4096):
        x, y = _randn(g, torch.bfloat16, 9, width).cuda(), _randn(g, torch.bfloat16, 9, width).cuda()
        clean, h = torch.empty_like(x), torch.empty_like(x)
        hl.op_residual_norm(x, y, None, clean, post="rms", pre="layer")
        x[4, 3], y[6, 1] = float("nan"), float("inf")
        hl.op_residual_norm(x, y, None, h, post="rms", pre="layer")
        torch.cuda.synchronize()
        good = [0, 1, 2, 3, 5, 7, 8]
        assert torch.equal(h[good], clean[good]) and h[4].isnan().all()
    empty = torch.empty(0, 144, device="cuda")
    hl.op_residual_norm(empty, None, None, empty, pre="rms")


# ---- attention -----------------------------------------------------------------------


def _attention_want(q, k, v, seqs, scale, causal, prefix, cap, slopes, pos_q, pos_k, sure):
    """(want, tolerance) for rows of q [n, hq, D], keys of k [m, hk, D]; seqs: (q rows, k
    rows) slices of each sequence; rows of no sequence are NaN. sure: the type's U."""
    D, hq, hk = q.shape[-1], q.shape[1], k.shape[1]
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    prefix, slopes, pos_q, pos_k = (None if x is None else x.cuda() for x in (prefix, slopes, pos_q, pos_k))
    want = torch.full(q.shape, math.nan, dtype=torch.float64, device="cuda")
    tol = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for n, (rq, rk) in enumerate(seqs):
        qs, ks, vs = q[rq].double(), k[rk].double(), v[rk].double()
        lq, lk = qs.shape[0], ks.shape[0]
        want[rq] = 0.0
        if lk == 0 or lq == 0:
            continue
        i, j = torch.arange(lq, device="cuda")[:, None] + lk - lq, torch.arange(lk, device="cuda")[None]
        hidden = torch.zeros(lq, lk, dtype=torch.bool, device="cuda")
        if causal:
            hidden = j > i
            if prefix is not None:
                hidden = hidden & (j >= int(prefix[n]))
        if pos_q is not None:
            far = (pos_q[rq].double()[:, None] - pos_k[rk].double()[None]).abs().sum(-1)
        else:
            far = (i - j).abs().double()
        for h in range(hq):
            kh = ks[:, h // (hq // hk)].masked_fill(~torch.isfinite(ks[:, h // (hq // hk)]), 0.0)
            vh = vs[:, h // (hq // hk)].masked_fill(~torch.isfinite(vs[:, h // (hq // hk)]), 0.0)
            s = scale * qs[:, h] @ kh.T
            size = abs(scale) * qs[:, h].abs() @ kh.abs().T
            err = (D + 8) * u * size
            if cap:
                s = cap * torch.tanh(s / cap)
                err = err + (2.0 ** -21 if sure > u else 6 * u) * cap
            if slopes is not None:
                s = s - slopes[h].double() * far
                err = err + 4 * u * (slopes[h].double() * far).abs()
            err = err + 4 * u * s.abs()
            s = s.masked_fill(hidden, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(hidden, 0.0, torch.exp(s - top.clamp_min(-1e300)))
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total.clamp_min(1e-300), 0.0)
            o = p @ vh
            want[rq, h] = o
            worst = torch.where(hidden, 0.0, err).amax(1, keepdim=True)
            size = p @ vh.abs()
            t = 2.2 * worst * size + (lk / 16 + 16) * u * size + 2.0 ** -100
            if sure > u:
                t = t + sure * size
            if sure == 2.0 ** -11:
                t = t + 2.0 ** -24 * lk * vh.abs().max()
            tol[rq, h] = t + sure * 1.01 * (o.abs() + t)
    return want.cpu(), tol.cpu()


def _check(hl, kind, q, k, v, seqs, stride="plain", scale=None, causal=False, prefix=None, cap=0.0, slopes=None,
           pos_q=None, pos_k=None, **layout):
    """One call against the formulas. q, k, v: [batch, token, head, dim] or packed."""
    D = q.shape[-1]
    qd, kd, vd = (_strided(x, stride) for x in (q, k, v))
    out = torch.full_like(qd, 77.0)
    dev = {n: (x.cuda() if x is not None else None) for n, x in
           dict(prefix=prefix, slopes=slopes, pos_q=pos_q, pos_k=pos_k, **layout).items()}
    need = hl.attention_workspace(qd, kd, vd, out, scale=scale, causal=causal, cap=cap, **dev)
    work = torch.full((need,), 255, dtype=torch.uint8, device="cuda") if need else None
    hl.op_attention(qd, kd, vd, out, scale=scale, causal=causal, cap=cap, workspace=work, **dev)
    torch.cuda.synchronize()
    flat = lambda x: x.reshape(-1, *x.shape[-2:])  # noqa: E731
    spread = lambda x, like: (None if x is None else x.reshape(-1, x.shape[-1]) if x.dim() == 3 else  # noqa: E731
                              x.repeat(like.shape[0], 1) if like.dim() == 4 else x)
    want, tol = _attention_want(flat(q), flat(k), flat(v), seqs, D ** -0.5 if scale is None else scale, causal, prefix,
                                cap, slopes, spread(pos_q, q), spread(pos_k, k), U(q.dtype))
    got = flat(out.cpu()).double()
    idle = want.isnan()
    assert (got[idle] == 77.0).all(), "a row of no query was written"
    off = (got - want).abs()[~idle]
    assert torch.isfinite(got[~idle]).all()
    assert (off <= tol[~idle]).all(), f"worst {float((off / tol[~idle].clamp_min(1e-300)).max()):.2f} of the tolerance"
    return out


def _qkv(kind, seed, lead_q, lead_k, hq, hk, D, std=1.5):
    g, t = _gen(seed), TYPES[kind]
    return _randn(g, t, *lead_q, hq, D, std=std), _randn(g, t, *lead_k, hk, D, std=1.0), _randn(g, t, *lead_k, hk, D)


def _batch(B, lq, lk, uq=None, uk=None):
    return [(slice(b * lq, b * lq + (uq[b] if uq else lq)), slice(b * lk, b * lk + (uk[b] if uk else lk)))
            for b in range(B)]


def _packed(cu_q, cu_k):
    return [(slice(a, b), slice(c, d)) for a, b, c, d in zip(cu_q, cu_q[1:], cu_k, cu_k[1:])]


SHAPES = [
    # batch, queries, keys, q heads, kv heads, dim
    (1, 1, 1, 1, 1, 1),
    (2, 3, 5, 2, 1, 24),
    (1, 64, 64, 3, 3, 30),
    (1, 65, 130, 2, 2, 32),
    (2, 128, 63, 4, 2, 33),
    (1, 200, 257, 6, 2, 64),
    (1, 33, 300, 3, 1, 72),
    (1, 130, 96, 2, 2, 80),
    (1, 70, 100, 2, 1, 96),
    (1, 257, 191, 5, 1, 128),
    (1, 300, 300, 2, 2, 127),
]


@pytest.mark.parametrize("mask", ["full", "causal"])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_attention_shapes(hl, kind, shape, mask):
    """Every width of a head, odd lengths, shared key heads; causal with fewer keys than
    queries leaves rows with nothing to see."""
    B, lq, lk, hq, hk, D = shape
    print(f"attention {kind} {shape} {mask}", flush=True)
    q, k, v = _qkv(kind, sum(shape), (B, lq), (B, lk), hq, hk, D)
    _check(hl, kind, q, k, v, _batch(B, lq, lk), causal=mask == "causal")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("stride", ["gaps", "odd", "heads"])
@pytest.mark.parametrize("D", [24, 30, 64, 128])
def test_attention_strides(hl, kind, stride, D):
    print(f"attention {kind} {stride} {D}", flush=True)
    q, k, v = _qkv(kind, D, (2, 90), (2, 110), 4, 2, D)
    _check(hl, kind, q, k, v, _batch(2, 90, 110), stride=stride, causal=True)


def test_attention_on_a_packed_qkv_projection(hl):
    """q, k and v as views of one [token, 3, head, dim] buffer, the output in q's place."""
    g = _gen(8)
    qkv = _randn(g, torch.float16, 200, 3, 6, 24)
    d = qkv.cuda()
    want, tol = _attention_want(qkv[:, 0], qkv[:, 1], qkv[:, 2], [(slice(0, 200), slice(0, 200))], 24 ** -0.5, False,
                                None, 0.0, None, None, None, 2.0 ** -11)
    q, k, v = d[:, 0], d[:, 1], d[:, 2]
    hl.op_attention(q, k, v, q)
    torch.cuda.synchronize()
    assert ((d[:, 0].cpu().double() - want).abs() <= tol).all()
    assert torch.equal(d[:, 1:].cpu(), qkv[:, 1:])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("cap", [0.0, 5.0, 50.0])
@pytest.mark.parametrize("bias", ["none", "index", "grid1", "grid2", "grid3", "grid4"])
def test_attention_caps_and_biases(hl, kind, cap, bias):
    print(f"attention {kind} cap {cap} bias {bias}", flush=True)
    B, lq, lk, hq, hk, D = 2, 75, 140, 4, 2, 40
    q, k, v = _qkv(kind, 21, (B, lq), (B, lk), hq, hk, D, std=3.0)
    more = {}
    if bias != "none":
        more["slopes"] = torch.tensor([0.5, 0.03, -0.01, 0.0])
    if bias.startswith("grid"):
        axes, g = int(bias[4:]), _gen(22)
        more["pos_q"] = torch.randint(-40, 40, (lq, axes), generator=g, dtype=torch.int32)
        more["pos_k"] = torch.randint(-40, 40, (B, lk, axes), generator=g, dtype=torch.int32)
        if axes == 2:  # far from zero: differences count, not the coordinates
            more["pos_q"] += 1 << 29
            more["pos_k"] += 1 << 29
    _check(hl, kind, q, k, v, _batch(B, lq, lk), cap=cap, causal=bias == "index", **more)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("bias", ["none", "index", "grid"])
def test_attention_documents(hl, kind, causal, bias):
    """Packed documents, some empty, one of one token, one without keys, and rows behind
    the last that belong to none."""
    cu_q = [0, 1, 1, 130, 131, 200, 200, 290]
    cu_k = [0, 3, 40, 169, 170, 170, 200, 333]
    q, k, v = _qkv(kind, 31, (300,), (350,), 4, 2, 64)
    more = {}
    if bias != "none":
        more["slopes"] = torch.tensor([0.2, 0.1, 0.05, 0.01])
    if bias == "grid":
        g = _gen(32)
        more["pos_q"] = torch.randint(0, 30, (300, 2), generator=g, dtype=torch.int32)
        more["pos_k"] = torch.randint(0, 30, (350, 2), generator=g, dtype=torch.int32)
    print(f"documents {kind} causal {causal} {bias}", flush=True)
    _check(hl, kind, q, k, v, _packed(cu_q, cu_k), causal=causal, cu_q=torch.tensor(cu_q, dtype=torch.int32),
           cu_k=torch.tensor(cu_k, dtype=torch.int32), **more)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_many_short_documents(hl, kind):
    """More sequences than a wave has lanes, most shorter than a tile."""
    g = _gen(41)
    lens = torch.randint(0, 9, (300,), generator=g)
    lens[17] = 150
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)]).to(torch.int32)
    n = int(cu[-1])
    q, k, v = _qkv(kind, 42, (n,), (n,), 2, 1, 32)
    _check(hl, kind, q, k, v, _packed(cu.tolist(), cu.tolist()), causal=True, cu_q=cu, cu_k=cu)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_prefix(hl, kind):
    B, lq, lk = 4, 150, 170
    q, k, v = _qkv(kind, 51, (B, lq), (B, lk), 2, 2, 64)
    prefix = torch.tensor([0, 1, 100, 1000], dtype=torch.int32)  # past the keys: clamped
    _check(hl, kind, q, k, v, _batch(B, lq, lk), causal=True, prefix=prefix)
    # fewer keys than queries: the first rows see the prefix alone
    q, k, v = _qkv(kind, 52, (B, 90), (B, 40), 2, 2, 64)
    _check(hl, kind, q, k, v, _batch(B, 90, 40), causal=True, prefix=torch.tensor([0, -3, 7, 40], dtype=torch.int32))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("causal", [False, True])
def test_attention_padded_batch(hl, kind, causal):
    """Lengths in use below the batch's: rows behind a sequence's last keep what they
    hold, keys behind it have no influence; lengths out of range are clamped."""
    B, lq, lk = 5, 70, 130
    uq, uk = [70, 1, 0, 33, 70], [130, 64, 65, 0, 7]
    q, k, v = _qkv(kind, 61, (B, lq), (B, lk), 4, 1, 48)
    for b in range(B):
        k[b, uk[b]:], v[b, uk[b]:] = math.nan, math.inf
    given_q, given_k = list(uq), list(uk)
    given_q[0], given_k[0], given_k[3] = 1000, 10 ** 9, -4
    _check(hl, kind, q, k, v, _batch(B, lq, lk, uq, uk), causal=causal,
           q_lens=torch.tensor(given_q, dtype=torch.int32), k_lens=torch.tensor(given_k, dtype=torch.int32))


TOKENS = [
    # batch, queries, keys, q heads, kv heads, dim
    (1, 1, 1, 4, 4, 64),
    (1, 1, 1023, 8, 2, 64),
    (3, 1, 2500, 8, 8, 128),
    (2, 1, 4097, 16, 2, 96),
    (2, 4, 3000, 8, 2, 24),
    (5, 2, 700, 9, 3, 30),
    (1, 1, 9000, 40, 1, 128),
    (1, 5, 2000, 24, 2, 33),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", TOKENS, ids=lambda s: "x".join(map(str, s)))
def test_attention_few_queries(hl, kind, causal, shape):
    """One or a few queries a sequence against a long cache, with lengths of its own."""
    B, lq, lk, hq, hk, D = shape
    print(f"few queries {kind} {shape}", flush=True)
    q, k, v = _qkv(kind, 71, (B, lq), (B, lk), hq, hk, D)
    _check(hl, kind, q, k, v, _batch(B, lq, lk), causal=causal)
    uk = [max(0, lk - 700 * b - 1) for b in range(B)]
    for b in range(B):
        k[b, uk[b]:], v[b, uk[b]:] = math.inf, math.nan
    _check(hl, kind, q, k, v, _batch(B, lq, lk, None, uk), causal=causal, cap=20.0,
           slopes=torch.linspace(0, 0.01, hq), k_lens=torch.tensor(uk, dtype=torch.int32))


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_few_queries_of_packed_caches(hl, kind):
    """One query each against caches packed behind one another, one of them empty."""
    cu_k = [0, 1, 900, 900, 2600, 2650]
    q, k, v = _qkv(kind, 81, (5, 1), (2700,), 8, 2, 64)
    seqs = [(slice(n, n + 1), slice(a, b)) for n, (a, b) in enumerate(zip(cu_k, cu_k[1:]))]
    _check(hl, kind, q, k, v, seqs, causal=True, cu_k=torch.tensor(cu_k, dtype=torch.int32))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [24, 64, 128])
def test_attention_unseen_keys_have_no_influence(hl, kind, D):
    """NaN and infinities in keys and values that a query does not see, in the same tile
    as ones it sees: later tokens of a causal sequence, the next document."""
    n = 150
    q, k, v = _qkv(kind, 91, (n,), (n,), 2, 2, D)
    bad = [60, 61, 100, 149]
    kb, vb = k.clone(), v.clone()
    kb[bad], vb[bad] = math.nan, math.inf
    vb[100], kb[100] = math.nan, -math.inf
    qd = q.cuda()
    out, clean = torch.empty_like(qd), torch.empty_like(qd)
    hl.op_attention(qd, kb.cuda(), vb.cuda(), out, causal=True)
    hl.op_attention(qd, k.cuda(), v.cuda(), clean, causal=True)
    torch.cuda.synchronize()
    want, tol = _attention_want(q, k, v, [(slice(0, n), slice(0, n))], D ** -0.5, True, None, 0.0, None, None, None,
                                U(q.dtype))
    assert ((out.cpu().double() - want).abs()[:60] <= tol[:60]).all()
    assert out[60:].isnan().all()  # these see a NaN
    cu = torch.tensor([0, 60, 62, 100, 101, 149, 150], dtype=torch.int32).cuda()
    hl.op_attention(qd, kb.cuda(), vb.cuda(), out, cu_q=cu, cu_k=cu)
    hl.op_attention(qd, k.cuda(), v.cuda(), clean, cu_q=cu, cu_k=cu)
    torch.cuda.synchronize()
    rest = [i for i in range(n) if i not in bad]
    assert torch.isfinite(out[rest]).all()
    assert torch.equal(out[rest], clean[rest])


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_score_spread(hl, kind):
    """Scores far apart, far from zero, rising along the keys (the running maximum moves
    at every step), and a constant row."""
    for name in ("wide", "rising", "falling", "high", "low", "flat"):
        g, t = _gen(101), TYPES[kind]
        q, k, v = _qkv(kind, 101, (1, 96), (1, 700), 2, 2, 64)
        more = {}
        if name == "wide":
            q = (q.float() * 6).to(t)
        elif name in ("rising", "falling"):
            more["slopes"] = torch.tensor([0.3, 0.02]) * (1 if name == "rising" else -1)
        elif name in ("high", "low"):
            q[..., 0] = 30.0 if name == "high" else -30.0
            k[..., 0] = 30.0
        else:
            q.zero_()
        print(f"spread {kind} {name}", flush=True)
        _check(hl, kind, q, k, v, _batch(1, 96, 700), **more)


def test_attention_bits_do_not_depend_on_the_run(hl):
    for lq, lk in ((200, 300), (1, 5000)):
        q, k, v = _qkv("bf16", 111, (2, lq), (2, lk), 8, 2, 128)
        qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
        outs = []
        for _ in range(4):
            out = torch.empty_like(qd)
            need = hl.attention_workspace(qd, kd, vd, out)
            work = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
            hl.op_attention(qd, kd, vd, out, workspace=work)
            outs.append(out)
        torch.cuda.synchronize()
        assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_attention_far_into_a_long_cache(hl):
    """A cache whose element offsets pass 2^31: the sequence at its end is read there."""
    lk, hk, D = 17000, 16, 128  # 17000 * 2048 elements a sequence, 65 of them: 4.5 GB
    cache = torch.zeros(65, lk, hk, D, dtype=torch.float16, device="cuda")
    q, k, v = _qkv("f16", 121, (1, 1), (1, 300), hk, hk, D)
    cache[64, :300] = k[0].cuda()
    values = torch.zeros_like(cache[:1]).expand(65, -1, -1, -1)  # one entry for all, stride 0
    values[0, :300] = v[0].cuda()
    lens = torch.zeros(65, dtype=torch.int32)
    lens[64] = 300
    qd = torch.zeros(65, 1, hk, D, dtype=torch.float16, device="cuda")
    qd[64] = q[0].cuda()
    out = torch.full_like(qd, 5.0)
    need = hl.attention_workspace(qd, cache, values, out, k_lens=lens.cuda())
    hl.op_attention(qd, cache, values, out, k_lens=lens.cuda(),
                    workspace=torch.empty(need, dtype=torch.uint8, device="cuda") if need else None)
    torch.cuda.synchronize()
    want, tol = _attention_want(q[0], k[0], v[0], [(slice(0, 1), slice(0, 300))], D ** -0.5, False, None, 0.0, None,
                                None, None, 2.0 ** -11)
    assert ((out[64].cpu().double() - want).abs() <= tol).all()
    assert (out[:64] == 0).all()  # sequences without keys


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [24, 33, 64, 128])
@pytest.mark.parametrize("rows", [1, 4, 6, 8])
def test_attention_few_queries_in_every_form(hl, kind, D, rows):
    """Positions, a cap, a prefix, lengths on both sides, strides, unseen NaN in a seen
    tile: one to eight rows of a key head against a few chunks of keys."""
    hk, lk, B = 2, 1700, 3
    lq, group = {1: (1, 1), 4: (2, 2), 6: (2, 3), 8: (8, 1)}[rows]
    print(f"few queries in every form {kind} {D} {rows}", flush=True)
    q, k, v = _qkv(kind, 301, (B, lq), (B, lk), hk * group, hk, D)
    seqs = _batch(B, lq, lk)
    _check(hl, kind, q, k, v, seqs, **_mode("grid", hk * group, lq, lk, B, 302))
    _check(hl, kind, q, k, v, seqs, causal=True, **_mode("both grid", hk * group, lq, lk, B, 303))
    _check(hl, kind, q, k, v, seqs, stride="odd", **_mode("negative", hk * group, lq, lk, B, 304))
    _check(hl, kind, q, k, v, seqs, stride="heads", causal=True, prefix=torch.tensor([0, 5, 1800], dtype=torch.int32))
    uq, uk = [lq, 0, max(1, lq - 1)], [lk, 900, 63]
    _check(hl, kind, q, k, v, _batch(B, lq, lk, uq, uk), stride="gaps", causal=True,
           q_lens=torch.tensor(uq, dtype=torch.int32), k_lens=torch.tensor(uk, dtype=torch.int32))
    if lq > 1:  # the last key is seen by the last query alone
        kb, vb = k.clone(), v.clone()
        kb[0, -1], vb[0, -1] = math.nan, math.inf
        qd = q.cuda()
        out = torch.empty_like(qd)
        need = hl.attention_workspace(qd, kb.cuda(), vb.cuda(), out, causal=True)
        work = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
        hl.op_attention(qd, kb.cuda(), vb.cuda(), out, causal=True, workspace=work)
        torch.cuda.synchronize()
        assert out[0, -1].isnan().all() and torch.isfinite(out[0, :-1]).all() and torch.isfinite(out[1:]).all()
        want, tol = _attention_want(q[0], k[0], v[0], [(slice(0, lq), slice(0, lk))], D ** -0.5, True, None, 0.0, None,
                                    None, None, U(q.dtype))
        assert ((out[0].cpu().double() - want).abs()[:-1] <= tol[:-1]).all()


# Enough sequences and key heads that tiles of 128 rows fill the device: the kernels of
# many rows, each width of a head in each of their forms.

MODES = {
    "plain": dict(),
    "index": dict(bias="index"),
    "grid": dict(bias="grid"),
    "cap": dict(cap=20.0),
    "both": dict(cap=30.0, bias="index"),
    "both grid": dict(cap=30.0, bias="grid"),
    "no scale": dict(bias="index", scale=0.0),
    "negative": dict(bias="index", scale=-0.2),
}


def _mode(mode, hq, lq, lk, B, seed):
    more = dict(MODES[mode])
    bias = more.pop("bias", None)
    if bias:
        more["slopes"] = torch.linspace(-0.02, 0.3, hq)
    if bias == "grid":
        g = _gen(seed)
        more["pos_q"] = torch.randint(-20, 20, (lq, 3), generator=g, dtype=torch.int32)
        more["pos_k"] = torch.randint(-20, 20, (lk, 3), generator=g, dtype=torch.int32)
    return more


@pytest.mark.parametrize("mode", list(MODES))
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [24, 64, 80, 128])
def test_attention_many_tiles(hl, kind, D, mode):
    B, lq, lk, hq, hk = 33, 75, 141, 8, 4
    print(f"many tiles {kind} {D} {mode}", flush=True)
    q, k, v = _qkv(kind, 201, (B, lq), (B, lk), hq, hk, D)
    _check(hl, kind, q, k, v, _batch(B, lq, lk), causal=mode in ("index", "cap", "both"),
           **_mode(mode, hq, lq, lk, B, 202))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [1, 30, 33, 72, 96, 127])
@pytest.mark.parametrize("stride", ["plain", "odd", "heads"])
def test_attention_many_tiles_of_odd_heads(hl, kind, D, stride):
    B, lq, lk, hq, hk = 64, 129, 70, 2, 2
    print(f"odd heads {kind} {D} {stride}", flush=True)
    q, k, v = _qkv(kind, 211, (B, lq), (B, lk), hq, hk, D)
    _check(hl, kind, q, k, v, _batch(B, lq, lk), stride=stride, causal=True, slopes=torch.tensor([0.1, 0.0]))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("mode", ["plain", "grid", "cap"])
def test_attention_many_tiles_of_documents(hl, kind, mode):
    """Packed documents of 0 to 300 tokens, more queries than keys in some."""
    g = _gen(221)
    lq, lk = torch.randint(0, 300, (40,), generator=g), torch.randint(0, 300, (40,), generator=g)
    lq[3] = lk[5] = lq[39] = 0
    cu_q, cu_k = (torch.cat([torch.zeros(1, dtype=torch.int64), n.cumsum(0)]).to(torch.int32) for n in (lq, lk))
    q, k, v = _qkv(kind, 222, (int(cu_q[-1]) + 7,), (int(cu_k[-1]) + 3,), 4, 2, 64)
    print(f"many documents {kind} {mode}", flush=True)
    _check(hl, kind, q, k, v, _packed(cu_q.tolist(), cu_k.tolist()), causal=True, cu_q=cu_q, cu_k=cu_k,
           **_mode(mode, 4, q.shape[0], k.shape[0], 1, 223))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [32, 128])
def test_attention_many_tiles_padded_with_a_prefix(hl, kind, D):
    """Lengths of their own on both sides, prefixes, NaN and infinities behind the last
    key and, in a prefix's tile, behind the prefix."""
    B, lq, lk = 70, 140, 200
    g = _gen(231)
    uq, uk = (torch.randint(0, n + 1, (B,), generator=g) for n in (lq, lk))
    prefix = torch.randint(0, 120, (B,), generator=g).to(torch.int32)
    q, k, v = _qkv(kind, 232, (B, lq), (B, lk), 2, 2, D)
    for b in range(B):
        k[b, uk[b]:], v[b, uk[b]:] = math.nan, math.inf
    _check(hl, kind, q, k, v, _batch(B, lq, lk, uq.tolist(), uk.tolist()), causal=True, prefix=prefix,
           q_lens=uq.to(torch.int32), k_lens=uk.to(torch.int32))


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_many_tiles_unseen_keys_have_no_influence(hl, kind):
    B, n, D = 64, 160, 64
    q, k, v = _qkv(kind, 241, (B, n), (B, n), 2, 2, D)
    kb, vb = k.clone(), v.clone()
    kb[3, 70], vb[3, 70] = math.nan, math.inf
    vb[9, 159] = math.nan
    qd = q.cuda()
    out, clean = torch.empty_like(qd), torch.empty_like(qd)
    hl.op_attention(qd, kb.cuda(), vb.cuda(), out, causal=True)
    hl.op_attention(qd, k.cuda(), v.cuda(), clean, causal=True)
    torch.cuda.synchronize()
    others = [b for b in range(B) if b not in (3, 9)]
    assert torch.equal(out[others], clean[others])
    assert out[3, 70:].isnan().all() and out[9, 159].isnan().all()
    assert torch.isfinite(out[3, :70]).all() and torch.isfinite(out[9, :159]).all()
    want, tol = _attention_want(q[3], k[3], v[3], [(slice(0, n), slice(0, n))], D ** -0.5, True, None, 0.0, None, None,
                                None, U(q.dtype))
    assert ((out[3].cpu().double() - want).abs()[:70] <= tol[:70]).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("mode", ["plain", "index"])
def test_attention_many_tiles_score_spread(hl, kind, mode):
    """The running maximum that moves at every stage, scores far apart and far from zero."""
    for name in ("wide", "rising", "falling", "high", "flat"):
        q, k, v = _qkv(kind, 251, (33, 70), (33, 400), 4, 4, 64)
        if name == "wide":
            q = (q.float() * 6).to(q.dtype)
        elif name in ("rising", "falling"):
            ramp = torch.linspace(0, 40, 400) if name == "rising" else torch.linspace(40, 0, 400)
            q[..., 0], k[..., 0] = 8.0, ramp[None, :, None].to(k.dtype)
        elif name == "high":
            q[..., 0], k[..., 0] = 30.0, 30.0
        else:
            q.zero_()
        print(f"many tiles spread {kind} {mode} {name}", flush=True)
        _check(hl, kind, q, k, v, _batch(33, 70, 400), **_mode(mode, 4, 70, 400, 33, 0))


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_without_keys_or_queries(hl, kind):
    """No keys at all: zeros; no queries: no work; a batch of none."""
    t = TYPES[kind]
    for B, lq, hq in ((2, 3, 2), (64, 100, 4)):
        q = torch.ones(B, lq, hq, 48, dtype=t, device="cuda")
        k = torch.empty(B, 0, hq, 48, dtype=t, device="cuda")
        out = torch.full_like(q, 7.0)
        hl.op_attention(q, k, k, out, slopes=torch.ones(hq, device="cuda"),
                        pos_q=torch.zeros(lq, 2, dtype=torch.int32, device="cuda"),
                        pos_k=torch.zeros(0, 2, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert (out == 0).all()
        hl.op_attention(q[:, :0], q, q, out[:, :0])
        hl.op_attention(q[:0], q[:0], q[:0], out[:0])


def test_attention_nan_in_one_query(hl):
    """A query with NaN is NaN and no other is, in a tile of many rows and of few."""
    for B, lq, lk in ((64, 130, 90), (1, 5, 900)):
        q, k, v = _qkv("bf16", 311, (B, lq), (B, lk), 2, 1, 64)
        qb = q.clone()
        qb[0, 2, 1, 5] = math.nan
        out, clean = torch.empty_like(q, device="cuda"), torch.empty_like(q, device="cuda")
        kd, vd = k.cuda(), v.cuda()
        need = hl.attention_workspace(out, kd, vd, out.clone())
        work = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
        hl.op_attention(qb.cuda(), kd, vd, out, workspace=work)
        hl.op_attention(q.cuda(), kd, vd, clean, workspace=work)
        torch.cuda.synchronize()
        assert out[0, 2, 1].isnan().all()
        out[0, 2, 1] = clean[0, 2, 1]
        assert torch.equal(out, clean)


def test_attention_on_two_streams_at_once(hl):
    """Two calls in flight, each with a workspace of its own, against the same call alone."""
    q, k, v = _qkv("f16", 321, (4, 1), (4, 6000), 8, 2, 128)
    q2, k2, v2 = _qkv("f16", 322, (3, 2), (3, 5000), 8, 2, 128)
    sets = []
    for a in ((q, k, v), (q2, k2, v2)):
        d = [x.cuda() for x in a]
        out, alone = torch.empty_like(d[0]), torch.empty_like(d[0])
        need = hl.attention_workspace(*d, out)
        assert need > 0
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        hl.op_attention(*d, alone, workspace=work)
        sets.append((d, out, alone, work, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for d, out, alone, work, s in sets:
            hl.op_attention(*d, out, workspace=work, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for d, out, alone, work, s in sets:
        assert torch.equal(out, alone)


def test_attention_refuses_a_small_workspace(hl):
    q, k, v = _qkv("f16", 331, (1, 1), (1, 6000), 8, 2, 64)
    d = [x.cuda() for x in (q, k, v)]
    out = torch.empty_like(d[0])
    need = hl.attention_workspace(*d, out)
    with pytest.raises(hl.HatError) as e:
        hl.op_attention(*d, out)
    assert str(need) in str(e.value)
    with pytest.raises(hl.HatError):
        hl.op_attention(*d, out, workspace=torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    with pytest.raises(hl.HatError):
        hl.op_attention(*d, out, workspace=torch.empty(need + 8, dtype=torch.uint8, device="cuda")[8:])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("shape", [(130, 1, 20, 8, 2), (70, 3, 70, 6, 2), (40, 16, 600, 4, 4), (150, 64, 64, 2, 2)],
                         ids=lambda s: "x".join(map(str, s)))
def test_attention_many_short_sequences(hl, kind, D, shape):
    """Few rows each, but sequences enough to fill the device."""
    B, lq, lk, hq, hk = shape
    q, k, v = _qkv(kind, 341, (B, lq), (B, lk), hq, hk, D)
    print(f"many short {kind} {D} {shape}", flush=True)
    _check(hl, kind, q, k, v, _batch(B, lq, lk), causal=True, slopes=torch.linspace(0, 0.2, hq))
    g = _gen(342)
    uk = torch.randint(0, lk + 1, (B,), generator=g)
    _check(hl, kind, q, k, v, _batch(B, lq, lk, None, uk.tolist()), k_lens=uk.to(torch.int32))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n", [6, 90])
def test_attention_packed_on_one_side(hl, kind, n):
    """A batch of queries against packed caches, and packed queries against a batch of
    padded ones, with positions, by few sequences and by many."""
    g = _gen(351)
    lk = torch.randint(0, 150, (n,), generator=g)
    cu_k = torch.cat([torch.zeros(1, dtype=torch.int64), lk.cumsum(0)]).to(torch.int32)
    q, k, v = _qkv(kind, 352, (n, 3), (int(cu_k[-1]) + 2,), 4, 2, 64)
    seqs = [(slice(3 * b, 3 * b + 3), slice(int(cu_k[b]), int(cu_k[b + 1]))) for b in range(n)]
    more = dict(slopes=torch.linspace(0.0, 0.2, 4),
                pos_q=torch.randint(0, 30, (n, 3, 2), generator=g, dtype=torch.int32),
                pos_k=torch.randint(0, 30, (k.shape[0], 2), generator=g, dtype=torch.int32))
    print(f"packed keys {kind} {n}", flush=True)
    _check(hl, kind, q, k, v, seqs, causal=True, cu_k=cu_k)
    _check(hl, kind, q, k, v, seqs, cu_k=cu_k, **more)
    lq = torch.randint(0, 50, (n,), generator=g)
    cu_q = torch.cat([torch.zeros(1, dtype=torch.int64), lq.cumsum(0)]).to(torch.int32)
    q, k, v = _qkv(kind, 353, (int(cu_q[-1]) + 2,), (n, 90), 4, 2, 64)
    uk = torch.randint(0, 91, (n,), generator=g)
    seqs = [(slice(int(cu_q[b]), int(cu_q[b + 1])), slice(90 * b, 90 * b + int(uk[b]))) for b in range(n)]
    print(f"packed queries {kind} {n}", flush=True)
    _check(hl, kind, q, k, v, seqs, causal=True, cu_q=cu_q, k_lens=uk.to(torch.int32))
    more = dict(slopes=torch.linspace(0.0, 0.2, 4),
                pos_q=torch.randint(0, 30, (q.shape[0], 2), generator=g, dtype=torch.int32),
                pos_k=torch.randint(0, 30, (n, 90, 2), generator=g, dtype=torch.int32))
    _check(hl, kind, q, k, v, seqs, cap=9.0, cu_q=cu_q, k_lens=uk.to(torch.int32), **more)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_offsets_out_of_range_are_clamped(hl, kind):
    """Offsets and lengths that point outside the tensors read and write nothing there."""
    q, k, v = _qkv(kind, 361, (300,), (300,), 32, 32, 32)
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    guard = torch.full((340, 32, 32), 55.0, dtype=q.dtype, device="cuda")
    out = guard[20:320]
    cu = torch.tensor([-50, 100, 100, 299, 100000, 2 ** 31 - 1], dtype=torch.int32).cuda()
    hl.op_attention(qd, kd, vd, out, cu_q=cu, cu_k=cu, causal=True)
    torch.cuda.synchronize()
    assert (guard[:20] == 55.0).all() and (guard[320:] == 55.0).all()
    good = torch.tensor([0, 100, 100, 299, 300, 300], dtype=torch.int32).cuda()
    want = torch.empty_like(qd)
    hl.op_attention(qd, kd, vd, want, cu_q=good, cu_k=good, causal=True)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("shape", [(33, 70, 6000, 4), (1, 2, 9000, 2)], ids=["many", "few"])
def test_attention_many_small_probabilities(hl, kind, shape):
    """One key far above thousands whose probabilities are 2^-15.5 of its own: subnormal
    in fp16, a fifth of the sum together."""
    B, lq, lk, h = shape
    t = TYPES[kind]
    q, k, v = torch.zeros(B, lq, h, 32, dtype=t), torch.zeros(B, lk, h, 32, dtype=t), torch.zeros(B, lk, h, 32, dtype=t)
    q[..., 0] = 1.0
    k[:, 7, :, 0] = 15.5
    v[:] = 1.0
    v[:, 7] = -1.0
    print(f"small probabilities {kind} {shape}", flush=True)
    _check(hl, kind, q, k, v, _batch(B, lq, lk), scale=math.log(2.0))


# ---- together ------------------------------------------------------------------------


def _block(hl, x, pos, qkv_w, proj_w, cu, work, stream=None):
    """A transformer block's attention half on image tokens: norm, projection (torch's),
    rotation, attention within each image, projection, join with the next norm."""
    T, C = x.shape
    h, xo, hn = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    hl.op_residual_norm(x, h=h, pre="rms", stream=stream)
    qkv = (h @ qkv_w).reshape(T, 3, 4, C // 4)
    q, k, v = qkv[:, 0], qkv[:, 1], qkv[:, 2]
    hl.op_rotary(q, k, pos, [C // 16, C // 16], stream=stream)
    out = torch.empty(T, 4, C // 4, dtype=x.dtype, device=x.device)
    hl.op_attention(q, k, v, out, cu_q=cu, cu_k=cu, cap=30.0, workspace=work, stream=stream)
    y = out.reshape(T, C) @ proj_w
    hl.op_residual_norm(x, y, xo, hn, scale=0.5, post="rms", pre="layer", stream=stream)
    return xo, hn


def _block_want(x, pos, qkv_w, proj_w, cu):
    T, C = x.shape
    rms = lambda v: v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-5)  # noqa: E731
    qkv = (rms(x) @ qkv_w).reshape(T, 3, 4, C // 4)
    q, k = (_rotary_want(qkv[None, :, i], pos, [C // 16, C // 16], "halves", False, False)[0][0] for i in (0, 1))
    o = torch.zeros(T, 4, C // 4, dtype=torch.float64)
    for a, b in zip(cu, cu[1:]):
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b]) * (C // 4) ** -0.5
        o[a:b] = torch.einsum("hij,jhd->ihd", torch.softmax(30 * torch.tanh(s / 30), -1), qkv[a:b, 2])
    xo = x + 0.5 * rms(o.reshape(T, C) @ proj_w)
    c = xo - xo.mean(1, keepdim=True)
    return xo, c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)


def _block_inputs(seed):
    g = _gen(seed)
    cu, C = [0, 64, 164, 192], 128
    x = _randn(g, torch.float32, 192, C)
    pos = torch.stack([torch.arange(192) // 10, torch.arange(192) % 10], 1).to(torch.int32)
    return x, pos, _randn(g, torch.float32, C, 3 * C, std=0.12), _randn(g, torch.float32, C, C, std=0.1), cu


def test_a_block_of_the_operators(hl):
    x, pos, a, b, cu = _block_inputs(131)
    got = _block(hl, x.cuda(), pos.cuda(), a.cuda(), b.cuda(), torch.tensor(cu, dtype=torch.int32).cuda(), None)
    torch.cuda.synchronize()
    want = _block_want(x.double(), pos, a.double(), b.double(), cu)
    # fp32 throughout: sums of 128 products twice, each within (128 + 8) u of values of a
    # few units, through a softmax of scores of a few units and two norms that divide by
    # spreads of about one: below 1000 u
    for g, w in zip(got, want):
        assert (g.cpu().double() - w).abs().max() <= 1000 * u * 4


def test_captured_and_replayed_on_a_stream(hl):
    """The three operators in a graph on a stream of their own, replayed with new inputs
    in the same buffers, the same work done eagerly on another stream between."""
    g = _gen(141)
    x = torch.zeros(2, 1, 8, 64, dtype=torch.bfloat16, device="cuda")
    k, v = (_randn(g, torch.bfloat16, 2, 3000, 2, 64).cuda() for _ in range(2))
    pos = torch.tensor([[5], [9]], dtype=torch.int32, device="cuda").reshape(2, 1, 1)
    lens = torch.tensor([3000, 1777], dtype=torch.int32, device="cuda")

    def passes(x, q, o, h, work, stream):
        hl.op_rotary(x, None, pos, [16], q_out=q, stream=stream)
        hl.op_attention(q, k, v, o, k_lens=lens, causal=True, workspace=work, stream=stream)
        hl.op_residual_norm(x.reshape(2, 512), o.reshape(2, 512), None, h, pre="rms", stream=stream)

    def buffers():
        q, o = torch.empty_like(x), torch.empty_like(x)
        need = hl.attention_workspace(q, k, v, o, k_lens=lens, causal=True)
        work = torch.empty(need, dtype=torch.uint8, device="cuda") if need else None
        return q, o, torch.empty(2, 512, dtype=torch.bfloat16, device="cuda"), work

    inside, outside = buffers(), buffers()
    s = torch.cuda.Stream()
    passes(x, *inside, s.cuda_stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        passes(x, *inside, torch.cuda.current_stream().cuda_stream)
    for seed in range(4):
        x.copy_(_randn(_gen(seed), torch.bfloat16, 2, 1, 8, 64))
        torch.cuda.synchronize()
        graph.replay()
        passes(x, *outside, None)
        torch.cuda.synchronize()
        for a, b in zip(inside[:3], outside[:3]):
            assert torch.equal(a, b)


def test_device_arrays_without_torch(hl):
    """The binding's own device tensors: fp32, no other library in the process's way."""
    rng = np.random.default_rng(7)
    q, k, v = (rng.standard_normal((50, 6, 24), dtype=np.float32) for _ in range(3))
    d = [hl.DeviceArray(a.shape, "float32", a) for a in (q, k, v)]
    out = hl.DeviceArray((50, 6, 24), "float32")
    hl.op_attention(*d, out)
    hl.synchronize()
    want, tol = _attention_want(*(torch.from_numpy(a) for a in (q, k, v)), [(slice(0, 50), slice(0, 50))], 24 ** -0.5,
                                False, None, 0.0, None, None, None, u)
    assert ((torch.from_numpy(out.numpy()).double() - want).abs() <= tol).all()
