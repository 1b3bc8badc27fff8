"""Windowed attention at scores, scales and values far from 1, against a 64-bit restatement.

u = 2^-24, e = finfo(t).eps / 2 (0.. one rounding to the storage type).  Queries and keys are small integers times a power of
two and scales are powers of two, so that every score is exact in fp32 and in 64 bits: what is left of the error is that of
the softmax, not of the dot products.  With x = (s - max) c, c = scale log2 e (two roundings) and one more in the product,
the weight w = 2^x is off by 3 u |ln w| + 2 u (the instruction's own error), the row's sum by the mean of that over the row:
  rel p_ij <= u (3 |ln w_ij| + 3 sum_j p_ij |ln w_ij| + n / 8 + 40)."""
import math

import pytest
import torch

from test_gpu_window_attn import DTYPES, U, _ref, _visible, _within

gpu = pytest.mark.gpu


def _integers(B, L, Hq, Hkv, D, dt, unit, top, seed):
    """q, k: integers in [-top, top] times `unit`; v, dO normal; histories that begin and end inside the row, one empty."""
    g = torch.Generator().manual_seed(seed)
    whole = lambda *s: (torch.randint(-top, top + 1, s, generator=g).double() * unit).to(dt)
    q, k = whole(B, L, Hq, D), whole(B, L, Hkv, D)
    v, go = (torch.randn(s, generator=g).to(dt) for s in ((B, L, Hkv, D), (B, L, Hq, D)))
    begin = torch.tensor([0, L // 3, 5, 0][:B], dtype=torch.int32)
    end = torch.tensor([L, L - 3, 5, L][:B], dtype=torch.int32)
    return q, k, v, go, begin, end


def _relp(r, vis):
    """The bound of rel p above, [B, H, L, L]; 0 where nothing is visible."""
    top = r["p"].amax(-1, keepdim=True)
    w = r["p"] / torch.where(top > 0, top, torch.ones_like(top))
    ln = torch.where(w > 0, w, torch.ones_like(w)).log().abs()
    return U * (3 * ln + 3 * (r["p"] * ln).sum(-1, keepdim=True) + r["n"] / 8 + 40) * vis[:, None]


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("shape", [(3, 150, 4, 2, 64, 40, 3), (130, 200, 4, 1, 32, 40, 3), (3, 70, 2, 2, 50, 70, 0)])
@pytest.mark.parametrize("scale,unit", [(2.0 ** 27, 1.0), (2.0 ** 33, 1.0), (2.0 ** 99, 1.0), (2.0 ** -3, 2.0 ** 11), (2.0 ** -30, 2.0 ** 11)])
def test_forward_at_large_scores(dev, shape, dt, scale, unit):
    """Scores of 2^-30 to 2^110: only a query without keys gives zeros and lse -inf, and the single-token form agrees.
    P is rounded to 16-bit types (e) or not; A = sum p |v|."""
    from deeprec_amd import kernels as Kn
    B, L, Hq, Hkv, D, W, S = shape
    n = min(B, 3)                                                            # the rest repeats these
    q, k, v, go, begin, end = _integers(n, L, Hq, Hkv, D, dt, unit, 4, L + D)
    vis = _visible(n, L, W, S, begin, end)
    r = _ref(q, k, v, go, vis, scale)
    e = torch.finfo(dt).eps / 2
    absV = r["V"].abs()
    lim = ((r["p"] * (_relp(r, vis) + (0.0 if dt == torch.float32 else e))) @ absV).permute(0, 2, 1, 3)
    lim = lim * (1 + e) + e * r["out"].abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps + 1e-30
    d = lambda t: t.repeat(-(-B // n), *[1] * (t.dim() - 1))[:B].to(dev)
    mask = dict(window=W, sinks=S, scale=scale, begin=d(begin), end=d(end))
    out, lse = Kn.window_attn_forward(d(q), d(k), d(v), **mask)
    _within("out", out[:n], r["out"], lim)
    none = ~vis.any(2)[:, None].expand(n, Hq, L)
    got = lse[:n].cpu().double()
    assert bool((got[none] == -math.inf).all())
    assert bool(((got - r["lse"]).abs()[~none] <= 4 * U * r["lse"].abs()[~none] + 1e-5).all())
    last = end.long().clamp(0, L) - 1
    rows = torch.arange(n)
    some = (end > begin) & (last >= 0)
    tok = Kn.window_attn_token(q[rows, last.clamp_min(0)].to(dev), k.to(dev), v.to(dev), W, S, scale, begin.to(dev), end.to(dev))
    want = torch.where(some[:, None, None], r["out"][rows, last.clamp_min(0)], torch.zeros((), dtype=torch.float64))
    _within("token", tok, want, torch.where(some[:, None, None], lim[rows, last.clamp_min(0)], torch.full((), 1e-30, dtype=torch.float64)))


def _limits(r, vis, dt, D, G, scale, e16, eP):
    """Bounds of out, dq, dk, dv [in the outputs' layout].  P enters its product with a relative error eP beside _relp's, dS with
    e16.  delta is as exact as P: <dO, O> with O in fp32, or from the rounded O (delta_0) and corrected by
    r = sum p (dP - delta_0), which is off by p's errors on |dP - delta_0| and fp32 sums; r P K, taken off dQ at the end, has P
    rounded once to a 16-bit type (e).  With |x|_1 the absolute sum of a dot product's terms:
      |ddS| <= p scale [(relp + e16) |dP - delta| + (2 D + 8) u (|dO v|_1 + |delta|) + err delta]
    (the D terms of dP are added to -delta: no partial sum exceeds |dO v|_1 + |delta|), and fp32 sums of m terms add
    (m / 8 + 8) u of their absolute sum."""
    e = torch.finfo(dt).eps / 2
    p, relp = r["p"], _relp(r, vis)
    absV, absK, absGO = r["V"].abs(), r["K"].abs(), r["GO"].abs()
    t = lambda x: x.transpose(2, 3)
    out = (p * (relp + eP)) @ absV
    dot = absGO @ t(absV) + r["delta"].abs()
    diff = (r["dp"] - r["delta"]).abs()
    err0 = (absGO * (out + e * r["o"].abs())).sum(-1, keepdim=True)          # delta_0 - delta: O off by its rounding
    err = (p * (relp * (diff + err0) + (2 * D + 8) * U * dot)).sum(-1, keepdim=True) + (r["n"] / 8 + 8) * U * (p * (diff + err0)).sum(-1, keepdim=True)
    if dt == torch.float32:
        err = err0 + (2 * D + 8) * U * (absGO * r["o"].abs()).sum(-1, keepdim=True)
    dS = p * scale * ((relp + e16) * (diff + (err0 if e16 else 0.0)) + (2 * D + 8) * U * dot + err)
    absS = p * scale * (diff + err0)
    dq = dS @ absK + (r["n"] / 8 + 8) * U * (absS @ absK) + (scale * e * err0 * (p @ absK) if dt != torch.float32 else 0.0)
    dk = t(dS) @ r["Q"].abs() + (r["nk"] * G / 8 + 8) * U * (t(absS) @ r["Q"].abs())
    dv = t(p * (relp + eP)) @ absGO + (r["nk"] * G / 8 + 8) * U * (t(p) @ absGO)
    fin = lambda lim, ref: lim * (1 + e) + e * ref.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2 + 1e-30
    return (fin(out.permute(0, 2, 1, 3), r["out"]), fin(dq.permute(0, 2, 1, 3), r["dq"]), fin(r["group"](dk), r["dk"]),
            fin(r["group"](dv), r["dv"]))


def _check(dev, q, k, v, go, W, S, scale, begin, end, limits):
    from deeprec_amd import kernels as Kn
    d = lambda t: t.to(dev)
    mask = dict(window=W, sinks=S, scale=scale, begin=d(begin), end=d(end))
    out, lse = Kn.window_attn_forward(d(q), d(k), d(v), **mask)
    grads = Kn.window_attn_backward(d(q), d(k), d(v), out, lse, d(go), **mask)
    B, L, Hq, D = q.shape
    vis = _visible(B, L, W, S, begin, end)
    r = _ref(q, k, v, go, vis, scale)
    lims = limits(r, vis)
    for name, x, lim in zip(("out", "dq", "dk", "dv"), (out,) + grads, lims):
        _within(name, x, r[name], lim)
    return out, lse, grads


@gpu
@pytest.mark.parametrize("shape", [(3, 150, 4, 2, 64, 40, 3), (2, 400, 2, 1, 50, 40, 3), (3, 90, 2, 2, 150, 90, 0)])
@pytest.mark.parametrize("shift", [0, 256, -256, 2048, -2048])
def test_backward_far_from_zero(dev, shape, shift):
    """Scores of about shift^2 / 8 (8192, 524288) that differ by a few: P has fp32's digits all the same, in every product."""
    B, L, Hq, Hkv, D, W, S = shape
    q, k, v, go, begin, end = _integers(B, L, Hq, Hkv, D, torch.float32, 1.0, 2, L + D)
    q[..., 0], k[..., 0] = float(shift), float(abs(shift))
    _check(dev, q, k, v, go, W, S, 0.125, begin, end, lambda r, vis: _limits(r, vis, torch.float32, D, Hq // Hkv, 0.125, 0.0, 0.0))


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("scale", [2.0 ** 33, 2.0 ** 99])
def test_backward_at_large_scores(dev, dt, scale):
    """One key, or several with equal scores, carries a row: dV is the sum of dO over the rows that chose it, dQ and dK stay
    within the rounding of dP - delta times scale (fp16 cannot hold that: its dQ and dK are not compared)."""
    from deeprec_amd import kernels as Kn
    B, L, Hq, Hkv, D, W, S = 3, 150, 4, 2, 64, 40, 3
    q, k, v, go, begin, end = _integers(B, L, Hq, Hkv, D, dt, 1.0, 4, 7)
    d = lambda t: t.to(dev)
    mask = dict(window=W, sinks=S, scale=scale, begin=d(begin), end=d(end))
    out, lse = Kn.window_attn_forward(d(q), d(k), d(v), **mask)
    dq, dk, dv = Kn.window_attn_backward(d(q), d(k), d(v), out, lse, d(go), **mask)
    vis = _visible(B, L, W, S, begin, end)
    r = _ref(q, k, v, go, vis, scale)
    e = torch.finfo(dt).eps / 2
    lim = _limits(r, vis, dt, D, Hq // Hkv, scale, e, 0.0 if dt == torch.float32 else e)
    _within("dv", dv, r["dv"], lim[3])
    if dt != torch.float16:
        _within("dq", dq, r["dq"], lim[1])
        _within("dk", dk, r["dk"], lim[2])


@gpu
@pytest.mark.parametrize("shape", [(2, 150, 4, 2, 64, 40, 3), (1, 700, 2, 1, 64, 100, 33)])
@pytest.mark.parametrize("scale,unit", [(2.0 ** -13, 8.0), (2.0 ** -19, 64.0), (2.0 ** 13, 2.0 ** -9)])
def test_fp16_gradients_at_any_scale(dev, shape, scale, unit):
    """A scale far from D^-0.5 with queries and keys that make up for it: dS is an ordinary number before the scale, which must
    not meet it in fp16.  The second shape's first items get their far gradients from a launch of their own."""
    B, L, Hq, Hkv, D, W, S = shape
    q, k, v, go, begin, end = _integers(B, L, Hq, Hkv, D, torch.float16, unit, 4, 17)
    e = 2.0 ** -11
    _check(dev, q, k, v, go, W, S, scale, begin, end, lambda r, vis: _limits(r, vis, torch.float16, D, Hq // Hkv, scale, e, e))


@gpu
@pytest.mark.parametrize("shape", [(2, 150, 4, 2, 64, 40, 3), (1, 700, 2, 1, 64, 100, 33), (2, 90, 2, 1, 80, 90, 0)])
@pytest.mark.parametrize("size", [4096.0])
def test_fp16_values_of_any_size(dev, shape, size):
    """Values that line up with dO: |dP| = D size, 262144, where dQ and dK are ordinary fp16 numbers."""
    B, L, Hq, Hkv, D, W, S = shape
    q, k, v, go, begin, end = _integers(B, L, Hq, Hkv, D, torch.float16, 2.0 ** -4 if size > 1 else 4.0, 4, 23)
    g = torch.Generator().manual_seed(5)
    sign = lambda *s: torch.randint(0, 2, s, generator=g).double() * 2 - 1
    pattern = sign(D)
    v = (sign(B, L, Hkv, 1) * pattern * size).half()
    go = (pattern.expand(B, L, Hq, D) * 1.0).half()
    scale = 0.125 if size > 1 else 2.0 ** -6
    e = 2.0 ** -11
    _check(dev, q, k, v, go, W, S, scale, begin, end, lambda r, vis: _limits(r, vis, torch.float16, D, Hq // Hkv, scale, e, e))


@gpu
@pytest.mark.parametrize("W,S", [(1000, 0), (250, 20)])
def test_fp16_small_probabilities(dev, W, S):
    """A sharp softmax with a loss scale: keys that no query weighs strongly still get their gradient, key by key.
    P goes into its products times 2^15, its last bit 2^-24 2^-15: half of it is 2^-40.  dS goes in as two halves, its largest
    brought to 2^13 or more: 2^-25 / 2^13 = 2^-38 of the largest |dS|."""
    L, D, dt = 1000, 64, torch.float16
    q, k, v, go, begin, end = _integers(1, L, 2, 1, D, dt, 1.0, 7, 29)
    go = (go.float() * 256).half()
    e = 2.0 ** -11

    def limits(r, vis):
        out, dq, dk, dv = _limits(r, vis, dt, D, 2, 0.125, e * e, e)
        seen = vis[:, None].double()
        big = (r["p"] * (r["dp"] - r["delta"])).abs().amax()
        dv = dv + r["group"](2.0 ** -40 * seen.transpose(2, 3) @ r["GO"].abs())
        dk = dk + r["group"](2.0 ** -38 * big * 0.125 * seen.transpose(2, 3) @ r["Q"].abs())
        dq = dq + (2.0 ** -38 * big * 0.125 * seen @ r["K"].abs()).permute(0, 2, 1, 3)
        out = out + (2.0 ** -40 * seen @ r["V"].abs()).permute(0, 2, 1, 3)
        return out, dq, dk, dv
    _check(dev, q, k, v, go, W, S, 0.125, begin, end, limits)


FAR = [(1, 400, 2, 1, D, 24, 5) for D in (7, 24, 32, 50, 80, 128, 150, 256)] + [(3, 330, 8, 2, 64, 16, 33), (2, 620, 1, 1, 16, 40, 64)]


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,L,Hq,Hkv,D,W,S", [(3, 150, 4, 2, 64, 40, 3), (2, 100, 2, 2, 128, 100, 0)] + FAR)
def test_errors_are_those_of_one_rounding(dev, B, L, Hq, Hkv, D, W, S, dt):
    """16-bit types: P and dS enter their products as two halves (e^2 left of them), delta is corrected, so beside the one
    rounding of the result there is nothing of the order e.  FAR: shapes whose first items get the gradients of far queries
    from a launch of their own, at every tile width.  Outside the history stands NaN.
    fp16: P times 2^15 and dS brought to 2^13 or more lose 2^-40 and 2^-38 of the largest."""
    q, k, v, go, begin, end = _integers(B, L, Hq, Hkv, D, dt, 0.25, 4, B + L + D)
    pos = torch.arange(L)[None]
    pad = (pos < begin[:, None]) | (pos >= end[:, None])
    for t in (q, k, v, go):
        t[pad] = math.nan
    scale = 0.25
    e = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2

    def limits(r, vis):
        lims = _limits(r, vis, dt, D, Hq // Hkv, scale, e * e, e * e)
        if dt != torch.float16:
            return lims
        seen, big = vis[:, None].double(), (r["p"] * (r["dp"] - r["delta"])).abs().amax() * scale
        back = lambda t: t.permute(0, 2, 1, 3)
        return (lims[0] + back(2.0 ** -40 * seen @ r["V"].abs()), lims[1] + back(2.0 ** -38 * big * seen @ r["K"].abs()),
                lims[2] + r["group"](2.0 ** -38 * big * seen.transpose(2, 3) @ r["Q"].abs()),
                lims[3] + r["group"](2.0 ** -40 * seen.transpose(2, 3) @ r["GO"].abs()))
    _check(dev, q, k, v, go, W, S, scale, begin, end, limits)


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,D", [(100, 64), (3000, 64), (700, 80)])
def test_token_errors_are_those_of_one_rounding(dev, L, D, dt):
    """The single-token form, in one workgroup and split over several."""
    from deeprec_amd import kernels as Kn
    B, Hq, Hkv = 3, 4, 2
    q, k, v, go, begin, end = _integers(B, L, Hq, Hkv, D, dt, 0.25, 4, L + D)
    out = Kn.window_attn_token(q[:, 0].to(dev), k.to(dev), v.to(dev), L, 0, 0.25, begin.to(dev), end.to(dev))
    lo, hi = begin.long()[:, None, None], end.long()[:, None, None]
    j = torch.arange(L)[None, None]
    vis = ((j >= lo) & (j < hi))                                             # [B, 1, L]: one query
    Q, K, V = q[:, 0].double()[:, :, None], *(t.double().permute(0, 2, 1, 3).repeat_interleave(Hq // Hkv, 1) for t in (k, v))
    s = (Q @ K.transpose(2, 3) * 0.25).masked_fill(~vis[:, None], -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
    r = dict(p=p, n=vis.sum(2)[:, None, :, None].double())
    e = torch.finfo(dt).eps / 2
    ref = (p @ V)[:, :, 0]
    lim = ((p * (_relp(r, vis) + e * e) + 2.0 ** -40 * vis[:, None]) @ V.abs())[:, :, 0]
    _within("out", out, ref, lim * (1 + e) + e * ref.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2 + 1e-30)


@gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_far_first_items_in_graphs(dev, dt):
    """Forward and backward captured twice, far first items by their own launch; replayed with eager calls between, once on
    scores beyond 65536, where the backward takes the rows' maxima itself: the same bits as the eager call every time."""
    from deeprec_amd import kernels as Kn
    B, L, Hq, Hkv, D, W, S = 3, 400, 4, 2, 64, 24, 5
    q, k, v, go, begin, end = (t.to(dev) for t in _integers(B, L, Hq, Hkv, D, dt, 0.25, 4, 3))
    mask = dict(window=W, sinks=S, begin=begin, end=end)

    def call():
        o, s = Kn.window_attn_forward(q, k, v, **mask)
        return (o, s) + Kn.window_attn_backward(q, k, v, o, s, go, **mask)
    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = call()
        graphs.append((gr, res))
    for size in (1.0, 4096.0, 0.5, 1.0):
        for t in (q, k, v, go):
            t.normal_()
        q.mul_(size)
        k.mul_(size if size < 2 else 64.0)
        mine = call()
        assert (float(mine[1][mine[1] > -math.inf].abs().max()) > 65536) == (size > 2)
        for gr, res in graphs:
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, mine))
        assert all(torch.equal(a, b) for a, b in zip(call(), mine))


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** 10])
def test_loss_scale_with_far_first_items(dev, dt, size):
    """dO far from 1 where the first items' far gradients join those of the window (fp16: each with a power of two of its own)."""
    B, L, Hq, Hkv, D, W, S = 2, 500, 4, 2, 64, 40, 20
    q, k, v, go, begin, end = _integers(B, L, Hq, Hkv, D, dt, 0.25, 4, 19)
    go = (go.float() * size).to(dt)
    e = torch.finfo(dt).eps / 2

    def limits(r, vis):
        lims = _limits(r, vis, dt, D, Hq // Hkv, 0.25, e * e, e * e)
        if dt != torch.float16:
            return lims
        seen, big = vis[:, None].double(), (r["p"] * (r["dp"] - r["delta"])).abs().amax() * 0.25
        back = lambda t: t.permute(0, 2, 1, 3)
        return (lims[0] + back(2.0 ** -40 * seen @ r["V"].abs()), lims[1] + back(2.0 ** -38 * big * seen @ r["K"].abs()),
                lims[2] + r["group"](2.0 ** -38 * big * seen.transpose(2, 3) @ r["Q"].abs()),
                lims[3] + r["group"](2.0 ** -40 * seen.transpose(2, 3) @ r["GO"].abs()))
    _check(dev, q, k, v, go, W, S, 0.25, begin, end, limits)
