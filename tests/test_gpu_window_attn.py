"""Windowed attention with first items: forward, backward and the single-token form against a 64-bit restatement.

Tolerances.  u = 2^-24 (fp32 arithmetic), e = finfo(t).eps / 2 (one rounding to the storage type).  Inputs are exact in
both.  For one query with n visible keys, A = sum_j p_j |v_j| bounds the terms of out:
  scores: dot products of D terms, |s - s~| <= (D + 4) u sum |q_d k_d| scale =: ds (their largest over the visible keys);
  p: relative 2 ds + (n / 8 + 32) u (maximum, exponential, sums), and P is rounded to the type before the second product
  (16-bit types: e relative): |out - ref| <= (2 ds + (n / 8 + 40) u + e16) A, then one rounding e |out|;  e16 = e for 16-bit
  types, 0 for fp32.
Gradients: dV_j = sum_i p_ij dO_i, with the same relative error of p on the absolute sum.  dS = p (dP - delta) scale: dP and
delta are D-term sums, delta is taken from the rounded out (an error e |O| |dO| summed), dS itself is rounded (e16):
  |ddS_ij| <= p scale [ (rel p + e16) (|dP| + |delta|) + (2 D + 8) u sum|dO v| + (2 D + 8) u sum |dO O| + (e + errA) sum|dO| |O|max ]
and dQ, dK sum that against |K|, |Q| (fp32 sums: another (n / 8 + 8) u of the absolute sums), then one rounding."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def _inputs(B, L, Hq, Hkv, D, dt, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).to(dt)
    q, k, v, go = r(B, L, Hq, D), r(B, L, Hkv, D), r(B, L, Hkv, D), r(B, L, Hq, D)
    b = torch.randint(0, L + 1, (B,), generator=g)
    e = torch.randint(0, L + 1, (B,), generator=g)
    begin, end = torch.minimum(b, e), torch.maximum(b, e)
    begin[0], end[0] = 0, L
    if B > 2:
        begin[1], end[1] = L // 2, L // 2                                    # empty
        begin[2], end[2] = -7, L + 9                                         # cut to the row
    if B > 3:
        begin[3], end[3] = L, 0                                              # upside down: empty
    return q, k, v, go, begin.to(torch.int32), end.to(torch.int32)


def _visible(B, L, W, S, begin, end):
    lo, hi = begin.long().clamp(0, L)[:, None, None], end.long().clamp(0, L)[:, None, None]
    i, j = torch.arange(L)[None, :, None], torch.arange(L)[None, None, :]
    return (lo <= j) & (j <= i) & (i < hi) & ((i - j < W) | (j - lo < S))


def _ref(q, k, v, go, vis, scale):
    """64-bit out, lse, dq, dk, dv and the absolute sums that bound the errors."""
    B, L, Hq, D = q.shape
    G = Hq // k.shape[2]
    Q, K, V, GO = (t.double().permute(0, 2, 1, 3) for t in (q, k, v, go))
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    m4 = vis[:, None]
    # what is not visible to anyone is not read: it may hold anything
    seen_q, seen_k = vis.any(2)[:, None, :, None], vis.any(1)[:, None, :, None]
    Q, GO = torch.where(seen_q, Q, torch.zeros_like(Q)), torch.where(seen_q, GO, torch.zeros_like(GO))
    K, V = torch.where(seen_k, K, torch.zeros_like(K)), torch.where(seen_k, V, torch.zeros_like(V))
    s = Q @ K.transpose(2, 3) * scale
    s = s.masked_fill(~m4, -math.inf)
    mx = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(mx), torch.zeros_like(mx), mx)).masked_fill(~m4, 0.0)
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    lse = (mx + l.log())[..., 0]
    o = p @ V
    dp = GO @ V.transpose(2, 3)
    delta = (GO * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    dq, dk, dv = ds @ K, ds.transpose(2, 3) @ Q, p.transpose(2, 3) @ GO
    group = lambda t: t.reshape(B, Hq // G, G, L, -1).sum(2).permute(0, 2, 1, 3)
    return dict(Q=Q, K=K, V=V, GO=GO, p=p, o=o, lse=lse, dp=dp, delta=delta, group=group, n=vis.sum(2)[:, None, :, None].double(),
                nk=vis.sum(1)[:, None, :, None].double(), out=o.permute(0, 2, 1, 3), dq=dq.permute(0, 2, 1, 3), dk=group(dk),
                dv=group(dv))


def _limits(r, dt, D, G, scale):
    e = torch.finfo(dt).eps / 2
    e16 = 0.0 if dt == torch.float32 else e
    ds = ((D + 4) * U * (r["Q"].abs() @ r["K"].abs().transpose(2, 3)) * scale * (r["p"] > 0)).amax(-1, keepdim=True)
    relp = 2 * ds + (r["n"] / 8 + 40) * U + e16 + 4 * U * torch.nan_to_num(r["lse"], posinf=0, neginf=0).abs()[..., None]
    absV, absGO = r["V"].abs(), r["GO"].abs()
    out = relp * (r["p"] @ absV)
    errO = (out + e * r["o"].abs())
    dS = r["p"] * scale * ((relp + e16) * (r["dp"].abs() + r["delta"].abs()) + (2 * D + 8) * U * (absGO @ absV.transpose(2, 3))
                           + (2 * D + 8) * U * (absGO * r["o"].abs()).sum(-1, keepdim=True)
                           + (absGO * errO).sum(-1, keepdim=True))
    absS = r["p"] * scale * (r["dp"] - r["delta"]).abs()
    dq = dS @ r["K"].abs() + (r["n"] / 8 + 8) * U * (absS @ r["K"].abs())
    dk = dS.transpose(2, 3) @ r["Q"].abs() + (r["nk"] * G / 8 + 8) * U * (absS.transpose(2, 3) @ r["Q"].abs())
    dv = (r["p"] * relp).transpose(2, 3) @ absGO + (r["nk"] * G / 8 + 8) * U * (r["p"].transpose(2, 3) @ absGO)
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps + 1e-30
    fin = lambda lim, ref: lim * (1 + e) + e * ref.abs() + tiny
    return (fin(out.permute(0, 2, 1, 3), r["out"]), fin(dq.permute(0, 2, 1, 3), r["dq"]), fin(r["group"](dk), r["dk"]),
            fin(r["group"](dv), r["dv"]))


def _within(name, got, ref, lim):
    err = (got.detach().cpu().double() - ref).abs()
    bad = ~(err <= lim)
    assert not bool(bad.any()), (name, int(bad.sum()), bad.numel(), float((err / lim).max()), bad.nonzero()[0].tolist())


SIZES = [  # B, L, Hq, Hkv, D, window, sinks
    (1, 1, 1, 1, 1, 1, 0), (2, 5, 1, 1, 3, 2, 1), (4, 33, 2, 1, 16, 7, 3), (5, 64, 2, 2, 32, 64, 0), (4, 65, 4, 2, 50, 16, 4),
    (3, 200, 2, 2, 64, 50, 2), (4, 130, 3, 1, 80, 33, 0), (2, 257, 8, 2, 128, 40, 7), (3, 100, 2, 1, 150, 1, 1),
    (2, 96, 1, 1, 256, 31, 17), (2, 300, 6, 2, 24, 1000, 5), (1, 700, 2, 1, 64, 100, 33), (3, 90, 5, 5, 7, 3, 64)]


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,L,Hq,Hkv,D,W,S", SIZES)
def test_window_attention(dev, B, L, Hq, Hkv, D, W, S, dt):
    from deeprec_amd import kernels as Kn
    q, k, v, go, begin, end = _inputs(B, L, Hq, Hkv, D, dt, B + L + D)
    scale = D ** -0.5
    vis = _visible(B, L, W, S, begin, end)
    r = _ref(q, k, v, go, vis, scale)
    lo, lq, lk, lv = _limits(r, dt, D, Hq // Hkv, scale)
    d = lambda t: t.to(dev)
    mask = dict(window=W, sinks=S, begin=d(begin), end=d(end))
    out, lse = Kn.window_attn_forward(d(q), d(k), d(v), **mask)
    _within("out", out, r["out"], lo)
    got = lse.cpu().double()
    none = ~vis.any(2)[:, None].expand(B, Hq, L)
    assert bool((got[none] == -math.inf).all()) and bool(((got - r["lse"]).abs()[~none] < 1e-5 * (1 + r["lse"].abs()[~none])).all())
    grads = Kn.window_attn_backward(d(q), d(k), d(v), out, lse, d(go), **mask)
    for name, x, ref, lim in zip(("dq", "dk", "dv"), grads, (r["dq"], r["dk"], r["dv"]), (lq, lk, lv)):
        assert x.dtype == dt
        _within(name, x, ref, lim)
    again = Kn.window_attn_backward(d(q), d(k), d(v), out, lse, d(go), **mask)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


TOKEN = [(1, 1, 1, 1, 1, 1, 0), (3, 9, 2, 1, 16, 4, 2), (5, 300, 8, 2, 64, 64, 4), (64, 200, 8, 2, 64, 256, 4),
         (2, 4000, 4, 4, 128, 3000, 5), (3, 2500, 16, 1, 50, 5000, 0), (2, 600, 40, 2, 80, 128, 64), (1, 5000, 3, 1, 256, 2048, 1),
         (4, 77, 2, 2, 150, 10, 33), (33, 513, 32, 1, 32, 512, 0)]


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,L,Hq,Hkv,D,W,S", TOKEN)
def test_window_attention_token(dev, B, L, Hq, Hkv, D, W, S, dt):
    from deeprec_amd import kernels as Kn
    _, k, v, _, begin, end = _inputs(B, L, 1, Hkv, D, dt, B + L + D)
    q = torch.randn((B, Hq, D), generator=torch.Generator().manual_seed(L)).to(dt)
    G, scale = Hq // Hkv, D ** -0.5
    lo, hi = begin.long().clamp(0, L)[:, None], end.long().clamp(0, L)[:, None]
    j = torch.arange(L)[None]
    vis = (lo <= j) & (j < hi) & ((hi - 1 - j < W) | (j - lo < S))                      # [B, L]
    Q, K, V = q.double(), k.double().repeat_interleave(G, 2), v.double().repeat_interleave(G, 2)
    s = torch.einsum("bhd,blhd->bhl", Q, K) * scale
    s = s.masked_fill(~vis[:, None], -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
    ref = torch.einsum("bhl,blhd->bhd", p, V)
    e = torch.finfo(dt).eps / 2
    ds = ((D + 4) * U * torch.einsum("bhd,blhd->bhl", Q.abs(), K.abs()) * scale * (p > 0)).amax(-1)
    n = vis.sum(1).double()[:, None]
    lim = (2 * ds + (n / 8 + 40) * U + (0 if dt == torch.float32 else e))[..., None] * torch.einsum("bhl,blhd->bhd", p, V.abs())
    lim = lim * (1 + e) + e * ref.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps + 1e-30
    # positions outside the history hold anything
    out_of = ~((lo <= j) & (j < hi))
    k[out_of], v[out_of] = math.nan, math.inf
    out = Kn.window_attn_token(q.to(dev), k.to(dev), v.to(dev), W, S, begin=begin.to(dev), end=end.to(dev))
    assert out.dtype == dt
    _within("out", out, ref, lim)


@gpu
def test_padding_holds_anything(dev):
    """NaN and infinity outside [begin, end) of q, k, v and the gradient reach no output."""
    from deeprec_amd import kernels as Kn
    for dt in DTYPES:
        q, k, v, go, begin, end = (t.to(dev) for t in _inputs(5, 90, 4, 2, 64, dt, 3))
        args = dict(window=20, sinks=3, begin=begin, end=end)
        out, lse = Kn.window_attn_forward(q, k, v, **args)
        grads = Kn.window_attn_backward(q, k, v, out, lse, go, **args)
        pos = torch.arange(90, device=dev)[None]
        pad = (pos < begin.clamp(0, 90)[:, None]) | (pos >= end.clamp(0, 90)[:, None])
        for t, x in ((q, math.nan), (k, math.inf), (v, math.nan), (go, -math.inf)):
            t[pad] = x
        o2, l2 = Kn.window_attn_forward(q, k, v, **args)
        assert torch.equal(out, o2) and torch.equal(lse, l2) and not bool(out[pad].any())
        for a, b in zip(grads, Kn.window_attn_backward(q, k, v, o2, l2, go, **args)):
            assert torch.equal(a, b) and not bool(a[pad].any())


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 50, 24])
def test_strides(dev, D, dt):
    """Slices of a packed projection, heads before positions, an offset that leaves the 16-byte grid, shared key heads."""
    from deeprec_amd import kernels as Kn
    B, L, H = 3, 70, 2
    packed = torch.randn((B, L, 3, H, D), device=dev).to(dt)
    q, k, v = packed.unbind(2)
    ref = Kn.window_attn_forward(q.contiguous(), k.contiguous(), v.contiguous(), 9, 2)
    go = torch.randn((B, L, H, D), device=dev).to(dt)
    gref = Kn.window_attn_backward(q.contiguous(), k.contiguous(), v.contiguous(), *ref, go, 9, 2)

    def same(q, k, v):
        o = Kn.window_attn_forward(q, k, v, 9, 2)
        assert all(torch.equal(a, b) for a, b in zip(o, ref))
        assert all(torch.equal(a, b) for a, b in zip(Kn.window_attn_backward(q, k, v, *o, go, 9, 2), gref))
        t = Kn.window_attn_token(q[:, -1], k, v, 9, 2)
        assert torch.equal(t, Kn.window_attn_token(q[:, -1].contiguous(), k.contiguous(), v.contiguous(), 9, 2))
    same(q, k, v)
    same(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)))
    off = [torch.cat((t.reshape(-1)[:1], t.reshape(-1)))[1:].view(t.shape) for t in (q, k, v)]
    same(*off)
    one = k[:, :, :1]                                                        # one key head for both, stride-0 batch
    kk = one[:1].expand(B, L, 1, D)
    a = Kn.window_attn_forward(q, kk, kk, 9, 2)[0]
    b = Kn.window_attn_forward(q, kk.expand(B, L, H, D), kk.expand(B, L, H, D), 9, 2)[0]
    assert torch.equal(a, b)


@gpu
def test_gradients_against_differences(dev):
    from deeprec_amd import kernels as Kn
    q, k, v, go, begin, end = _inputs(1, 40, 2, 1, 8, torch.float32, 11)
    vis = _visible(1, 40, 6, 2, begin, end)

    def loss(q, k, v):
        return float((_ref(q, k, v, go, vis, 0.3)["out"] * go.double()).sum())
    d = lambda t: t.to(dev)
    out, lse = Kn.window_attn_forward(d(q), d(k), d(v), 6, 2, scale=0.3)
    grads = Kn.window_attn_backward(d(q), d(k), d(v), out, lse, d(go), 6, 2, scale=0.3)
    for which in range(3):
        for at in ((0, 0, 0, 0), (0, 1, 0, 3), (0, 17, 0, 7), (0, 39, 0, 1)):
            vals = []
            for sign in (1, -1):
                t = [x.double().clone() for x in (q, k, v)]
                t[which][at] += sign * 1e-5
                vals.append(loss(*t))
            num = (vals[0] - vals[1]) / 2e-5
            assert abs(num - float(grads[which][at])) < 2e-5 * (1 + abs(num)), (which, at)


@gpu
def test_token_equals_last_query(dev):
    """The serving form of the last position agrees with the training form to rounding."""
    from deeprec_amd import kernels as Kn
    q, k, v, _, begin, end = (t.to(dev) for t in _inputs(6, 150, 8, 2, 64, torch.float32, 4))
    out, _ = Kn.window_attn_forward(q, k, v, 40, 3, begin=begin, end=end)
    last = (end.long().clamp(0, 150) - 1)
    rows = torch.arange(6, device=dev)
    tok = Kn.window_attn_token(q[rows, last.clamp_min(0)], k, v, 40, 3, begin=begin, end=end)
    some = end.long().clamp(0, 150) > begin.long().clamp(0, 150)
    want = torch.where(some[:, None, None], out[rows, last.clamp_min(0)], torch.zeros_like(tok))
    assert float((tok - want).abs().max()) < 1e-5


@gpu
def test_window_attention_graph_and_streams(dev):
    from deeprec_amd import kernels as Kn
    q, k, v, go, begin, end = (t.to(dev) for t in _inputs(4, 300, 4, 2, 64, torch.bfloat16, 9))
    args = dict(window=64, sinks=4, begin=begin, end=end)

    def call():
        o, s = Kn.window_attn_forward(q, k, v, **args)
        return (o, s) + Kn.window_attn_backward(q, k, v, o, s, go, **args) + (Kn.window_attn_token(q[:, 0], k, v, **args),)
    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                                       # two graphs over the same tensors
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = call()
        graphs.append((gr, res))
    side = torch.cuda.Stream()
    for _ in range(3):
        for t in (q, k, v, go):
            t.normal_()
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            mine = call()
        torch.cuda.synchronize()
        for a, b, c in zip(graphs[0][1], graphs[1][1], mine):
            assert torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_window_attention_refusals(dev):
    from deeprec_amd import kernels as Kn
    from deeprec_amd._abi import DeepRecError
    q, k = torch.zeros((2, 8, 4, 16), device=dev), torch.zeros((2, 8, 2, 16), device=dev)
    Kn.window_attn_forward(q, k, k, 3)
    for bad in (dict(window=0), dict(window=3, sinks=65), dict(window=3, sinks=-1)):
        with pytest.raises(ValueError, match="window must"):
            Kn.window_attn_forward(q, k, k, **bad)
    with pytest.raises(ValueError, match="no multiple"):
        Kn.window_attn_forward(q[:, :, :3], k, k, 3)
    with pytest.raises(ValueError, match="same length"):
        Kn.window_attn_forward(q, k[:, :7], k[:, :7], 3)
    with pytest.raises(ValueError, match="last dim"):
        Kn.window_attn_forward(q.transpose(1, 3), k.transpose(1, 3), k.transpose(1, 3), 3)
    with pytest.raises(ValueError, match="head dim"):
        Kn.window_attn_forward(torch.zeros((1, 2, 1, 257), device=dev), torch.zeros((1, 2, 1, 257), device=dev),
                               torch.zeros((1, 2, 1, 257), device=dev), 3)
    with pytest.raises(TypeError):
        Kn.window_attn_forward(q, k.half(), k.half(), 3)
    with pytest.raises(ValueError, match="begin"):
        Kn.window_attn_forward(q, k, k, 3, begin=torch.zeros(3, dtype=torch.int32, device=dev))
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(DeepRecError, match="scale"):
            Kn.window_attn_forward(q, k, k, 3, scale=bad)
    out, lse = Kn.window_attn_forward(q, k, k, 3)
    with pytest.raises(ValueError):
        Kn.window_attn_backward(q, k, k, out[:1], lse, out, 3)
    e = Kn.window_attn_forward(q[:0], k[:0], k[:0], 3)
    assert e[0].shape == (0, 8, 4, 16) and Kn.window_attn_token(q[:0, 0], k[:0], k[:0], 3).shape == (0, 4, 16)


def test_window_attention_refusals_cpu():
    import ctypes as C
    from deeprec_amd import _abi
    lib = _abi.lib()
    p, s = C.c_void_p(4096), (C.c_int64 * 3)(64, 16, 8)
    fwd = [p, s, p, s, p, s, 2, 4, 2, 1, 8, 0, 3, 1, 0.5, None, None, p, p, None]

    def call(i, v):
        return lib.dr_window_attn_forward(*[v if j == i else y for j, y in enumerate(fwd)])
    for i, v in ((0, None), (1, None), (6, -1), (7, 0), (9, 3), (9, 2 ** 17), (10, 257), (10, 0), (11, 4), (12, 0), (13, 65), (14, 0.0),
                 (17, None), (18, None), (0, C.c_void_p(4098))):
        assert call(i, v) == -1, (i, v)
    assert call(6, 0) == 0
    assert lib.dr_window_attn_backward_bytes(2, 4, 3, 2, 8, 3, 1) == -1
    assert lib.dr_window_attn_token(p, s, p, s, p, s, 1, 9000, 2, 1, 8, 0, 9000, 1, 0.5, None, None, p, p, 16, None) == -2


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("size", [2.0 ** -13, 2.0 ** 10])
def test_gradient_scale(dev, dt, size):
    """Gradients far from 1 (none or a large loss scale): a power of two in, the same power of two out, to the type's range.
    With dO = size * (exact in every type), dQ, dK, dV are size times those of dO up to rounding where neither is subnormal;
    compared with the 64-bit restatement at the usual limits, and 2^-24 (half the smallest subnormal) for fp16."""
    from deeprec_amd import kernels as Kn
    B, L, Hq, Hkv, D, W, S = 2, 150, 4, 2, 64, 40, 3
    q, k, v, go, begin, end = _inputs(B, L, Hq, Hkv, D, dt, 21)
    go = (go.float() * size).to(dt)
    scale = D ** -0.5
    r = _ref(q, k, v, go, _visible(B, L, W, S, begin, end), scale)
    _, lq, lk, lv = _limits(r, dt, D, Hq // Hkv, scale)
    d = lambda t: t.to(dev)
    mask = dict(window=W, sinks=S, begin=d(begin), end=d(end))
    out, lse = Kn.window_attn_forward(d(q), d(k), d(v), **mask)
    for name, x, ref, lim in zip(("dq", "dk", "dv"), Kn.window_attn_backward(d(q), d(k), d(v), out, lse, d(go), **mask),
                                 (r["dq"], r["dk"], r["dv"]), (lq, lk, lv)):
        _within(name, x, ref, lim + (2.0 ** -24 if dt == torch.float16 else 0.0))


@gpu
def test_nan_is_not_an_empty_row(dev):
    """A NaN that a query sees comes out of every form as NaN: only a query without keys gives zeros and lse -inf."""
    from deeprec_amd import kernels as Kn
    q, k, v, go, _, _ = (t.to(dev) for t in _inputs(2, 40, 2, 1, 32, torch.float32, 4))
    k[0] = math.nan
    end = torch.tensor([40, 0], dtype=torch.int32, device=dev)
    out, lse = Kn.window_attn_forward(q, k, v, 8, 2, end=end)
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    assert not bool(out[1].any()) and bool((lse[1] == -math.inf).all())
    one = Kn.window_attn_token(q[:, 0], k, v, 8, 2, end=end)
    assert bool(one[0].isnan().all()) and not bool(one[1].any())
    many = Kn.window_attn_token(q[:1, 0], k[:1, :1].expand(1, 2000, 1, 32), v[:1, :1].expand(1, 2000, 1, 32), 2000)  # split keys
    assert bool(many.isnan().all())


@gpu
def test_scale_range(dev):
    from deeprec_amd import kernels as Kn
    from deeprec_amd._abi import DeepRecError
    q, k, v, _, _, _ = (t.to(dev) for t in _inputs(1, 40, 1, 1, 32, torch.float32, 4))
    for bad in (1e-39, 3e38):
        with pytest.raises(DeepRecError, match="scale"):
            Kn.window_attn_forward(q, k, v, 8, scale=bad)
    out, _ = Kn.window_attn_forward(q, k, v, 8, scale=1e-30)                 # every visible key weighs the same
    vd = v[0, :, 0].double().cpu()
    want = torch.stack([vd[max(0, i - 7):i + 1].mean(0) for i in range(40)])
    assert float((out[0, :, 0].cpu().double() - want).abs().max()) < 1e-5    # 8 terms of about 1, sums in fp32


def test_window_attention_refuses_a_grid_too_large_cpu():
    import ctypes as C
    from deeprec_amd import _abi
    lib = _abi.lib()
    p, s = C.c_void_p(4096), (C.c_int64 * 3)(64, 16, 8)
    assert lib.dr_window_attn_forward(p, s, p, s, p, s, 2 ** 24, 4, 1, 1, 8, 0, 3, 1, 0.5, None, None, p, p, None) == -1
    assert lib.dr_item_logprobs_forward(p, 2 ** 27, 8, 8, 0, None, 32, 0, 0, None, p, p, None, None, None, 0, None) == -1
    for bad in (1e-39, 3e38):
        assert lib.dr_window_attn_forward(p, s, p, s, p, s, 2, 4, 2, 1, 8, 0, 3, 1, bad, None, None, p, p, None) == -1


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,L,Hq,Hkv,D", [(1, 20000, 2, 1, 24), (1, 33000, 1, 1, 64), (2, 900, 20, 1, 128), (1, 700, 4, 2, 200)])
def test_token_over_many_splits(dev, B, L, Hq, Hkv, D, dt):
    """Long caches, whose keys are shared out over up to 256 workgroups (the first two), against 64 bits."""
    from deeprec_amd import kernels as Kn
    g = torch.Generator().manual_seed(L)
    r = lambda *s: torch.randn(s, generator=g).to(dt)
    q, k, v = r(B, Hq, D), r(B, L, Hkv, D), r(B, L, Hkv, D)
    end = torch.full((B,), L - 3, dtype=torch.int32)
    out = Kn.window_attn_token(q.to(dev), k.to(dev), v.to(dev), L, end=end.to(dev))
    K, V = (t[:, :L - 3].double().repeat_interleave(Hq // Hkv, 2) for t in (k, v))
    scale = D ** -0.5
    s = torch.einsum("bhd,blhd->bhl", q.double(), K) * scale
    p = torch.softmax(s, -1)
    ref = torch.einsum("bhl,blhd->bhd", p, V)
    e = torch.finfo(dt).eps / 2
    ds = ((D + 4) * U * torch.einsum("bhd,blhd->bhl", q.double().abs(), K.abs()) * scale).amax(-1, keepdim=True)
    lse = torch.logsumexp(s, -1, keepdim=True).abs()
    rel = 2 * ds + (L / 8 + 40) * U + (0.0 if dt == torch.float32 else e) + 4 * U * lse
    lim = rel * torch.einsum("bhl,blhd->bhd", p, V.abs()) * (1 + e) + e * ref.abs() + 1e-30 + torch.finfo(dt).smallest_normal * e
    _within("out", out, ref, lim)


@gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128])
def test_many_rows_with_shared_heads(dev, D, dt):
    """Enough rows that the forward takes two heads of a group at a time (full tiles; B is cut for the 64-bit restatement,
    whose rows are compared one by one)."""
    from deeprec_amd import kernels as Kn
    B, L, Hq, Hkv, W, S = 130, 200, 4, 1, 40, 3
    q, k, v, go, begin, end = _inputs(B, L, Hq, Hkv, D, dt, D)
    d = lambda t: t.to(dev)
    mask = dict(window=W, sinks=S, begin=d(begin), end=d(end))
    out, lse = Kn.window_attn_forward(d(q), d(k), d(v), **mask)
    few = torch.tensor([0, 1, 2, 3, 70, 129])
    vis = _visible(len(few), L, W, S, begin[few], end[few])
    r = _ref(q[few], k[few], v[few], go[few], vis, D ** -0.5)
    _within("out", out.cpu()[few], r["out"], _limits(r, dt, D, Hq // Hkv, D ** -0.5)[0])
    got, none = lse.cpu().double()[few], ~vis.any(2)[:, None].expand(len(few), Hq, L)
    assert bool((got[none] == -math.inf).all()) and bool(((got - r["lse"]).abs()[~none] < 1e-5 * (1 + r["lse"].abs()[~none])).all())
    # the other rows: as each row alone (one head at a time) gives them, but for the order of no sum
    for b in (5, 64, 128):
        alone, ls = Kn.window_attn_forward(d(q[b:b + 1]), d(k[b:b + 1]), d(v[b:b + 1]), window=W, sinks=S, begin=d(begin[b:b + 1]),
                                           end=d(end[b:b + 1]))
        assert torch.equal(alone[0], out[b]) and torch.equal(ls[0], lse[b])
