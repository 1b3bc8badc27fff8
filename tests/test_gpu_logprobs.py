"""Catalog log-probabilities, entropy, best items and their gradient against 64-bit restatements.

Tolerances (u = 2^-24, rows of n offered logits of spread R = max - min over those that matter, at most 40 here):
  exp(x - M): the difference is rounded once (u R absolute in the exponent), the product with log2 e and the exponential
  add 2 u R + 2 u; sums of n positive terms in partial sums of at most n/64 + 16 steps.  So every weight and Z are right
  to E = u (4 R + n / 64 + 32) relative, and logp to E + 2 u |logp| + 2 u R absolute, H to E (H + R) + 2 u H.
  Gradient: p (G + gH (log p + H)) to (E + 4 u) of the sum of the absolute terms (with the errors of log p and H times gH
  p), then one rounding to the logits' type."""
import math

import pytest
import torch

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


def _case(N, V, T, dt, seed, idt=torch.int32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((N, V), generator=g) * 2
    x[torch.rand((N, V), generator=g) < 0.05] = -math.inf
    if N > 2:
        x[1] = -math.inf                                                     # nothing offered
        x[2] = -math.inf
        x[2, V // 2] = 1.0                                                   # one item
    if N > 4:
        x[3] = torch.finfo(dt).min                                           # masked by the type's lowest value
        x[3, ::3] = torch.randn(len(x[3, ::3]), generator=g)
        x[4] = 0.5                                                           # nothing but ties
    x = x.to(dt)
    t = torch.randint(0, V, (N, T), generator=g)
    if T > 1:
        t[:, 1] = t[:, 0]                                                    # the same item twice
    t[torch.rand((N, T), generator=g) < 0.2] = -1
    t[0, 0] = V                                                              # out of range
    return x, t.to(idt)


def _ref(x, t):
    x = x.double()
    m = x.amax(-1, keepdim=True)
    none = (m == -math.inf)[:, 0]
    e = torch.exp(x - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    z = e.sum(-1, keepdim=True)
    lp = torch.where(none[:, None], torch.full_like(x, -math.inf), x - m - z.log())
    p = lp.exp()
    H = torch.special.entr(p).sum(-1)
    ok = (t >= 0) & (t < x.shape[1])
    logp = torch.where(ok, lp.gather(1, t.long().clamp(0, x.shape[1] - 1)), torch.zeros((), dtype=torch.float64))
    return lp, p, H, logp, ok, none


def _spread(x):
    f = x.double().clone()
    f[f < -1e4] = math.inf
    lo = f.amin(-1)
    return torch.where(torch.isinf(lo), torch.zeros_like(lo), x.double().amax(-1) - lo).clamp_min(0.0)


def _check_forward(r, x, t, K):
    N, V = x.shape
    lp, p, H, logp, ok, none = _ref(x, t)
    R = _spread(x)
    E = U * (4 * R + V / 64 + 32)
    got = r.logp.cpu().double()
    fin = torch.isfinite(logp)
    assert torch.equal(got[~fin], logp[~fin])
    err = (got - logp).abs()
    lim = (E + 2 * U * R)[:, None] + 2 * U * torch.where(fin, logp, torch.zeros_like(logp)).abs()
    assert bool((err[fin] <= lim[fin]).all()), float((err / lim)[fin].max())
    eh = (r.entropy.cpu().double() - H).abs()
    assert bool((eh <= E * (H + R + 1) + 2 * U * H).all()), float(eh.max())
    lse = r.lse.cpu().double()
    assert torch.equal(lse[:, 0], x.double().amax(-1))
    if K:
        order = torch.argsort(-x.double(), dim=1, stable=True)[:, :K]        # value, then lower index
        want = torch.full((N, K), -1, dtype=torch.int64)
        want[:, :order.shape[1]] = order
        vals = torch.full((N, K), -math.inf, dtype=torch.float64)
        vals[:, :order.shape[1]] = lp.gather(1, order)
        want[torch.isinf(torch.where(want >= 0, x.double().gather(1, want.clamp_min(0)), torch.tensor(-math.inf).double()))] = -1
        assert torch.equal(r.top_idx.cpu().long(), want)
        vals[want < 0] = -math.inf
        g, f = r.top_logp.cpu().double(), want >= 0
        assert bool((g[~f] == -math.inf).all())
        assert bool(((g - vals).abs()[f] <= ((E + 2 * U * R)[:, None] + 2 * U * vals.abs())[f]).all())


SIZES = [(1, 1, 1, 1), (5, 7, 2, 3), (9, 2048, 3, 64), (9, 2049, 1, 10), (6, 5003, 64, 5), (1, 100001, 1, 10), (3, 40000, 2, 64),
         (700, 3707, 3, 1), (1500, 129, 1, 20), (5, 13, 1, 30), (1100, 4101, 2, 16)]


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,T,K", SIZES)
def test_logprobs_forward(dev, N, V, T, K, dt):
    from deeprec_amd import kernels as Kn
    x, t = _case(N, V, T, dt, N + V + T)
    r = Kn.item_logprobs_forward(x.to(dev), t.to(dev), K=K)
    _check_forward(r, x, t, K)
    r2 = Kn.item_logprobs_forward(x.to(dev), t.to(dev).long())               # without a list, 64-bit ids: the same bits
    assert torch.equal(r2.logp, r.logp) and torch.equal(r2.entropy, r.entropy) and r2.top_idx is None
    r3 = Kn.item_logprobs_forward(x.to(dev), K=K)
    assert r3.logp is None and torch.equal(r3.top_idx, r.top_idx) and torch.equal(r3.lse, r.lse)


@gpu
@pytest.mark.parametrize("kind", ["ascending", "descending", "ties", "bf16 steps"])
@pytest.mark.parametrize("V", [1500, 30000])
def test_best_items_hard_orders(dev, kind, V):
    """Orders that keep the candidate lists busy: every element better than all before it, all equal, few values."""
    from deeprec_amd import kernels as Kn
    x = torch.arange(V).float() / V
    if kind == "descending":
        x = x.flip(0)
    elif kind == "ties":
        x = torch.zeros(V)
        x[1::2] = -0.0                                                       # -0 and +0 are equal values
    elif kind == "bf16 steps":
        x = (x * 8).to(torch.bfloat16).float()
    x = x.repeat(5, 1)
    t = torch.zeros((5, 1), dtype=torch.int32)
    for K in (1, 10, 64):
        _check_forward(Kn.item_logprobs_forward(x.to(dev), t.to(dev), K=K), x, t, K)


@gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("N,V,T,K", SIZES)
def test_logprobs_backward(dev, N, V, T, K, dt):
    from deeprec_amd import kernels as Kn
    x, t = _case(N, V, T, dt, 2 * N + V + T)
    g = torch.Generator().manual_seed(N)
    gl, gh = torch.randn((N, T), generator=g), torch.randn(N, generator=g)
    lp, p, H, logp, ok, none = _ref(x, t)
    R = _spread(x)
    E = (U * (4 * R + V / 64 + 32))[:, None]
    lpz = torch.where(p > 0, lp, torch.zeros_like(lp))
    r = Kn.item_logprobs_forward(x.to(dev), t.to(dev))
    for use_h in (True, False):
        h = gh.double()[:, None] if use_h else torch.zeros((N, 1), dtype=torch.float64)
        G = (gl.double() * ok).sum(1, keepdim=True)
        hit = torch.zeros((N, V), dtype=torch.float64).scatter_add_(1, t.long().clamp(0, V - 1), gl.double() * ok)
        hit[none] = 0
        ref = hit - p * (G + h * (lpz + H[:, None]))
        Gabs = (gl.double().abs() * ok).sum(1, keepdim=True)
        A = torch.zeros((N, V), dtype=torch.float64).scatter_add_(1, t.long().clamp(0, V - 1), gl.double().abs() * ok) \
            + p * (Gabs + h.abs() * (lpz.abs() + H[:, None]))
        lim = (2 * E + (T + 8) * U) * A + 2 * h.abs() * p * (E * (H[:, None] + R[:, None] + 2) + 4 * U * R[:, None])
        eps = torch.finfo(dt).eps / 2
        lim = lim * (1 + eps) + eps * ref.abs() + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        dx = Kn.item_logprobs_backward(x.to(dev), t.to(dev), r.lse, r.entropy, gl.to(dev), gh.to(dev) if use_h else None)
        assert dx.dtype == dt and dx.shape == x.shape
        err = (dx.cpu().double() - ref).abs()
        assert bool((err <= lim).all()), (float((err / lim.clamp_min(1e-300)).max()), float(err.max()))


@gpu
def test_logprobs_gradient_against_differences(dev):
    """Central differences of the fp64 restatement's loss, at a few elements."""
    from deeprec_amd import kernels as Kn
    x, t = _case(3, 50, 2, torch.float32, 5)
    x = torch.where(torch.isinf(x), torch.zeros_like(x), x)
    gl, gh = torch.tensor([[1.0, -0.5]] * 3), torch.tensor([0.3, -0.2, 0.1])

    def loss(y):
        _, _, H, logp, _, _ = _ref(y, t)
        return float((logp * gl.double()).sum() + (H * gh.double()).sum())
    r = Kn.item_logprobs_forward(x.to(dev), t.to(dev))
    dx = Kn.item_logprobs_backward(x.to(dev), t.to(dev), r.lse, r.entropy, gl.to(dev), gh.to(dev)).cpu().double()
    for n in range(3):
        for v in [0, 7, 49] + [int(q) for q in t[n] if 0 <= q < 50]:
            d = torch.zeros_like(x.double())
            d[n, v] = 1e-5
            num = (loss(x.double() + d) - loss(x.double() - d)) / 2e-5
            assert abs(num - float(dx[n, v])) < 1e-5, (n, v)


@gpu
def test_logprobs_strided_rows_and_offsets(dev):
    from deeprec_amd import kernels as Kn
    for dt in DTYPES:
        for V in (300, 5001):
            big = torch.randn((6, V + 13), device=dev).to(dt)
            t = torch.randint(0, V, (6, 1), device=dev, dtype=torch.int32)
            gl, gh = torch.randn(6, 1, device=dev), torch.randn(6, device=dev)
            a = Kn.item_logprobs_forward(big[:, 5:5 + V].contiguous(), t, K=7)
            b = Kn.item_logprobs_forward(big[:, 5:5 + V], t, K=7)
            assert torch.equal(a.top_idx, b.top_idx)
            _check_forward(b, big[:, 5:5 + V].cpu(), t.cpu(), 7)
            da = Kn.item_logprobs_backward(big[:, 5:5 + V].contiguous(), t, a.lse, a.entropy, gl, gh)
            db = Kn.item_logprobs_backward(big[:, 5:5 + V], t, a.lse, a.entropy, gl, gh)
            assert torch.equal(da, db)


@gpu
def test_logprobs_nan_and_infinity(dev):
    from deeprec_amd import kernels as Kn
    x = torch.randn((4, 3000), device=dev)
    x[0, 17], x[1, 2999] = math.nan, math.inf
    t = torch.zeros((4, 1), dtype=torch.int32, device=dev)
    r = Kn.item_logprobs_forward(x, t, K=5)
    assert bool(torch.isnan(r.logp[:2]).all()) and bool(torch.isnan(r.entropy[:2]).all())
    assert bool(torch.isfinite(r.logp[2:]).all())
    finite = torch.where(torch.isnan(x[0]), torch.full_like(x[0], -math.inf), x[0])
    assert torch.equal(r.top_idx[0].long(), torch.argsort(-finite, stable=True)[:5]) and int(r.top_idx[1, 0]) == 2999
    dx = Kn.item_logprobs_backward(x, t, r.lse, r.entropy, torch.ones(4, 1, device=dev))
    assert bool(torch.isnan(dx[:2]).all()) and bool(torch.isfinite(dx[2:]).all())


@gpu
def test_logprobs_graph_replay_and_streams(dev):
    from deeprec_amd import kernels as Kn
    x = torch.randn((4, 20000), device=dev)
    t = torch.randint(0, 20000, (4,), device=dev)
    g = torch.ones(4, device=dev)

    def call():
        r = Kn.item_logprobs_forward(x, t, K=8)
        return r, Kn.item_logprobs_backward(x, t, r.lse, r.entropy, g, g)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, dx = call()
    side = torch.cuda.Stream()
    for _ in range(3):
        x.normal_()
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            r2, dx2 = call()
        torch.cuda.synchronize()
        assert torch.equal(dx, dx2) and all(torch.equal(a, b) for a, b in zip(r, r2))


@gpu
def test_logprobs_refusals(dev):
    from deeprec_amd import kernels as Kn
    x = torch.zeros((4, 10), device=dev)
    t = torch.zeros(4, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError, match="K must be"):
        Kn.item_logprobs_forward(x, t, K=65)
    with pytest.raises(ValueError, match="at most"):
        Kn.item_logprobs_forward(x, torch.zeros((4, 65), dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="column stride"):
        Kn.item_logprobs_forward(x.t(), torch.zeros(10, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError, match="overlap"):
        Kn.item_logprobs_forward(x[:1].expand(4, 10), t)
    with pytest.raises(ValueError, match="targets"):
        Kn.item_logprobs_forward(x, t[:3])
    with pytest.raises(TypeError):
        Kn.item_logprobs_forward(x.double(), t)
    r = Kn.item_logprobs_forward(x, t)
    with pytest.raises(ValueError, match="g_logp"):
        Kn.item_logprobs_backward(x, t, r.lse, r.entropy, torch.zeros(3, device=dev))
    e = Kn.item_logprobs_forward(x[:0], t[:0], K=3)
    assert e.logp.shape == (0,) and e.top_idx.shape == (0, 3)


def test_logprobs_refusals_cpu():
    import ctypes as C
    from deeprec_amd import _abi
    lib = _abi.lib()
    p = C.c_void_p(4096)
    n = 1 << 20
    ok = [p, 4, 10, 10, 0, p, 32, 1, 3, p, p, p, p, p, p, n, None]

    def call(i, v):
        return lib.dr_item_logprobs_forward(*[v if j == i else y for j, y in enumerate(ok)])
    for i, v in ((0, None), (1, -1), (2, 0), (3, 9), (4, 3), (5, None), (6, 16), (7, 65), (8, 65), (9, None), (10, None),
                 (11, None), (12, None), (14, C.c_void_p(4100)), (0, C.c_void_p(4098))):
        assert call(i, v) == -1, (i, v)
    wide = [100001 if j in (2, 3) else y for j, y in enumerate(ok)]           # a row split over workgroups needs scratch
    wide[15] = 16
    assert lib.dr_item_logprobs_bytes(4, 100001, 3) > 16 and lib.dr_item_logprobs_forward(*wide) == -2
    assert lib.dr_item_logprobs_bytes(4, 10, 3) == 0
    assert lib.dr_item_logprobs_bytes(-1, 5, 1) < 0 and lib.dr_item_logprobs_bytes(4, 5, 65) < 0
    assert lib.dr_item_logprobs_backward(p, 4, 10, 9, 0, p, 32, 1, p, p, p, p, p, None) == -1
    assert lib.dr_item_logprobs_backward(p, 4, 10, 10, 0, p, 32, 1, p, None, p, p, p, None) == -1
