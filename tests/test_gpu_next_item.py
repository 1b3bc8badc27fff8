"""The long-history next-item path as it is used: scaled embedding, windowed attention, log-probabilities over the catalog,
gradients, clipping, update -- and serving one token at a time over a cache; and the optimizer's clip_norm in the models.

Tolerances (2-norm, relative): a chain of fp32 sums of D, L and V terms errs by at most u (n + 16) per stage; softmax and
the products between the stages amplify a relative error by a small factor, taken as 8 in all: 8 (D + L + V + 40) 2^-24.
bf16: some ten roundings to 8 bits on the way of a gradient, amplified by 2: 20 x 2^-8."""
import math

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
B, L, V, D, Hq, Hkv, Dh, W, S = 6, 60, 500, 64, 2, 1, 32, 12, 2
NAMES = ["weight", "Wq", "Wk", "Wv", "Wo"]


def _setup(dt):
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(s, generator=g)
    p = dict(weight=r(V, D) * 0.125, Wq=r(D, Hq * Dh) * 0.2, Wk=r(D, Hkv * Dh) * 0.2, Wv=r(D, Hkv * Dh) * 0.125,
             Wo=r(Hq * Dh, D) * 0.125)
    p = {n: t.to(dt) for n, t in p.items()}
    length = torch.tensor([L, 1, 0, 17, L, 33])
    begin = (L - length).to(torch.int32)
    seq = torch.randint(1, V, (B, L), generator=g)
    seq[torch.arange(L)[None] < begin[:, None]] = 0                          # item 0 pads on the left
    tgt = torch.randint(1, V, (B, 2), generator=g)
    tgt[2] = -1                                                              # the empty history has no target
    return p, begin, seq.to(torch.int32), tgt.to(torch.int32)


def _ref_loss(p, begin, seq, tgt):
    """The same loss from elementary 64-bit operations under autograd."""
    w = p["weight"]
    x = w[seq.long()] * math.sqrt(D)
    x = torch.where((seq == 0)[..., None], x.detach(), x)                    # the padding row gets no gradient from here
    q = (x @ p["Wq"]).view(B, L, Hq, Dh).transpose(1, 2)
    k, v = ((x @ p[n]).view(B, L, Hkv, Dh).transpose(1, 2).repeat_interleave(Hq // Hkv, 1) for n in ("Wk", "Wv"))
    i, j, lo = torch.arange(L)[:, None], torch.arange(L)[None], begin.long()[:, None, None]
    vis = ((j <= i)[None] & (j >= lo) & ((i - j < W)[None] | (j - lo < S)))[:, None]
    s = (q @ k.transpose(2, 3) * Dh ** -0.5).masked_fill(~vis, -1e300)
    o = torch.where(vis.any(-1, keepdim=True), torch.softmax(s, -1) @ v, torch.zeros((), dtype=s.dtype))
    h = o.transpose(1, 2).reshape(B, L, Hq * Dh)[:, -1] @ p["Wo"]
    lp = torch.log_softmax(h @ w.t(), -1)
    logp = torch.where(tgt >= 0, lp.gather(1, tgt.long().clamp_min(0)), torch.zeros((), dtype=lp.dtype))
    return -(logp.sum() + 0.1 * torch.special.entr(lp.exp()).sum()) / B


def _hidden(p, begin, seq):
    from deeprec_amd.models import _common as M
    x = M.embedding(p["weight"], seq, math.sqrt(D), padding_idx=0)
    x2 = x.view(B * L, D)
    q, k, v = ((x2 @ p[n]).view(B, L, -1, Dh) for n in ("Wq", "Wk", "Wv"))
    o = M.window_attention(q, k, v, W, S, begin=begin)
    return o.reshape(B, L, Hq * Dh)[:, -1] @ p["Wo"], q, k, v


def _loss(p, begin, seq, tgt):
    from deeprec_amd.models import _common as M
    h = _hidden(p, begin, seq)[0]
    r = M.item_logprobs(h @ p["weight"].t(), tgt, k=5)
    return -(r.logp.sum() + 0.1 * r.entropy.sum()) / B, r


@gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_training_step(dev, dt):
    from deeprec_amd import kernels as K
    p, begin, seq, tgt = _setup(dt)
    ref = {n: t.double().requires_grad_(True) for n, t in p.items()}
    ref_loss = _ref_loss(ref, begin, seq, tgt)
    ref_loss.backward()
    w = {n: t.to(dev).requires_grad_(True) for n, t in p.items()}
    loss, r = _loss(w, begin.to(dev), seq.to(dev), tgt.to(dev))
    loss.backward()
    tol = 8 * (D + L + V + 40) * 2.0 ** -24 if dt == torch.float32 else 20 * 2.0 ** -8
    assert abs(float(loss) - float(ref_loss)) <= tol * abs(float(ref_loss))
    for n in NAMES:
        g, x = w[n].grad.cpu().double(), ref[n].grad
        assert float((g - x).norm()) <= tol * float(x.norm()), (n, float((g - x).norm() / x.norm()))
    total = math.sqrt(sum(float(x.grad.norm()) ** 2 for x in ref.values()))
    grads, norm = K.clip_by_global_norm([w[n].grad for n in NAMES], total / 2)
    assert abs(float(norm) - total) <= tol * total
    assert abs(float(K.global_norm(grads)) - total / 2) <= (tol + 2.0 ** -7 * (dt != torch.float32)) * total
    with torch.no_grad():
        for n, g in zip(NAMES, grads):
            w[n] -= 0.1 * g
    assert r.top_idx.shape == (B, 5) and not r.top_logp.requires_grad


@gpu
def test_entropy_alone_and_no_gradient(dev):
    from deeprec_amd.models import _common as M
    x = torch.randn((4, 90), device=dev, requires_grad=True)
    t = torch.zeros(4, dtype=torch.int64, device=dev)
    r = M.item_logprobs(x, t)
    r.entropy.sum().backward()
    y = x.detach().double().requires_grad_(True)
    torch.special.entr(torch.softmax(y, -1)).sum().backward()
    assert float((x.grad.double() - y.grad).abs().max()) < 1e-6
    with torch.no_grad():
        assert torch.equal(M.item_logprobs(x, t).logp, r.logp)


@gpu
def test_serving_equals_training_form(dev):
    """Prompt once, then token by token over the cache: the last position's items and log-probabilities agree."""
    from deeprec_amd import kernels as K
    p, begin, seq, _ = _setup(torch.float32)
    p, begin, seq = {n: t.to(dev) for n, t in p.items()}, begin.to(dev), seq.to(dev)
    h, q, k, v = _hidden(p, begin, seq)
    want = K.item_logprobs_forward(h @ p["weight"].t(), K=5)
    kc, vc = torch.full_like(k, math.nan), torch.full_like(v, math.nan)      # a cache whose tail is not filled yet
    for t in range(L - 3, L):
        kc[:, :t + 1], vc[:, :t + 1] = k[:, :t + 1], v[:, :t + 1]
        end = torch.full((B,), t + 1, dtype=torch.int32, device=dev)
        o = K.window_attn_token(q[:, t], kc, vc, W, S, begin=begin, end=end)
    got = K.item_logprobs_forward(o.reshape(B, -1) @ p["Wo"] @ p["weight"].t(), K=5)
    assert torch.equal(got.top_idx[begin < L], want.top_idx[begin < L])
    tol = 8 * (D + L + V + 40) * 2.0 ** -24
    assert float((got.top_logp - want.top_logp).abs().max()) <= tol * float(want.top_logp.abs().max())


def _attrec(clip_norm, dev, seed=5):
    from deeprec_amd.models.seq_rec.AttRec import AttRec
    rng = np.random.default_rng(seed)
    nu, ni, d, l, t, bs = 60, 90, 16, 5, 2, 64
    init = {n: (rng.standard_normal((r, d)) * 0.3).astype(np.float32) for n, r in
            (("P", nu), ("V", nu), ("Q", ni), ("X", ni), ("A", ni))}
    init["W"] = (rng.standard_normal((ni, 2 * d)) * 0.1).astype(np.float32)
    init["b"] = np.zeros(ni, np.float32)
    init["linear_project"] = (rng.standard_normal((d, d)) * 0.3).astype(np.float32)
    m = AttRec(None, nu, ni, batch_size=bs, clip_norm=clip_norm)
    m.build_network(L=l, num_T=t, num_factor=d, init=init)
    i32 = lambda *s, hi: torch.from_numpy(rng.integers(0, hi, s).astype(np.int32)).to(dev)
    return m, [(i32(bs, hi=nu), i32(bs, l, hi=ni), i32(bs, t, hi=ni), i32(bs, t, hi=ni)) for _ in range(4)]


@gpu
def test_model_clip_norm(dev):
    """AttRec(clip_norm): a step equals the step of the unclipped model whose recorded rows and dense gradient were scaled
    by hand to the norm computed in 64 bits; a norm that is never reached changes no bit; hipGraph replay equals eager."""
    a, batches = _attrec(0.05, dev)
    b, _ = _attrec(None, dev)
    for m in (a, b):
        m._zero_dense_grads()
        m._forward_backward(*batches[0])
    tabs = (b.P, b.X, b.Q)
    total = math.sqrt(sum(float(r.double().pow(2).sum()) for t in tabs for _, r in t.pending)
                      + float(b.linear_project.grad.double().pow(2).sum()))
    assert total > 0.1
    c = 0.05 / total
    for t in tabs:
        t.pending = [(i, (r.double() * c).float()) for i, r in t.pending]
    b.linear_project.grad = (b.linear_project.grad.double() * c).float()
    a._apply_step()
    b._apply_step()
    for n in "PXQ":
        x, y = getattr(a, n).w, getattr(b, n).w
        # factor and products rounded once more: 2^-22 of a gradient that Adagrad turns into at most lr (0.05) a step
        assert float((x - y).abs().max()) <= 0.05 * 2.0 ** -20 + 2.0 ** -23 * float(y.abs().max()), n
    far, _ = _attrec(1e9, dev)
    off, _ = _attrec(None, dev)
    eager, _ = _attrec(0.05, dev)
    graphed, _ = _attrec(0.05, dev)
    for bt in batches:
        far.train_op(*bt), off.train_op(*bt), eager.train_op(*bt)
        graphed._step(*bt)
    assert graphed._step.replays >= 2 and graphed._step.capture_error is None
    for n in "PXQ":
        assert torch.equal(getattr(far, n).w, getattr(off, n).w)
        assert torch.equal(getattr(eager, n).w, getattr(graphed, n).w)
        assert not torch.equal(getattr(eager, n).w, getattr(off, n).w)


@gpu
def test_caser_and_prme_accept_clip_norm(dev):
    from deeprec_amd.models.seq_rec.Caser import Caser
    from deeprec_amd.models.seq_rec.PRME import PRME
    g = torch.Generator().manual_seed(1)
    i32 = lambda *s, hi: torch.randint(1, hi, s, generator=g).to(torch.int32).to(dev)
    m = PRME(None, 40, 50, batch_size=16, clip_norm=0.01).build_network(L=1, num_T=1, num_factor=12)
    before = m.Q.w.clone()
    m.train_op(i32(16, hi=40), i32(16, 1, hi=50), i32(16, 1, hi=50), i32(16, 1, hi=50))
    assert not torch.equal(before, m.Q.w) and bool(torch.isfinite(m.Q.w).all())
    m = Caser(None, 40, 50, batch_size=16, clip_norm=0.01)
    m.build_network(L=4, num_T=2, num_factor=16, num_neg=2)
    norm = []
    real = m.optimizer.clip
    m.optimizer.clip = lambda *a: norm.append(real(*a))
    m.train_op(i32(16, hi=40), i32(16, 4, hi=50), i32(16, 2, hi=50), i32(16, 2, hi=50))
    assert len(norm) == 1 and float(norm[0]) > 0


def test_clip_refuses_sharded_tables():
    from deeprec_amd.models._common import Shard, Table, TFOptimizer
    opt = TFOptimizer("sgd", 0.1, clip_norm=1.0)
    with pytest.raises(ValueError, match="sharded"):
        opt.clip([Table(torch.zeros(4, 2), Shard(1, 0, force=True))])
    assert TFOptimizer("sgd", 0.1).clip([]) is None


@gpu
def test_captured_training_step(dev):
    """Forward and backward of the whole path in one hipGraph: every replay equals the eager step on the same values."""
    p, begin, seq, tgt = _setup(torch.float32)
    begin, seq, tgt = begin.to(dev), seq.to(dev), tgt.to(dev)

    def step(w):
        loss, _ = _loss(w, begin, seq, tgt)
        return (loss.detach(),) + torch.autograd.grad(loss, [w[n] for n in NAMES])

    def leaves():
        return {n: t.to(dev).requires_grad_(True) for n, t in p.items()}
    w = leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(w)
    for _ in range(3):
        with torch.no_grad():
            for n in NAMES:
                p[n] = torch.randn(p[n].shape) * 0.125
                w[n].copy_(p[n])
            seq.copy_(seq[:, torch.randperm(L, device=dev)])
        graph.replay()
        eager = step(leaves())
        torch.cuda.synchronize()
        for a, b in zip(res, eager):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6 * float(b.float().abs().max()))   # library products may differ in order


def test_embedding_refuses_a_padding_row_outside_the_table():
    from deeprec_amd.models import _common as M
    for bad in (-1, 5):
        with pytest.raises(ValueError, match="padding_idx"):
            M.embedding(torch.zeros(5, 2), torch.zeros(3, dtype=torch.int32), padding_idx=bad)
