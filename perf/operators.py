"""Plain forms, inputs and sizes of the operators of the long-history next-item path.

The path: item rows looked up and scaled (gradient by sorted ids), causal attention over a window of the history plus
its first few items, log-probabilities of the next items over the whole catalog, and the global norm of all gradients
with clipping.  `run` computes one pass through one operator: in elementary torch operations where `own` is false,
through deeprec_amd.kernels where it is true.  A case is a dict of plain values; `op` names the pass:

  lookup       scaled embedding lookup
  lookup_grad  its gradient: a dense table gradient, duplicate ids summed
  attn         windowed attention, forward (prompts, scoring)
  attn_train   windowed attention, forward and backward
  attn_token   windowed attention of one new token over a cache
  logp         log-probabilities of given items, entropy, the K best items
  logp_train   the same without the list, and its gradient
  clip         global gradient norm over many tensors, clipped copies
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one batch of short sessions (1000 x 5 items, 1683 rows of 150): what a small training step looks up; latency counts
        dict(name="lookup_sessions", op="lookup", dt="f32", rows=1683, d=150, n=5000),
        # 4096 histories of 50 items from a catalog of 10^5, half precision tables
        dict(name="lookup_histories", op="lookup", dt="bf16", rows=100001, d=128, n=204800),
        # the gradient of that lookup: popular items repeat thousands of times, item 0 is the padding
        dict(name="lookup_grad_histories", op="lookup_grad", dt="bf16", rows=100001, d=128, n=204800),
        # a large catalog in fp32, most rows untouched by the batch
        dict(name="lookup_grad_catalog", op="lookup_grad", dt="f32", rows=1000003, d=100, n=131072),
        # serving: 64 users, one new item each, 2048 cached positions of which a window and the first few count
        dict(name="attn_token_serve", op="attn_token", dt="bf16", B=64, L=2048, Hq=8, Hkv=2, D=64, window=256, sinks=4),
        # a training step over histories of 200 items padded on the left, fp32 like the tables
        dict(name="attn_train_sessions", op="attn_train", dt="f32", B=64, L=200, Hq=2, Hkv=2, D=64, window=50, sinks=2),
        # training over long histories, grouped heads, half precision, odd length
        dict(name="attn_train_long", op="attn_train", dt="bf16", B=4, L=2047, Hq=8, Hkv=2, D=128, window=256, sinks=4),
        # serving: 8 users scored over the catalog, the 10 best items wanted
        dict(name="logp_serve", op="logp", dt="bf16", N=8, V=100001, T=1, K=10),
        # training on a catalog of 3707 items, three targets a row, some of them missing, entropy in the loss
        dict(name="logp_train_targets", op="logp_train", dt="f16", N=4096, V=3707, T=3, K=0),
        # evaluation of 4096 histories over 10^5 items, seen items masked, the 10 best wanted: the largest read
        dict(name="logp_evaluate", op="logp", dt="f32", N=4096, V=100000, T=1, K=10),
        # the dense weights of a small tower and its projections: a dozen small gradients
        dict(name="clip_tower", op="clip", kind="tower", scale=1, dt="f32"),
        # a whole step: recorded gradient rows of histories beside fifty odd-sized weights of mixed types
        dict(name="clip_step", op="clip", kind="step", scale=12, dt="mixed"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "attn", "attn_train", "attn_token", "logp", "logp_train", "clip"])
    dt = rng.choice(["f32", "f16", "bf16"])
    if op in ("lookup", "lookup_grad"):
        d = _log(rng, 8, 256)
        return dict(op=op, dt=dt, rows=_log(rng, 500, 1000000), d=d, n=_log(rng, 64, 200000))
    if op in ("attn", "attn_train"):
        Hkv = rng.choice([1, 2, 4])
        G = rng.choice([1, 2, 4])
        L = _log(rng, 1, 2000)
        most = max(1, min(128, (4 * 8 * 2047 * 2047) // (L * L * Hkv * G)))
        return dict(op=op, dt=dt, B=_log(rng, 1, most), L=L, Hq=Hkv * G, Hkv=Hkv, D=rng.choice([16, 32, 50, 64, 80, 128]),
                    window=_log(rng, 1, 256), sinks=rng.choice([0, 1, 4, 7]))
    if op == "attn_token":
        Hkv = rng.choice([1, 2, 4])
        return dict(op=op, dt=dt, B=_log(rng, 1, 128), L=_log(rng, 1, 4096), Hq=Hkv * rng.choice([1, 2, 4, 8]), Hkv=Hkv,
                    D=rng.choice([16, 32, 50, 64, 80, 128]), window=_log(rng, 1, 2048), sinks=rng.choice([0, 1, 4, 7]))
    if op in ("logp", "logp_train"):
        V = _log(rng, 100, 100000)
        N = _log(rng, 1, min(4096, 200000000 // V))
        return dict(op=op, dt=dt, N=N, V=V, T=rng.choice([1, 2, 5]), K=0 if op == "logp_train" else min(V, _log(rng, 1, 50)))
    return dict(op=op, kind=rng.choice(["tower", "step"]), scale=_log(rng, 1, 12), dt=rng.choice(["f32", "mixed"]))


def _clip_shapes(case):
    """Shapes and types of the gradients of one step; odd sizes, an empty tensor, vectors beside matrices."""
    s, mixed = case["scale"], case["dt"] == "mixed"
    other = ["bf16", "f32", "f16"] if mixed else ["f32"]
    if case["kind"] == "tower":
        dims = [128, 128, 80, 40, 20, 10]
        shapes = [(a * s, b) for a, b in zip(dims[:-1], dims[1:])] + [(b,) for b in dims[1:]] + [(150, 150), (0,)]
        return [(x, other[i % len(other)]) for i, x in enumerate(shapes)]
    rows = [((17066 * s, 128), "f32"), ((341 * s, 128), "f32"), ((2047 * s, 256), "f32"), ((2047 * s,), "f32")]
    rest = [((37 * s + 13 * i, 64 + i), other[i % len(other)]) for i in range(50)]
    return rows + rest


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 1000003 + 12345)
    op = case["op"]

    def normal(*shape, dt=None, std=1.0):
        return (torch.randn(shape, generator=g, device=dev) * std).to(DT[dt or case["dt"]])

    if op in ("lookup", "lookup_grad"):
        rows, d, n = case["rows"], case["d"], case["n"]
        ids = (torch.rand(n, generator=g, device=dev).double() ** 4 * rows).long().clamp_(0, rows - 1).to(torch.int32)
        st = dict(op=op, ids=ids, rows=rows, scale=math.sqrt(d))
        if op == "lookup":
            st["table"] = normal(rows, d, std=0.05)
        else:
            st["gout"] = normal(n, d, std=0.01)
        return st
    if op in ("attn", "attn_train", "attn_token"):
        B, L, Hq, Hkv, D = case["B"], case["L"], case["Hq"], case["Hkv"], case["D"]
        st = dict(op=op, window=case["window"], sinks=case["sinks"])
        # histories of very different lengths, padded on the left as the loaders do; one in eight is empty
        length = (torch.rand(B, generator=g, device=dev) * (L + 1)).long().clamp_(0, L)
        length = torch.where(torch.rand(B, generator=g, device=dev) < 0.5, torch.full_like(length, L), length)
        length = torch.where(torch.rand(B, generator=g, device=dev) < 0.125, torch.zeros_like(length), length)
        if op == "attn_token":
            # a cache is filled from its start
            st["begin"], st["end"] = torch.zeros_like(length).to(torch.int32), length.to(torch.int32)
            st["q"] = normal(B, Hq, D, std=1.5)
        else:
            st["begin"], st["end"] = (L - length).to(torch.int32), torch.full_like(length, L).to(torch.int32)
            st["q"] = normal(B, L, Hq, D, std=1.5)
        st["k"], st["v"] = normal(B, L, Hkv, D), normal(B, L, Hkv, D)
        if op == "attn_train":
            st["gout"] = normal(B, L, Hq, D)
        return st
    if op in ("logp", "logp_train"):
        N, V, T = case["N"], case["V"], case["T"]
        x = torch.randn((N, V), generator=g, device=dev).mul_(2.0)
        x.masked_fill_(torch.rand((N, V), generator=g, device=dev) < 0.02, -math.inf)       # seen items
        tgt = torch.randint(0, V, (N, T), generator=g, device=dev)
        x.scatter_(1, tgt, 4.0)
        tgt = tgt.masked_fill(torch.rand((N, T), generator=g, device=dev) < 0.1, -1)        # missing targets
        st = dict(op=op, logits=x.to(DT[case["dt"]]), targets=tgt.to(torch.int32), K=case["K"])
        if op == "logp_train":
            st["g_logp"] = torch.randn((N, T), generator=g, device=dev)
            st["g_entropy"] = torch.randn((N,), generator=g, device=dev) * 0.1
        return st
    grads = [normal(*shape, dt=dt, std=0.02) for shape, dt in _clip_shapes(case)]
    return dict(op=op, grads=grads, out=[torch.empty_like(t) for t in grads], clip_norm=1.0)


# ---- plain forms -------------------------------------------------------------------------------------------------
def _lookup(st):
    t = st["table"]
    return (t[st["ids"].long()].float() * st["scale"]).to(t.dtype)


def _lookup_grad(st):
    ids, gout = st["ids"].long(), st["gout"]
    g = gout.float() * st["scale"] * (ids != 0)[:, None]                                    # row 0 is the padding
    out = torch.zeros((st["rows"], gout.shape[1]), dtype=torch.float32, device=gout.device)
    return out.index_add_(0, ids, g).to(gout.dtype)


def _visible(st, L):
    """[B, L, L]: key j is visible to query i."""
    i = torch.arange(L, device=st["q"].device)[None, :, None]
    j = torch.arange(L, device=st["q"].device)[None, None, :]
    b, e = st["begin"].long()[:, None, None], st["end"].long()[:, None, None]
    return (j >= b) & (j <= i) & (i < e) & ((i - j < st["window"]) | (j - b < st["sinks"]))


def _attn_parts(st):
    q, k, v = (st[x].float().permute(0, 2, 1, 3) for x in "qkv")                            # [B, H, L, D]
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    scale = 1.0 / math.sqrt(q.shape[3])
    s = (q @ k.transpose(2, 3)).mul_(scale)
    s.masked_fill_(~_visible(st, q.shape[2])[:, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(-1e30)
    p = (s - m).exp_()
    l = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(l > 0, l, torch.ones_like(l)))
    return q, k, v, p, scale, G


def _attn(st):
    _, _, v, p, _, _ = _attn_parts(st)
    return (p @ v).permute(0, 2, 1, 3).to(st["q"].dtype)


def _attn_train(st):
    dt = st["q"].dtype
    q, k, v, p, scale, G = _attn_parts(st)
    o = p @ v
    go = st["gout"].float().permute(0, 2, 1, 3)
    B, H, L, D = q.shape
    dv = p.transpose(2, 3) @ go
    ds = go @ v.transpose(2, 3)
    ds = ds.sub_((go * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = ds @ k
    dk = ds.transpose(2, 3) @ q
    back = lambda t: t.permute(0, 2, 1, 3).to(dt)
    shared = lambda t: back(t.reshape(B, H // G, G, L, D).sum(2))
    return back(o), back(dq), shared(dk), shared(dv)


def _attn_token(st):
    q, k, v = st["q"], st["k"], st["v"]
    B, L, Hkv, D = k.shape
    W, S, dev = min(st["window"], L), min(st["sinks"], L), q.device
    b, e = st["begin"].long()[:, None], st["end"].long()[:, None]
    first = torch.maximum(b, e - W)                                                         # first key of the window
    sink = b + torch.arange(S, device=dev)[None]
    near = first + torch.arange(W, device=dev)[None]
    at = torch.cat((sink, near), 1)
    ok = torch.cat((sink < first, near < e), 1)
    at = at.clamp_(0, L - 1)
    rows = torch.arange(B, device=dev)[:, None]
    kk, vv = k[rows, at].float().permute(0, 2, 1, 3), v[rows, at].float().permute(0, 2, 1, 3)    # [B, Hkv, n, D]
    qq = q.float().reshape(B, Hkv, -1, D)
    s = (qq @ kk.transpose(2, 3)) * (1.0 / math.sqrt(D))
    s = s.masked_fill(~ok[:, None, None], -math.inf)
    p = (s - s.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    l = p.sum(-1, keepdim=True)
    o = (p @ vv) / torch.where(l > 0, l, torch.ones_like(l))
    return o.reshape(q.shape).to(q.dtype)


def _softmax_parts(x):
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = (x - m).exp()
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    lp = x - lse
    p = e / z
    ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(-1)
    return lse, lp, p, ent


def _logp(st):
    x = st["logits"].float()
    lse, lp, _, ent = _softmax_parts(x)
    t = st["targets"].long()
    at = lp.gather(1, t.clamp_min(0))
    logp = torch.where(t >= 0, at, torch.zeros_like(at))
    if not st["K"]:
        return logp, ent
    # order by value, equal values by the lower index: one 64-bit key of both
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() * (1 << 32)
    key += (1 << 32) - 1 - torch.arange(x.shape[1], device=x.device)
    best = torch.topk(key, st["K"], dim=1).values
    idx = (1 << 32) - 1 - (best & ((1 << 32) - 1))
    top = lp.gather(1, idx)
    idx = torch.where(torch.isinf(top), torch.full_like(idx, -1), idx)
    return logp, ent, idx.to(torch.int32), top


def _logp_train(st):
    x = st["logits"].float()
    _, lp, p, ent = _softmax_parts(x)
    t = st["targets"].long()
    g = st["g_logp"] * (t >= 0)
    at = lp.gather(1, t.clamp_min(0))
    logp = torch.where(t >= 0, at, torch.zeros_like(at))
    dx = torch.where(p > 0, lp, torch.zeros_like(lp)).add_(ent[:, None]).mul_(st["g_entropy"][:, None])
    dx = dx.add_(g.sum(1, keepdim=True)).mul_(p).neg_()
    dx.scatter_add_(1, t.clamp_min(0), g)
    return logp, ent, dx.to(st["logits"].dtype)


def _clip(st):
    flat = torch.cat([t.reshape(-1).float() for t in st["grads"]])
    norm = (flat * flat).sum().sqrt()
    flat = flat * (st["clip_norm"] / norm.clamp_min(st["clip_norm"]))
    parts = flat.split([t.numel() for t in st["grads"]])
    return [p.view(t.shape).to(t.dtype) for p, t in zip(parts, st["grads"])], norm.reshape(1)


_PLAIN = dict(lookup=_lookup, lookup_grad=_lookup_grad, attn=_attn, attn_train=_attn_train, attn_token=_attn_token,
              logp=_logp, logp_train=_logp_train, clip=_clip)


def _run_own(st):
    from deeprec_amd import kernels as K
    op = st["op"]
    if op == "lookup":
        return K.embed_forward(st["table"], st["ids"], scale=st["scale"])
    if op == "lookup_grad":
        return K.embed_backward(st["gout"], st["ids"], st["rows"], scale=st["scale"], padding_idx=0)
    if op in ("attn", "attn_train"):
        mask = dict(window=st["window"], sinks=st["sinks"], begin=st["begin"], end=st["end"])
        out, lse = K.window_attn_forward(st["q"], st["k"], st["v"], **mask)
        if op == "attn":
            return out
        dq, dk, dv = K.window_attn_backward(st["q"], st["k"], st["v"], out, lse, st["gout"], **mask)
        return out, dq, dk, dv
    if op == "attn_token":
        return K.window_attn_token(st["q"], st["k"], st["v"], window=st["window"], sinks=st["sinks"], begin=st["begin"],
                                   end=st["end"])
    if op == "logp":
        r = K.item_logprobs_forward(st["logits"], st["targets"], K=st["K"])
        return (r.logp, r.entropy, r.top_idx, r.top_logp) if st["K"] else (r.logp, r.entropy)
    if op == "logp_train":
        r = K.item_logprobs_forward(st["logits"], st["targets"])
        dx = K.item_logprobs_backward(st["logits"], st["targets"], r.lse, r.entropy, st["g_logp"], st["g_entropy"])
        return r.logp, r.entropy, dx
    out, norm = K.clip_by_global_norm(st["grads"], st["clip_norm"], out=st["out"])
    return out, norm


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    op, es = case["op"], SIZE.get(case["dt"], 4)
    if op == "lookup":
        return dict(bytes=case["n"] * (4 + case["d"] * es) + min(case["n"], case["rows"]) * case["d"] * es,
                    flops=case["n"] * case["d"])
    if op == "lookup_grad":
        return dict(bytes=case["n"] * (4 + case["d"] * es) + case["rows"] * case["d"] * es, flops=2 * case["n"] * case["d"])
    if op in ("attn", "attn_train", "attn_token"):
        B, L, Hq, Hkv, D, W, S = (case[x] for x in ("B", "L", "Hq", "Hkv", "D", "window", "sinks"))
        if op == "attn_token":
            n = min(L, W + S)
            return dict(bytes=B * (2 * Hkv * n + 2 * Hq) * D * es, flops=4 * B * Hq * n * D)
        w = min(W, L)
        pairs = L * w - w * (w - 1) // 2                                                    # the causal window
        pairs += sum(min(S, i + 1 - w) for i in range(w, L)) if S else 0                    # first items behind it
        if op == "attn":
            return dict(bytes=B * L * D * es * (2 * Hq + 2 * Hkv), flops=4 * B * Hq * pairs * D)
        return dict(bytes=B * L * D * es * (4 * Hq + 4 * Hkv), flops=14 * B * Hq * pairs * D)
    if op in ("logp", "logp_train"):
        N, V, T, K = case["N"], case["V"], case["T"], case["K"]
        moved = N * V * es * (2 if op == "logp_train" else 1)
        return dict(bytes=moved + N * (8 * T + 8 * K + 4), flops=(8 if op == "logp_train" else 4) * N * V)
    count = [(math.prod(s), SIZE[t]) for s, t in _clip_shapes(case)]
    return dict(bytes=sum(2 * n * b for n, b in count), flops=sum(3 * n for n, _ in count))


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "lookup":
        return torch.nn.functional.embedding(st["ids"].long(), st["table"].double()) * math.sqrt(case["d"])
    if op == "lookup_grad":
        # by sorting: the sum of a run is a difference of running sums, exact enough in 64 bits
        order = torch.argsort(st["ids"].long(), stable=True)
        sid = st["ids"].long()[order]
        run = torch.cat((torch.zeros((1, case["d"]), dtype=torch.float64, device=sid.device),
                         st["gout"].double()[order].cumsum(0)))
        lo = torch.searchsorted(sid, torch.arange(case["rows"], device=sid.device))
        hi = torch.searchsorted(sid, torch.arange(case["rows"], device=sid.device), right=True)
        out = (run[hi] - run[lo]) * math.sqrt(case["d"])
        out[0] = 0.0
        return out
    if op in ("attn", "attn_train"):
        B, L, Hq, Hkv, D = (case[x] for x in ("B", "L", "Hq", "Hkv", "D"))
        if B * Hq * L * L > 1 << 28:
            return None
        q, k, v = (st[x].double().requires_grad_(op == "attn_train") for x in "qkv")
        pos = torch.arange(L, device=q.device)
        gap = pos[:, None] - pos[None, :]
        rel = pos[None, :] - st["begin"].long()[:, None]                                    # [B, L]: place in the history
        seen = ((gap >= 0)[None] & (rel >= 0)[:, None, :] & ((gap < case["window"])[None] | (rel < case["sinks"])[:, None, :]))
        seen = seen & (pos[None, :] < st["end"].long()[:, None])[:, :, None]
        heads = torch.arange(Hq, device=q.device) // (Hq // Hkv)
        s = torch.matmul(q.transpose(1, 2), k[:, :, heads].permute(0, 2, 3, 1)) / math.sqrt(D)
        bias = torch.zeros(seen.shape, dtype=torch.float64, device=q.device).masked_fill(~seen, -math.inf)
        w = torch.nan_to_num(torch.softmax(s + bias[:, None], -1), nan=0.0) if op == "attn" else \
            torch.softmax(s + torch.where(seen.any(-1, keepdim=True), bias, torch.zeros_like(bias))[:, None], -1) \
            * seen.any(-1)[:, None, :, None]
        o = torch.matmul(w, v[:, :, heads].transpose(1, 2)).transpose(1, 2)
        if op == "attn":
            return o
        return (o.detach(),) + torch.autograd.grad(o, (q, k, v), st["gout"].double())
    if op == "attn_token":
        B, L, Hq, Hkv, D = (case[x] for x in ("B", "L", "Hq", "Hkv", "D"))
        heads = torch.arange(Hq, device=st["q"].device) // (Hq // Hkv)
        s = (st["k"].double()[:, :, heads] * st["q"].double()[:, None]).sum(-1) / math.sqrt(D)   # [B, L, Hq]
        pos, last = torch.arange(L, device=s.device)[None], st["end"].long()[:, None] - 1
        seen = (pos <= last) & ((last - pos < case["window"]) | (pos < case["sinks"]))
        w = torch.nan_to_num(torch.softmax(s.masked_fill(~seen[:, :, None], -math.inf), 1), nan=0.0)
        return (w[..., None] * st["v"].double()[:, :, heads]).sum(1)
    if op in ("logp", "logp_train"):
        if case["N"] * case["V"] > 1 << 29:
            return None
        x = st["logits"].double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        ent = torch.special.entr(p).sum(-1)
        rows = torch.arange(case["N"], device=x.device)[:, None]
        t = st["targets"].long()
        logp = lp[rows, t.clamp_min(0)] * (t >= 0)
        if op == "logp":
            if not case["K"]:
                return logp, ent
            top = torch.topk(lp, case["K"], dim=1).values
            return logp, ent, None, top
        g = st["g_logp"].double() * (t >= 0)
        onehot = torch.zeros_like(x).index_put_((rows.expand_as(t), t.clamp_min(0)), g, accumulate=True)
        dx = onehot - p * g.sum(1, keepdim=True)
        dx -= st["g_entropy"].double()[:, None] * (-torch.special.entr(p) + p * ent[:, None])
        return logp, ent, dx
    total = math.sqrt(sum(float(t.double().pow(2).sum()) for t in st["grads"]))
    c = st["clip_norm"] / max(total, st["clip_norm"])
    return [t.double() * c for t in st["grads"]], torch.full((1,), total, dtype=torch.float64)
