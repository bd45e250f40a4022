"""Measured cases of the token-transformer operators: attention with a learned relative position bias (`ops.rel_attention`), the gated
residual between two norms (`ops.residual_norm`) and distillation from a teacher's top logits (`ops.topk_distill`).

`own` selects what `run` computes: the plain form in elementary torch operations (32 bits, rounded once at the end), or the calls a
user makes of `passion_amd.ops`."""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _dev():
    return torch.device("cuda:0")


# ------------------------------------------------------------------------------------------------------------------ the cases
def _attn(name, **kw):
    c = dict(name=name, op="attn", b=1, nq=1, nk=1, h=8, hkv=8, d=64, gd=1, gh=1, gw=1, nb=0, dtype="bf16", drop=0.0, bwd=True, q0=0)
    c.update(kw)
    return c


def listed():
    return [
        # one new token against a long sequence: the serving form, latency and cache bandwidth (1D log-spaced buckets, shared heads, padding)
        _attn("attn one token", b=4, nq=1, nk=6000, h=8, hkv=2, gw=8192, nb=32, drop=0.1, bwd=False, q0=5999),
        # the 5^3 tokens of a default 80^3 crop in the f32 parity mode, training step
        _attn("attn 5^3 f32", b=1, nq=125, nk=125, gd=5, gh=5, gw=5, dtype="f32"),
        # intra-modal attention of a 128^3 patch: four modalities as the batch, 8^3 tokens, one table row per offset
        _attn("attn 8^3 x 4", b=4, nq=512, nk=512, gd=8, gh=8, gw=8),
        # inter-modal attention: four modalities' tokens in one sequence, missing modalities masked
        _attn("attn 4 x 8^3 masked", b=4, nq=2048, nk=2048, gd=8, gh=8, gw=8, drop=0.3),
        # a long 1D sequence with grouped wide heads, ragged length, training step
        _attn("attn long 1D", b=1, nq=8000, nk=8000, h=8, hkv=4, d=128, gw=8000, nb=32),
        # few tokens in flight: the residual + norm between two blocks while answering
        dict(name="norm tokens", op="norm", b=4, n=1, c=512, kind="layer", tx="f32", th="bf16", gate="sample", scale=True, bwd=False),
        # the token width of the flagship model, training step, f32 residual stream and bf16 blocks
        dict(name="norm 2048 x 512", op="norm", b=1, n=2048, c=512, kind="layer", tx="f32", th="bf16", gate="sample", scale=True, bwd=True),
        # an odd width, norms without bias, a gate per token
        dict(name="norm odd", op="norm", b=3, n=4001, c=765, kind="rms", tx="f32", th="f32", gate="token", scale=False, bwd=True),
        # a wide model at a large batch
        dict(name="norm large", op="norm", b=8, n=4096, c=2048, kind="rms", tx="bf16", th="bf16", gate="sample", scale=True, bwd=True),
        # voxel classes: a 128^3 patch, 4 classes, the teacher's best two kept
        dict(name="distil voxels", op="distil", r=128 ** 3, v=4, k=2, dtype="f32", temp=4.0, bwd=True),
        # a few rows of a large set of classes, loss only
        dict(name="distil small", op="distil", r=64, v=32001, k=8, dtype="f32", temp=2.0, bwd=False),
        # token distillation over a large set of classes, training step
        dict(name="distil large", op="distil", r=4096, v=50000, k=32, dtype="bf16", temp=2.0, bwd=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    # (a softmax over one key and a norm over one channel have gradients of zero: nothing but rounding to compare, so the ranges start above them)
    what = rng.choice(["attn", "attn", "norm", "distil"])
    if what == "attn":
        d = rng.choice([8, 32, 64, 64, 96, 128])
        hkv = rng.choice([1, 2, 4, 8])
        h = hkv * rng.choice([1, 2, 4]) if hkv < 8 else 8
        h = min(h, 8)
        dtype = rng.choice(["f32", "bf16", "bf16"])
        form = rng.choice(["token", "grid", "line", "line"])
        drop = rng.choice([0.0, 0.1, 0.5])
        if form == "token":
            nk = _log(rng, 1, 16000)
            nq = rng.choice([1, 1, 2, 5])
            nk = max(nk, nq)
            return dict(op="attn", b=rng.choice([1, 2, 7, 16]), nq=nq, nk=nk, h=h, hkv=hkv, d=d, gd=1, gh=1, gw=nk + rng.randrange(0, 100), nb=32,
                        dtype=dtype, drop=drop, bwd=False, q0=nk - nq)
        if form == "grid":
            g = [rng.randrange(2, 11) for _ in range(3)]
            vol = g[0] * g[1] * g[2]
            n = vol * rng.choice([1, 1, 2, 4]) if vol <= 600 else vol
            return dict(op="attn", b=rng.choice([1, 2, 4]), nq=n, nk=n, h=h, hkv=hkv, d=d, gd=g[0], gh=g[1], gw=g[2], nb=0, dtype=dtype, drop=drop,
                        bwd=rng.random() < 0.7, q0=0)
        nk = _log(rng, 16, 4000)
        nq = nk if rng.random() < 0.5 else rng.randrange(1, nk + 1)
        return dict(op="attn", b=rng.choice([1, 2]), nq=nq, nk=nk, h=h, hkv=hkv, d=d, gd=1, gh=1, gw=nk + rng.randrange(0, 50), nb=rng.choice([8, 32, 64]),
                    dtype=dtype, drop=drop, bwd=rng.random() < 0.7, q0=rng.randrange(0, nk - nq + 1))
    if what == "norm":
        c = rng.choice([_log(rng, 4, 8000), 8 * _log(rng, 1, 1000)])
        rows = _log(rng, 1, max(1, min(20000, 40_000_000 // c)))
        b = rng.choice([1, 2, 3, 8])
        tx, th = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
        return dict(op="norm", b=b, n=max(1, rows // b), c=c, kind=rng.choice(["layer", "rms"]), tx=tx, th=th, gate=rng.choice(["none", "sample", "token"]),
                    scale=rng.random() < 0.5, bwd=rng.random() < 0.7)
    v = _log(rng, 2, 130000)
    k = max(1, min(v, _log(rng, 1, 64)))
    r = _log(rng, 1, max(1, min(1_000_000, 100_000_000 // v)))
    return dict(op="distil", r=r, v=v, k=k, dtype=rng.choice(["f32", "bf16"]), temp=rng.choice([1.0, 2.0, 4.0]), bwd=rng.random() < 0.7)


# ------------------------------------------------------------------------------------------------------------------- inputs
def _axis_bucket(n, nb, far):
    """log-spaced two-sided buckets of the offsets -(n-1) .. n-1: a quarter of them exact on either side, the rest up to `far`"""
    off = torch.arange(-(n - 1), n, dtype=torch.float64)
    half = nb // 2
    exact = max(1, half // 2)
    a = off.abs()
    big = exact + (torch.log(a.clamp(min=1) / exact) / math.log(max(far, exact + 1) / exact) * (half - exact)).floor()
    return (torch.where(a < exact, a, big.clamp(max=half - 1)) + half * (off > 0)).to(torch.int32)


def prepare(case, seed):
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)

    def rnd(*shape, dtype=torch.float32, s=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * s).to(dtype)

    c = case
    if c["op"] == "attn":
        dt = _DT[c["dtype"]]
        nd = (2 * c["gd"] - 1) * (2 * c["gh"] - 1) * (2 * c["gw"] - 1)
        st = dict(case=c, q=rnd(c["b"], c["nq"], c["h"], c["d"], dtype=dt), k=rnd(c["b"], c["nk"], c["hkv"], c["d"], dtype=dt),
                  v=rnd(c["b"], c["nk"], c["hkv"], c["d"], dtype=dt), grid=(c["gd"], c["gh"], c["gw"]), scale=c["d"] ** -0.5,
                  buckets=_axis_bucket(c["gw"], c["nb"], 128).to(dev) if c["nb"] else None, mask=None)
        st["table"] = rnd(c["nb"] or nd, c["h"], dtype=dt, s=0.5)
        if c["drop"] > 0:       # whole runs of keys missing, as absent modalities or padding leave them
            run = min(c["nk"], c["gd"] * c["gh"] * c["gw"] if not c["nb"] else max(1, c["nk"] // 10))
            gone = torch.rand(c["b"], -(-c["nk"] // run), generator=g, device=dev) < c["drop"]
            gone[0, 0] = False
            st["mask"] = ~gone.repeat_interleave(run, 1)[:, :c["nk"]].contiguous()
        if c["bwd"]:
            st["dout"] = rnd(c["b"], c["nq"], c["h"], c["d"], dtype=dt)
        return st
    if c["op"] == "norm":
        tx, th = _DT[c["tx"]], _DT[c["th"]]
        shape = (c["b"], c["n"], c["c"])

        def norm():
            m = torch.nn.LayerNorm(c["c"], eps=1e-5, device=dev) if c["kind"] == "layer" else torch.nn.RMSNorm(c["c"], eps=1e-6, device=dev)
            with torch.no_grad():
                m.weight.copy_(1 + rnd(c["c"], s=0.2))
                if c["kind"] == "layer":
                    m.bias.copy_(rnd(c["c"], s=0.2))
            return m

        st = dict(case=c, x=rnd(*shape, dtype=tx), h=rnd(*shape, dtype=th, s=2.0) + 0.3, post=norm(), pre=norm(), gate=None, scale=None)
        if c["gate"] != "none":
            st["gate"] = rnd(c["b"], 1 if c["gate"] == "sample" else c["n"], c["c"], dtype=th)
        if c["scale"]:
            st["scale"] = 0.1 + rnd(c["c"], s=0.05)
        if c["bwd"]:
            st["dr"], st["dy"] = rnd(*shape, dtype=tx), rnd(*shape, dtype=th)
        return st
    dt = _DT[c["dtype"]]
    logits = rnd(c["r"], c["v"], dtype=dt, s=3.0)
    teacher = rnd(c["r"], c["k"], s=3.0).sort(1, descending=True)[0] + 3.0
    # k distinct classes a row: a start, and steps that never come back to it
    start = torch.randint(0, c["v"], (c["r"], 1), generator=g, device=dev)
    step = max(1, c["v"] // c["k"])
    index = (start + step * torch.arange(c["k"], device=dev)) % c["v"]
    index = torch.where(torch.rand(c["r"], 1, generator=g, device=dev) < 0.05, -1, index)      # rows without a teacher (padding)
    st = dict(case=c, logits=logits, values=teacher.to(dt), index=index, temp=c["temp"])
    if c["bwd"]:
        st["grad"] = torch.rand(c["r"], generator=g, device=dev) / c["r"]
    return st


# ------------------------------------------------------------------------------------------------------- attention, plain form
def _offsets(c, dev):
    """index of (cell of query i) - (cell of key j) among the grid's offsets"""
    gd, gh, gw = c["gd"], c["gh"], c["gw"]

    def cell(t):
        t = t % (gd * gh * gw)
        return t // (gh * gw), t // gw % gh, t % gw

    a = cell(torch.arange(c["q0"], c["q0"] + c["nq"], device=dev))
    b = cell(torch.arange(c["nk"], device=dev))
    z, y, x = (u[:, None] - w[None, :] + n - 1 for u, w, n in zip(a, b, (gd, gh, gw)))
    return (z * (2 * gh - 1) + y) * (2 * gw - 1) + x


def _plain_attn(s):
    c = s["case"]
    dt, dev = s["q"].dtype, s["q"].device
    rep = c["h"] // c["hkv"]
    q = s["q"].float().transpose(1, 2).contiguous()
    k, v = (s[n].float().transpose(1, 2).repeat_interleave(rep, 1).contiguous() for n in "kv")
    off = _offsets(c, dev)
    rows = s["table"].float() if s["buckets"] is None else s["table"].float()[s["buckets"].long()]        # one row per offset
    att = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    att += rows.t()[:, off].unsqueeze(0)
    if s["mask"] is not None:
        att.masked_fill_(~s["mask"][:, None, None, :], -math.inf)
    top = att.amax(3, keepdim=True)
    att = att.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = att.sum(3, keepdim=True)
    att = att.mul_(torch.where(total > 0, 1 / total, 0.0))
    out = torch.matmul(att, v)
    res = dict(out=out.transpose(1, 2).to(dt))
    if not c["bwd"]:
        return res
    do = s["dout"].float().transpose(1, 2).contiguous()
    delta = (do * out).sum(3, keepdim=True)
    dv = torch.matmul(att.transpose(2, 3).contiguous(), do)
    ds = torch.matmul(do, v.transpose(2, 3).contiguous()).sub_(delta).mul_(att)
    dq = torch.matmul(ds, k) * s["scale"]
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * s["scale"]
    shape = (c["b"], c["hkv"], rep, c["nk"], c["d"])
    dk, dv = (t.view(shape).sum(2).transpose(1, 2).to(dt) for t in (dk, dv))
    by_pair = ds.sum(0)
    if c["nb"]:       # a line: equal offsets are the diagonals, summed as the columns of a skewed view
        nq, nk = c["nq"], c["nk"]
        wide = torch.cat([by_pair.flip(2), by_pair.new_zeros(c["h"], nq, nq)], 2).view(c["h"], -1)[:, :nq * (nk + nq - 1)]
        diag = wide.view(c["h"], nq, nk + nq - 1).sum(1, dtype=torch.float64)
        per = torch.zeros(c["h"], 2 * c["gw"] - 1, dtype=torch.float64, device=dev)
        first = c["q0"] - (nk - 1) + c["gw"] - 1
        per[:, first:first + nk + nq - 1] = diag
    else:
        per = torch.zeros(c["h"], rows.shape[0], dtype=torch.float64, device=dev).index_add_(1, off.view(-1), by_pair.view(c["h"], -1).double())
    if s["buckets"] is not None:
        per = torch.zeros(c["h"], s["table"].shape[0], dtype=torch.float64, device=dev).index_add_(1, s["buckets"].long(), per)
    return dict(res, dq=dq.transpose(1, 2).to(dt), dk=dk, dv=dv, dtable=per.t().to(dt))


def _own_attn(s):
    from passion_amd import ops
    c = s["case"]
    if not c["bwd"]:
        with torch.no_grad():
            return dict(out=ops.rel_attention(s["q"], s["k"], s["v"], s["table"], s["grid"], buckets=s["buckets"], key_mask=s["mask"], scale=s["scale"],
                                              q_start=c["q0"]))
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v", "table")]
    out = ops.rel_attention(*leaves, s["grid"], buckets=s["buckets"], key_mask=s["mask"], scale=s["scale"], q_start=c["q0"])
    dq, dk, dv, dtable = torch.autograd.grad(out, leaves, s["dout"])
    return dict(out=out.detach(), dq=dq, dk=dk, dv=dv, dtable=dtable)


# ------------------------------------------------------------------------------------------------- residual and norms, plain form
def _norm_fwd(t, m, layer):
    eps = m.eps
    mean = t.mean(-1, keepdim=True) if layer else 0.0
    u = t - mean
    rstd = (u.square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = u * rstd
    w = m.weight.to(t.dtype)
    return hat * w + (m.bias.to(t.dtype) if layer else 0.0), hat, rstd


def _norm_bwd(g, hat, rstd, m, layer):
    """gradient of the input; column sums for the weight (and bias)"""
    dw = (g * hat).sum((0, 1), dtype=torch.float64).float()
    db = g.sum((0, 1), dtype=torch.float64).float() if layer else None
    gw = g * m.weight.to(g.dtype)
    dx = gw - hat * (gw * hat).mean(-1, keepdim=True)
    if layer:
        dx = dx - gw.mean(-1, keepdim=True)
    return dx * rstd, dw, db


def _plain_norm(s):
    c = s["case"]
    layer = c["kind"] == "layer"
    x, h = s["x"].float(), s["h"].float()
    u, hat1, rstd1 = _norm_fwd(h, s["post"], layer)
    gate = s["gate"].float() if s["gate"] is not None else None
    scale = s["scale"]
    m = u if gate is None else u * gate
    r = x + (m if scale is None else m * scale)
    y, hat2, rstd2 = _norm_fwd(r, s["pre"], layer)
    res = dict(r=r.to(s["x"].dtype), y=y.to(s["h"].dtype))
    if not c["bwd"]:
        return res
    d2, dw2, db2 = _norm_bwd(s["dy"].float(), hat2, rstd2, s["pre"], layer)
    dr = s["dr"].float() + d2
    dm = dr if scale is None else dr * scale
    du = dm if gate is None else dm * gate
    dh, dw1, db1 = _norm_bwd(du, hat1, rstd1, s["post"], layer)
    res.update(dx=dr.to(s["x"].dtype), dh=dh.to(s["h"].dtype), dw_post=dw1, dw_pre=dw2)
    if layer:
        res.update(db_post=db1, db_pre=db2)
    if gate is not None:
        dg = dm * u
        res["dgate"] = (dg.sum(1, keepdim=True, dtype=torch.float64) if c["gate"] == "sample" else dg).to(s["gate"].dtype)
    if scale is not None:
        res["dscale"] = (dr * m).sum((0, 1), dtype=torch.float64).float()
    return res


def _own_norm(s):
    from passion_amd import ops
    c = s["case"]
    if not c["bwd"]:
        with torch.no_grad():
            r, y = ops.residual_norm(s["x"], s["h"], post=s["post"], pre=s["pre"], gate=s["gate"], scale=s["scale"])
        return dict(r=r, y=y)
    names = ["dx", "dh", "dw_post", "dw_pre"]
    leaves = [s["x"].detach().requires_grad_(), s["h"].detach().requires_grad_(), s["post"].weight, s["pre"].weight]
    if c["kind"] == "layer":
        names += ["db_post", "db_pre"]
        leaves += [s["post"].bias, s["pre"].bias]
    gate = scale = None
    if s["gate"] is not None:
        gate = s["gate"].detach().requires_grad_()
        names.append("dgate")
        leaves.append(gate)
    if s["scale"] is not None:
        scale = s["scale"].detach().requires_grad_()
        names.append("dscale")
        leaves.append(scale)
    r, y = ops.residual_norm(leaves[0], leaves[1], post=s["post"], pre=s["pre"], gate=gate, scale=scale)
    grads = torch.autograd.grad([r, y], leaves, [s["dr"], s["dy"]])
    return dict(r=r.detach(), y=y.detach(), **dict(zip(names, grads)))


# ------------------------------------------------------------------------------------------------------ distillation, plain form
def _plain_distil(s):
    c = s["case"]
    t = s["temp"]
    z = s["logits"].float() / t
    lse = torch.logsumexp(z, 1, keepdim=True)
    ok = s["index"] >= 0
    at = s["index"].clamp(min=0)
    tv = torch.where(ok, s["values"].float() / t, -math.inf)
    live = ok.any(1, keepdim=True)
    logp = tv - torch.where(live, torch.logsumexp(tv, 1, keepdim=True), 0.0)
    p = logp.exp()
    logq = z.gather(1, at) - lse
    loss = (t * t) * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    if not c["bwd"]:
        return dict(loss=loss)
    dz = (z - lse).exp_()
    dz *= live
    dz.scatter_add_(1, at, -p)
    dz *= (s["grad"] * t)[:, None]
    return dict(loss=loss, dlogits=dz.to(s["logits"].dtype))


def _own_distil(s):
    from passion_amd import ops
    if not s["case"]["bwd"]:
        with torch.no_grad():
            return dict(loss=ops.topk_distill(s["logits"], s["values"], s["index"], s["temp"]))
    logits = s["logits"].detach().requires_grad_()
    loss = ops.topk_distill(logits, s["values"], s["index"], s["temp"])
    (d,) = torch.autograd.grad(loss, [logits], s["grad"])
    return dict(loss=loss.detach(), dlogits=d)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attn, "norm": _own_norm, "distil": _own_distil}[op](state)
    with torch.no_grad():
        return {"attn": _plain_attn, "norm": _plain_norm, "distil": _plain_distil}[op](state)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "attn":
        e = 4 if c["dtype"] == "f32" else 2
        q, kv = c["b"] * c["nq"] * c["h"] * c["d"], c["b"] * c["nk"] * c["hkv"] * c["d"]
        tab = (c["nb"] or (2 * c["gd"] - 1) * (2 * c["gh"] - 1) * (2 * c["gw"] - 1)) * c["h"]
        nbytes = e * (2 * q + 2 * kv + tab) + (4 * (2 * c["gw"] - 1) if c["nb"] else 0) + (c["b"] * c["nk"] if c["drop"] else 0)
        pairs = c["b"] * c["h"] * c["nq"] * c["nk"] * c["d"]
        if not c["bwd"]:
            return dict(bytes=nbytes, flops=4 * pairs)
        return dict(bytes=nbytes + e * (2 * q + 2 * kv + tab), flops=14 * pairs)
    if c["op"] == "norm":
        ex, eh = (4 if c[n] == "f32" else 2 for n in ("tx", "th"))
        rows, n = c["b"] * c["n"], c["b"] * c["n"] * c["c"]
        gate = {"none": 0, "sample": c["b"] * c["c"] * eh, "token": n * eh}[c["gate"]]
        cols = c["c"] * 4 * ((4 if c["kind"] == "layer" else 2) + (1 if c["scale"] else 0))
        nbytes = n * 2 * (ex + eh) + gate + cols
        if c["bwd"]:
            nbytes += n * 2 * (ex + eh) + gate + cols
        return dict(bytes=nbytes, flops=n * (40 if c["bwd"] else 15) + rows)
    e = 4 if c["dtype"] == "f32" else 2
    n = c["r"] * c["v"]
    side = c["r"] * (c["k"] * (e + 8) + 4)
    return dict(bytes=n * e + side + (n * e + 4 * c["r"] if c["bwd"] else 0), flops=n * (8 if c["bwd"] else 4))


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_attn(s):
    c = s["case"]
    dev, rep = s["q"].device, c["h"] // c["hkv"]
    grid = torch.tensor([c["gd"], c["gh"], c["gw"]], device=dev)

    def cells(first, n):
        t = torch.arange(first, first + n, device=dev) % int(grid.prod())
        return torch.stack([t // int(grid[1] * grid[2]), (t // int(grid[2])) % int(grid[1]), t % int(grid[2])], 1)

    box = 2 * grid - 1
    weight = torch.stack([box[1] * box[2], box[2], box.new_ones(())])
    at_q, at_k = (cells(c["q0"], c["nq"]) * weight).sum(1), ((cells(0, c["nk"]) - (grid - 1)) * weight).sum(1)
    off = at_q.view(-1, 1) - at_k.view(1, -1)
    which = off if s["buckets"] is None else s["buckets"].long()[off]
    table = s["table"].double()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=dev)
    if c["bwd"]:
        dq, dk, dv = torch.zeros_like(out), *(torch.zeros(s["k"].shape, dtype=torch.float64, device=dev) for _ in range(2))
        dtab = torch.zeros_like(table)
    for h in range(c["h"]):
        bias = table[:, h][which]
        for b in range(c["b"]):
            q, k, v = s["q"][b, :, h].double(), s["k"][b, :, h // rep].double(), s["v"][b, :, h // rep].double()
            keep = torch.ones(c["nk"], dtype=torch.bool, device=dev) if s["mask"] is None else s["mask"][b]
            if not bool(keep.any()):
                continue
            sc = torch.mm(q, k.t().contiguous()) * s["scale"] + bias
            sc[:, ~keep] = -math.inf
            p = torch.softmax(sc, 1)
            out[b, :, h] = torch.mm(p, v)
            if c["bwd"]:
                do = s["dout"][b, :, h].double()
                dp = torch.mm(do, v.t().contiguous())
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                dq[b, :, h] = torch.mm(ds, k) * s["scale"]
                dk[b, :, h // rep] += torch.mm(ds.t().contiguous(), q) * s["scale"]
                dv[b, :, h // rep] += torch.mm(p.t().contiguous(), do)
                n_off = int(box.prod())
                per = torch.bincount(off.reshape(-1), weights=ds.reshape(-1), minlength=n_off)
                dtab[:, h] += per if s["buckets"] is None else torch.bincount(s["buckets"].long(), weights=per, minlength=table.shape[0])
    return dict(out=out, dq=dq, dk=dk, dv=dv, dtable=dtab) if c["bwd"] else dict(out=out)


def _exact_norm(s):
    """by torch's own differentiation of the definition, in 64 bits"""
    c = s["case"]
    d = {n: s[n].detach().double() for n in ("x", "h", "gate", "scale", "dr", "dy") if s.get(n) is not None}
    par = {"w1": s["post"].weight, "w2": s["pre"].weight}
    if c["kind"] == "layer":
        par.update(b1=s["post"].bias, b2=s["pre"].bias)
    d.update({n: p.detach().double() for n, p in par.items()})
    names = [n for n in ("x", "h", "gate", "scale", "w1", "w2", "b1", "b2") if n in d]
    with torch.enable_grad():
        for n in names:
            d[n].requires_grad_(c["bwd"])

        def norm(t, i, m):
            if c["kind"] == "layer":
                t = t - t.mean(2, keepdim=True)
                return t / torch.sqrt((t * t).mean(2, keepdim=True) + m.eps) * d["w%d" % i] + d["b%d" % i]
            return t / torch.sqrt((t * t).mean(2, keepdim=True) + m.eps) * d["w%d" % i]

        m = norm(d["h"], 1, s["post"])
        for n in ("gate", "scale"):
            if n in d:
                m = m * d[n]
        r = d["x"] + m
        y = norm(r, 2, s["pre"])
        res = dict(r=r.detach(), y=y.detach())
        if c["bwd"]:
            label = dict(x="dx", h="dh", gate="dgate", scale="dscale", w1="dw_post", w2="dw_pre", b1="db_post", b2="db_pre")
            grads = torch.autograd.grad((r * d["dr"]).sum() + (y * d["dy"]).sum(), [d[n] for n in names])
            res.update({label[n]: t for n, t in zip(names, grads)})
    return res


def _exact_distil(s):
    c, t = s["case"], s["temp"]
    loss = torch.zeros(c["r"], dtype=torch.float64, device=s["logits"].device)
    d = torch.zeros(c["r"], c["v"], dtype=torch.float64, device=loss.device) if c["bwd"] else None
    rows = max(1, 60_000_000 // c["v"])
    for a in range(0, c["r"], rows):
        sl = slice(a, a + rows)
        logq = torch.log_softmax(s["logits"][sl].double() / t, 1)
        there = s["index"][sl] >= 0
        e = torch.where(there, torch.exp((s["values"][sl].double() - s["values"][sl].double().amax(1, keepdim=True)) / t), 0.0)
        p = e / e.sum(1, keepdim=True).clamp(min=1e-300)
        at = torch.where(there, s["index"][sl], 0)
        loss[sl] = t * t * torch.where(p > 0, p * (p.clamp(min=1e-300).log() - logq.gather(1, at)), 0.0).sum(1)
        if c["bwd"]:
            g = torch.exp(logq) * there.any(1, keepdim=True)
            d[sl] = g.scatter_add(1, at, -p) * (s["grad"][sl].double() * t)[:, None]
    return dict(loss=loss, dlogits=d) if c["bwd"] else dict(loss=loss)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "norm": _exact_norm, "distil": _exact_distil}[case["op"]](s)
