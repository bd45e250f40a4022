"""ops.residual_norm (csrc/residual_norm.hip): r = x + scale * gate * post(h), y = pre(r), against the definition in 64 bits differentiated by
torch, at the widths, row counts and parts where its layouts change, and its refusals.

Tolerances, from the arithmetic: a moment is a sum over C <= 8192 f32 values in a tree (8 in a register, 6 shuffles, up to 16 wavefronts: depth below 32),
so it is off by at most 32 * 2^-24 = 1.9e-6 of the sum of magnitudes; a norm multiplies two such factors and rounds five more times, two norms follow one
another and the backward runs through both again: below 1e-5 of the largest value in well-conditioned rows (a variance of order one).  Column sums are
sequential over a workgroup's rows (at most 64 rounds here), its 256 rows a round and a quarter of 1024 partials: below 600 additions in sequence,
600 * 2^-24 = 3.6e-5 of the sum of magnitudes, taken from the 64-bit terms themselves.  A stored value rounds once more (helpers: near)."""
import pytest
import torch

from _op_util import near, replayed

F, H = torch.float32, torch.bfloat16


def _mods(C, kind, seed, device):
    g = torch.Generator().manual_seed(seed)
    m = torch.nn.LayerNorm(C, eps=1e-5) if kind == "layer" else torch.nn.RMSNorm(C, eps=1e-6)
    with torch.no_grad():
        m.weight.copy_(1 + 0.3 * torch.randn(C, generator=g))
        if kind == "layer":
            m.bias.copy_(0.3 * torch.randn(C, generator=g))
    return m.to(device)


def _inputs(B, N, C, tx, th, gate, scale, seed=3):
    g = torch.Generator().manual_seed(seed)
    d = dict(x=torch.randn(B, N, C, generator=g).to(tx), h=(2 * torch.randn(B, N, C, generator=g) + 0.5).to(th))
    if gate:
        d["gate"] = torch.randn(B, 1 if gate == "sample" else N, C, generator=g).to(th)
    if scale:
        d["scale"] = 0.5 + 0.2 * torch.randn(C, generator=g)
    d["dr"], d["dy"] = torch.randn(B, N, C, generator=g).to(tx), torch.randn(B, N, C, generator=g).to(th)
    return d


def _reference(d, post, pre, use_dr=True, use_dy=True):
    """outputs, input gradients, and for every broadcast input the per-row terms of its gradient, in 64 bits"""
    shape = d["x"].shape
    leaf = {n: d[n].double().requires_grad_() for n in ("x", "h")}
    full = {}

    def spread(name, t):
        if t is None:
            return None
        full[name] = t.detach().double().cpu().expand(shape).clone().requires_grad_()
        return full[name]

    def norm(t, m, tag):
        if m is None:
            return t
        w = spread("w_" + tag, m.weight)
        if isinstance(m, torch.nn.LayerNorm):
            c = t - t.mean(-1, keepdim=True)
            return c / (c.square().mean(-1, keepdim=True) + m.eps).sqrt() * w + spread("b_" + tag, m.bias)
        return t / (t.square().mean(-1, keepdim=True) + m.eps).sqrt() * w

    u = norm(leaf["h"], post, "post")
    for n in ("gate", "scale"):
        if n in d:
            u = u * spread(n, d[n])
    r = leaf["x"] + u
    y = norm(r, pre, "pre") if pre is not None else None
    loss = 0.0
    if use_dr:
        loss = loss + (r * d["dr"].double()).sum()
    if y is not None and use_dy:
        loss = loss + (y * d["dy"].double()).sum()
    ins = {**leaf, **full}
    grads = dict(zip(ins, torch.autograd.grad(loss, list(ins.values()), allow_unused=True)))
    return r.detach(), None if y is None else y.detach(), {n: (torch.zeros(shape, dtype=torch.float64) if t is None else t) for n, t in grads.items()}


def _run(d, post, pre, use_dr=True, use_dy=True):
    from passion_amd import ops
    dev = torch.device("cuda:0")
    t = {n: v.to(dev) for n, v in d.items()}
    names = [n for n in ("x", "h", "gate", "scale") if n in t]
    for n in names:
        t[n].requires_grad_()
    params = {}
    for tag, m in (("post", post), ("pre", pre)):
        if m is not None:
            params["w_" + tag] = m.weight
            if isinstance(m, torch.nn.LayerNorm):
                params["b_" + tag] = m.bias
    out = ops.residual_norm(t["x"], t["h"], post, pre, t.get("gate"), t.get("scale"))
    r, y = out if pre is not None else (out, None)
    outs, gs = [], []
    if use_dr:
        outs, gs = [r], [t["dr"]]
    if y is not None and use_dy:
        outs, gs = outs + [y], gs + [t["dy"]]
    leaves = {**{n: t[n] for n in names}, **params}
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), gs, allow_unused=True)))
    return r, y, grads


def _check(d, post, pre, **kw):
    r, y, got = _run(d, post, pre, **kw)
    rr, yr, want = _reference(d, post, pre, **kw)
    near(r, rr, 1e-5, "r")
    if yr is not None:
        near(y, yr, 1e-5, "y")
    for n, g in got.items():
        if g is None:                         # autograd: nothing reaches it
            assert float(want[n].abs().max()) == 0, n
            continue
        if n in ("x", "h"):
            near(g, want[n], 2e-5, "d" + n)
            continue
        dims = [0, 1] if n != "gate" else [1] if d["gate"].shape[1] == 1 else []
        s, a = want[n], want[n].abs()
        for i in dims:
            s, a = s.sum(i, keepdim=True), a.sum(i, keepdim=True)
        near(g.reshape(s.shape), s, 6e-5, "d" + n, room=a + 0.2 * a.mean())      # + a share of the inputs' own error (2e-5 a term)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,th", [(F, F), (F, H), (H, H)])
@pytest.mark.parametrize("C", [1, 3, 8, 64, 100, 512, 520, 765, 1024, 2048, 2056, 4104, 8192])
def test_widths(C, tx, th):
    """from one channel to the widest row: sub-wavefront rows, one wavefront, several, 512 and 1024 threads, unaligned rows"""
    kind = "layer" if C > 1 else "rms"                # one channel leaves LayerNorm nothing
    d = _inputs(2, 9, C, tx, th, "sample", True)
    if C == 1:
        d["h"] = d["h"].abs() + 1                     # away from 0, where x / |x| jumps
        d["x"] = d["x"].abs() + 8
        post = None
    else:
        post = _mods(C, kind, 1, "cuda")
    _check(d, post, _mods(C, kind, 2, "cuda") if C > 3 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,th", [(F, F), (F, H), (H, H)])
@pytest.mark.parametrize("C,kind,gate", [(2051, "layer", "token"), (4095, "rms", "sample"), (4099, "layer", "sample"), (6001, "rms", "token"), (8191, "layer", None), (6008, "rms", "token")])
def test_wide_rows_of_odd_widths(C, kind, gate, tx, th):
    """rows of more than 2048 channels that start off the 16-byte points: the scalar forms of 512 and 1024 threads, forward and backward"""
    _check(_inputs(2, 7, C, tx, th, gate, True), _mods(C, kind, 1, "cuda"), _mods(C, "layer", 2, "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate", [None, "sample", "token"])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("parts", ["both", "post", "pre", "none"])
def test_parts(kind, gate, scale, parts):
    C = 96
    d = _inputs(3, 37, C, F, H, gate, scale)
    _check(d, _mods(C, kind, 1, "cuda") if parts in ("both", "post") else None, _mods(C, kind, 2, "cuda") if parts in ("both", "pre") else None)


@pytest.mark.gpu
@pytest.mark.parametrize("B,N,C", [(1, 1, 512), (4, 1, 512), (1, 2, 4096), (2, 5000, 16), (7, 333, 256), (1, 4097, 512), (300, 2, 24)])
def test_rows(B, N, C):
    d = _inputs(B, N, C, F, H, "sample", True)
    _check(d, _mods(C, "layer", 1, "cuda"), _mods(C, "rms", 2, "cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("use_dr,use_dy", [(True, False), (False, True)])
def test_one_output_used(use_dr, use_dy):
    d = _inputs(2, 50, 128, F, F, "token", True)
    _check(d, _mods(128, "layer", 1, "cuda"), _mods(128, "layer", 2, "cuda"), use_dr=use_dr, use_dy=use_dy)


@pytest.mark.gpu
def test_large_offset_keeps_the_variance():
    """rows whose mean is 1000 times their spread: the variance is taken about the mean (of the wavefront first), not from a difference of squares.
    The subtraction x - mean is exact to 2^-24 * 1000 = 6e-5 of the spread, which bounds y"""
    from passion_amd import ops
    for C in (256, 2048, 6000):
        g = torch.Generator().manual_seed(0)
        x = (1000 + torch.randn(1, 8, C, generator=g))
        m = _mods(C, "layer", 5, "cuda")
        _, y = ops.residual_norm(x.cuda(), torch.zeros_like(x).cuda(), None, m)
        c = x.double() - x.double().mean(-1, keepdim=True)
        want = c / (c.square().mean(-1, keepdim=True) + m.eps).sqrt() * m.weight.double().cpu() + m.bias.double().cpu()
        near(y, want.detach(), 1.3e-4, f"y at {C}")


@pytest.mark.gpu
def test_gradient_against_differences():
    """f32, central differences along a random direction of every input: the quotient is off by step^2 times a third derivative (order one here: 1e-4) and
    by the outputs' rounding over the step, 2^-24 * sqrt(elements) * |out| / 1e-2 = 6e-4 of the typical sum"""
    from passion_amd import ops
    d = {n: v.cuda() for n, v in _inputs(2, 7, 40, F, F, "sample", True).items()}
    post, pre = _mods(40, "layer", 1, "cuda"), _mods(40, "rms", 2, "cuda")
    names = ("x", "h", "gate", "scale")

    def value(t):
        r, y = ops.residual_norm(t["x"], t["h"], post, pre, t["gate"], t["scale"])
        return (r.double() * d["dr"].double()).sum() + (y.double() * d["dy"].double()).sum()

    leaves = {n: d[n].clone().requires_grad_() for n in names}
    grads = dict(zip(names, torch.autograd.grad(value(leaves), list(leaves.values()))))
    g = torch.Generator(device="cuda").manual_seed(9)
    for n in names:
        way = torch.randn(d[n].shape, generator=g, device="cuda")
        way /= way.square().mean().sqrt()
        with torch.no_grad():
            plus, minus = (value({**d, n: d[n] + s * 1e-2 * way}) for s in (1, -1))
        quotient, slope = float(plus - minus) / 2e-2, float((grads[n].double() * way.double()).sum())
        assert abs(quotient - slope) < 1e-2 * float(grads[n].norm()), (n, quotient, slope)


@pytest.mark.gpu
def test_strides_streams_and_repeatability():
    from passion_amd import ops
    d = {n: v.cuda() for n, v in _inputs(3, 129, 192, F, H, "sample", True).items()}
    post, pre = _mods(192, "layer", 1, "cuda"), _mods(192, "layer", 2, "cuda")

    def step(x, h):
        x, h, gate = x.detach().requires_grad_(), h.detach().requires_grad_(), d["gate"].detach().requires_grad_()
        r, y = ops.residual_norm(x, h, post, pre, gate, d["scale"])
        return (r, y, *torch.autograd.grad([r, y], [x, h, gate, post.weight, pre.bias], [d["dr"], d["dy"]]))

    base = step(d["x"], d["h"])
    again = step(d["x"], d["h"])
    turned = step(d["x"].transpose(0, 1).contiguous().transpose(0, 1), d["h"].transpose(1, 2).contiguous().transpose(1, 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(d["x"], d["h"])
    torch.cuda.synchronize()
    for a, b, c, e in zip(base, again, turned, other):
        assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, e)


@pytest.mark.gpu
def test_captured_and_replayed():
    from passion_amd import ops
    post, pre = _mods(512, "layer", 1, "cuda"), _mods(512, "layer", 2, "cuda")
    sets = [[v.cuda() for v in _inputs(2, 65, 512, F, H, "sample", True, seed=s).values()] for s in range(4)]
    statics = [t.clone() for t in sets[0]]

    def step(x, h, gate, scale, dr, dy):
        ins = [t.detach().requires_grad_() for t in (x, h, gate, scale)]
        r, y = ops.residual_norm(ins[0], ins[1], post, pre, ins[2], ins[3])
        return (r, y, *torch.autograd.grad([r, y], ins + [post.weight, pre.weight], [dr, dy]))

    replayed(lambda: step(*statics), statics, sets, step)


@pytest.mark.gpu
@pytest.mark.parametrize("tx,th", [(F, F), (F, H), (H, H)])
def test_the_default_eps_of_an_rms_norm(tx, th):
    """nn.RMSNorm(C) without eps adds f32's epsilon, whatever the input's type: rows about as large as its root, where it decides the result"""
    from passion_amd import ops
    C = 64
    d = _inputs(1, 5, C, tx, th, None, False)
    x, h = (4e-4 * d["x"].double()).to(tx), (4e-4 * d["h"].double()).to(th)
    m = torch.nn.RMSNorm(C).cuda()
    r, y = ops.residual_norm(x.cuda(), torch.zeros_like(h).cuda(), None, m)
    assert torch.equal(r.cpu(), x)
    near(y, m(x.cuda().float()).detach().double().cpu(), 1e-5, "pre")
    r = ops.residual_norm(torch.zeros_like(x).cuda(), h.cuda(), m)
    near(r, m(h.cuda().float()).detach().double().cpu(), 1e-5, "post")


def test_the_default_eps_is_the_module_s():
    from passion_amd import ops
    for dt in (F, H):
        x = torch.full((1, 64), 1e-4).to(dt)
        eps = ops._norm_spec(torch.nn.RMSNorm(64), 64, "pre")[3]
        want = torch.nn.RMSNorm(64).to(dt)(x).detach().double()
        got = x.double() / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()
        assert float((got - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())


@pytest.mark.gpu
def test_as_many_rows_as_are_taken():
    """the last rows of the longest sample there may be"""
    from passion_amd import ops
    N = 2 ** 31 - 2 ** 27 - 1
    x = torch.zeros(N, 1, dtype=H, device="cuda")
    h = torch.full_like(x, 2.0)
    x[-5000:, 0] = torch.arange(5000, device="cuda") % 100
    r = ops.residual_norm(x, h)
    assert bool((r[:-5000] == 2).all()) and torch.equal(r[-5000:], x[-5000:] + 2)


def test_more_rows_are_refused():
    """the kernels count a sample's rows, and the steps past its end, in 32 bits"""
    from passion_amd import _lib, ops
    lib, N = _lib.load(), 2 ** 31 - 2 ** 27
    assert 0 < lib.passion_residual_norm_part_floats(1, N - 1, 1) <= 2048 * 6 and lib.passion_residual_norm_part_floats(65530, N - 1, 8) > 0
    fwd = lambda n: lib.passion_residual_norm_fwd(256, 0, 256, 0, None, None, 0, 0.0, None, 0, 0, None, None, None, 0, 0.0, 1, n, 1, 256, None, None, None)
    assert lib.passion_residual_norm_part_floats(1, N, 1) == -1003 and fwd(N) == -1003 and fwd(2 ** 31 - 1) == -1003
    x = torch.zeros(1, 1).expand(N, 1)
    with pytest.raises(ValueError):
        ops.residual_norm(x, x)


@pytest.mark.gpu
def test_no_rows():
    from passion_amd import ops
    x = torch.zeros(2, 0, 64, device="cuda", requires_grad=True)
    m = torch.nn.LayerNorm(64).cuda()
    r, y = ops.residual_norm(x, x.detach(), m, m)
    assert r.shape == y.shape == (2, 0, 64)
    (r.sum() + y.sum()).backward()
    assert float(m.weight.grad.abs().max()) == 0


def test_refusals():
    from passion_amd import _lib, ops
    x = torch.zeros(2, 3, 16)
    ln = torch.nn.LayerNorm(16)
    for bad in (dict(x=x, h=x[:, :2]), dict(x=x, h=x.half()), dict(x=x.bfloat16(), h=x), dict(x=x, h=x, post=torch.nn.LayerNorm(8)),
                dict(x=x, h=x, pre=torch.nn.BatchNorm1d(16)), dict(x=x, h=x, gate=x[:1]), dict(x=x, h=x, gate=x[:, :1].half()),
                dict(x=x, h=x, scale=torch.zeros(15)), dict(x=torch.zeros(1, 8193), h=torch.zeros(1, 8193))):
        with pytest.raises(ValueError):
            ops.residual_norm(**bad)
    with pytest.raises(_lib.PassionHipError):
        ops.residual_norm(x, x, ln, ln)             # CPU tensors


def test_c_entry_refuses_on_the_host():
    from passion_amd import _lib
    lib = _lib.load()
    fwd = lambda B, N, C, xd, hd, post, gm: lib.passion_residual_norm_fwd(256, xd, 256, hd, None, None, post, 1e-5, 256 if gm else None, gm, 0, None, None, None, 1,
                                                                          1e-5, B, N, C, 256, 256, None, None)
    assert fwd(0, 4, 64, 0, 0, 1, 0) == -1003 and fwd(1, 0, 64, 0, 0, 1, 0) == -1003 and fwd(1, 4, 8193, 0, 0, 1, 0) == -1003
    assert fwd(1, 4, 64, 1, 0, 1, 0) == -1003 and fwd(1, 4, 64, 0, 0, 3, 0) == -1003 and fwd(65531, 4, 64, 0, 0, 1, 0) == -1003
    assert lib.passion_residual_norm_fwd(None, 0, 256, 0, None, None, 0, 0.0, None, 0, 0, None, None, None, 0, 0.0, 1, 1, 8, 256, None, None, None) == -1003
    assert lib.passion_residual_norm_part_floats(1, 4, 0) == -1003
