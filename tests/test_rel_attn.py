"""ops.rel_attention (csrc/rel_attn.hip) against the definition in 64 bits: every way to the bias (small box of offsets, 1D window, memory, none), head widths, shared heads,
ragged and cross lengths, single tokens, masks that leave rows empty and hide NaN, repeated cells, excluded entries -- forward and every gradient.

Tolerances, element by element, from the roundings the kernels make (u = 2^-8 for bf16: probabilities and dS are rounded to the matrix operands' type once; for f32 the
matrix products are f32 and u stands for their accumulated error: a score sums D <= 128 products, at most 132 * 2^-24 * scale * sum |q k| = 5.7e-5 at D = 128, and an
output sums up to 4096 keys in sequence per lane, below 2.4e-4 of the sum of magnitudes in the worst case):
  out: u p|v|;   dv: u p^T|dout|;   delta: E = |dout| . (u p|v| + u |out|) since it is formed from the stored out;
  dS: u |dS| + p E;   dq, dk: scale times that against |k|, |q|;   dtable: its sum by bucket -- plus one rounding of what is stored (near)."""
import math

import pytest
import torch

from _op_util import near, replayed

F, H = torch.float32, torch.bfloat16
U = {F: 3e-4, H: 2.0 ** -8 + 1e-4}


def _offset_index(grid, Nq, Nk, q0):
    D, Hh, W = (1,) * (3 - len(grid)) + tuple(grid)
    t = torch.arange(max(Nk, q0 + Nq)) % (D * Hh * W)
    cell = torch.stack([t // (Hh * W), t // W % Hh, t % W], 1)
    d = cell[q0:q0 + Nq, None] - cell[None, :Nk] + torch.tensor([D - 1, Hh - 1, W - 1])
    return (d[..., 0] * (2 * Hh - 1) + d[..., 1]) * (2 * W - 1) + d[..., 2]


def _make(B, Nq, Nk, heads, Hkv, D, dt, grid=None, nb=None, q0=0, mask=None, seed=0, table_dt=None):
    g = torch.Generator().manual_seed(seed)
    c = dict(q=torch.randn(B, Nq, heads, D, generator=g).to(dt), k=torch.randn(B, Nk, Hkv, D, generator=g).to(dt), v=torch.randn(B, Nk, Hkv, D, generator=g).to(dt),
             dout=torch.randn(B, Nq, heads, D, generator=g).to(dt), table=None, buckets=None, grid=grid, q0=q0, mask=None, scale=D ** -0.5)
    if grid is not None:
        n = math.prod(2 * s - 1 for s in grid)
        if nb is not None:
            c["buckets"] = torch.randint(0, nb, (n,), generator=g).int()
        c["table"] = torch.randn(nb or n, heads, generator=g).to(table_dt or dt)
    if mask == "random":
        c["mask"] = torch.rand(B, Nk, generator=g) < 0.6
    elif mask == "runs":
        c["mask"] = (torch.arange(Nk)[None] // 70 + torch.arange(B)[:, None]) % 3 != 1
    elif mask == "empty":
        c["mask"] = torch.rand(B, Nk, generator=g) < 0.6
        c["mask"][-1] = False
    return c


def _reference(c, grads=True):
    """everything in 64 bits on the GPU, with the error rooms"""
    t = {n: c[n].cuda().double() if c[n] is not None else None for n in ("q", "k", "v", "dout", "table")}
    B, Nq, heads, D = t["q"].shape
    Hkv = t["k"].shape[2]
    u = U[c["q"].dtype]
    q, do = (t[n].transpose(1, 2).contiguous() for n in ("q", "dout"))
    k, v = (t[n].transpose(1, 2).repeat_interleave(heads // Hkv, 1).contiguous() for n in ("k", "v"))
    if c["mask"] is not None:
        gone = ~c["mask"].cuda().bool()[:, None, :, None]
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    s = q @ k.transpose(2, 3).contiguous() * c["scale"]
    which = None
    if t["table"] is not None:
        off = _offset_index(c["grid"], Nq, k.shape[2], c["q0"]).cuda()
        which = off if c["buckets"] is None else c["buckets"].cuda().long()[off]
        inside = (which >= 0) & (which < t["table"].shape[0])
        bias = torch.where(inside[..., None], t["table"][which.clamp(0, t["table"].shape[0] - 1)], 0.0).permute(2, 0, 1)
        s = s + torch.where(bias <= -1e30, -math.inf, bias)
    if c["mask"] is not None:
        s = s.masked_fill(gone.transpose(2, 3), -math.inf)
    top = s.amax(3, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    tot = e.sum(3, keepdim=True)
    p = torch.where(tot > 0, e / tot, 0.0)
    out = p @ v
    room = p @ v.abs()
    res = dict(out=(out.transpose(1, 2), room.transpose(1, 2)))
    if not grads:
        return res
    dp = do @ v.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    err = u * ds.abs() + p * (do.abs() * u * (room + out.abs())).sum(3, keepdim=True)
    share = lambda a: a.view(B, Hkv, heads // Hkv, *a.shape[2:]).sum(2).transpose(1, 2)
    T = lambda a: a.transpose(2, 3).contiguous()
    res["dq"] = ((ds @ k * c["scale"]).transpose(1, 2), (err @ k.abs() * c["scale"] / u + u * (ds.abs() @ k.abs()) * c["scale"]).transpose(1, 2))
    res["dk"] = (share(T(ds) @ q * c["scale"]), share(T(err) @ q.abs() * c["scale"] / u + u * (T(ds.abs()) @ q.abs()) * c["scale"]))
    res["dv"] = (share(T(p) @ do), share(T(p) @ do.abs()))
    if which is not None:
        n = t["table"].shape[0]
        tab, rm = torch.zeros(n + 1, heads, dtype=torch.float64, device="cuda"), torch.zeros(n + 1, heads, dtype=torch.float64, device="cuda")
        at = torch.where(inside, which, n).view(-1)
        tab.index_add_(0, at, ds.sum(0).permute(1, 2, 0).reshape(-1, heads))
        rm.index_add_(0, at, err.sum(0).permute(1, 2, 0).reshape(-1, heads) / u)
        res["dtable"] = (tab[:n], rm[:n])
    return res


def _run(c, **over):
    from passion_amd import ops
    c = {**c, **over}
    on = lambda t: None if t is None else t.cuda()
    leaves = {n: on(c[n]).detach().requires_grad_() for n in ("q", "k", "v", "table") if c[n] is not None}
    out = ops.rel_attention(leaves["q"], leaves["k"], leaves["v"], leaves.get("table"), c["grid"], on(c["buckets"]), on(c["mask"]), c["scale"], c["q0"])
    grads = torch.autograd.grad(out, list(leaves.values()), on(c["dout"]))
    with torch.no_grad():
        again = ops.rel_attention(leaves["q"], leaves["k"], leaves["v"], leaves.get("table"), c["grid"], on(c["buckets"]), on(c["mask"]), c["scale"], c["q0"])
    assert torch.equal(out, again)
    return dict(out=out.detach(), **{"d" + n: g for n, g in zip(leaves, grads)})


def _check(c):
    got, want = _run(c), _reference(c)
    assert set(got) == set(want)
    for n in got:
        w, room = want[n]
        near(got[n], w, U[c["q"].dtype], n, room=room + 1e-6 * room.mean())


BOTH = pytest.mark.parametrize("dt", [F, H])


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid,groups,B,heads,Hkv,D,mask", [((3, 4, 5), 1, 2, 4, 4, 32, None), ((5, 5, 5), 1, 1, 8, 8, 64, None), ((8, 8, 8), 1, 2, 8, 8, 64, "runs"),
                                                          ((5, 5, 5), 3, 2, 8, 2, 64, "runs"), ((2, 3), 7, 3, 4, 1, 8, "random"), ((7,), 30, 1, 2, 2, 128, None),
                                                          ((1, 1, 1), 40, 1, 4, 4, 24, None), ((9, 9, 6), 1, 1, 4, 2, 96, "empty"), ((8, 8, 9), 1, 5, 8, 8, 128, None)])
def test_grids(grid, groups, B, heads, Hkv, D, mask, dt):
    """offsets in a small box, cells repeated by further modalities"""
    n = math.prod(grid) * groups
    _check(_make(B, n, n, heads, Hkv, D, dt, grid, mask=mask))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("Nq,Nk,q0,more,D", [(1, 1, 0, 0, 64), (2, 2, 0, 3, 64), (31, 33, 1, 0, 32), (64, 64, 0, 0, 64), (65, 129, 64, 0, 128), (20, 200, 100, 13, 40), (200, 200, 0, 0, 72),
                                              (33, 1000, 7, 0, 64), (1000, 1000, 0, 9, 64), (90, 31, 5, 100, 64), (500, 1, 0, 500, 64)])
def test_lines(Nq, Nk, q0, more, D, dt):
    """1D rasters: windows at both ends, ragged lengths, queries that start inside the keys or behind them"""
    _check(_make(2, Nq, Nk, 4, 2, D, dt, (max(Nk, q0 + Nq) + more,), nb=32, q0=q0))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid,Nq,Nk,q0,nb", [((40, 40), 1600, 1600, 0, None), ((40, 40), 70, 900, 400, 12), ((2500,), 300, 2600, 2400, 64), ((17, 16, 16), 100, 500, 33, 700)])
def test_large_boxes(grid, Nq, Nk, q0, nb, dt):
    """more offsets than LDS holds, 1D rasters that wrap around, few and many buckets"""
    _check(_make(1, Nq, Nk, 4, 4, 64, dt, grid, nb=nb, q0=q0, mask="random"))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("Nq,Nk,heads,Hkv,D,mask", [(1, 1, 1, 1, 8, None), (100, 100, 8, 8, 64, "random"), (130, 70, 6, 3, 48, "empty"), (3, 500, 4, 4, 128, "runs"), (257, 300, 3, 1, 16, None),
                                                    (64, 2048, 16, 16, 64, "runs")])
def test_without_a_table(Nq, Nk, heads, Hkv, D, mask, dt):
    _check(_make(2, Nq, Nk, heads, Hkv, D, dt, mask=mask))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("Nq", [1, 2, 4, 5, 16, 17])
@pytest.mark.parametrize("Nk,heads,Hkv,B", [(1, 4, 4, 3), (63, 8, 2, 2), (64, 8, 8, 1), (65, 8, 1, 2), (1000, 8, 2, 5), (5003, 4, 1, 1), (20000, 8, 8, 1)])
def test_few_queries(Nq, Nk, heads, Hkv, B, dt):
    """one new token and a few, split over the keys, heads of a key / value head in one tile"""
    Nq = min(Nq, Nk)
    c = _make(B, Nq, Nk, heads, Hkv, 64, dt, (Nk + 5,), nb=32, q0=Nk - Nq, mask="random" if B > 1 else None)
    if Nk < 6000:
        return _check(c)
    from passion_amd import ops
    out = ops.rel_attention(*(c[n].cuda() for n in ("q", "k", "v", "table")), c["grid"], c["buckets"].cuda(), q_start=c["q0"])
    w, room = _reference(c, grads=False)["out"]
    near(out, w, U[dt], "out", room=room)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid,B,Nq,Nk,heads,Hkv,D,nb,q0,mask", [((1700,), 1, 200, 1500, 2, 2, 128, 8, 190, None), ((1700,), 1, 1500, 200, 2, 1, 64, None, 0, None),
                                                                   ((1100,), 2, 1100, 700, 2, 1, 40, 32, 0, "runs"), ((1300,), 1, 1300, 1300, 1, 1, 64, None, 0, "runs"),
                                                                   ((300,), 3, 290, 257, 1, 1, 16, 12, 10, "empty"), ((10, 10, 10), 1, 1000, 1000, 2, 1, 96, None, 0, "runs"),
                                                                   ((40, 40), 1, 700, 1500, 1, 1, 32, 12, 0, "random"), (None, 1, 900, 1100, 2, 1, 72, None, 0, "runs")])
def test_few_tiles_of_long_rows(grid, B, Nq, Nk, heads, Hkv, D, nb, q0, mask, dt):
    """the backward in parts of the keys (dQ) and of the queries (dK, dV, the table's gradient), the parts of unequal lengths, some without a valid key"""
    _check(_make(B, Nq, Nk, heads, Hkv, D, dt, grid, nb, q0, mask))


@pytest.mark.gpu
@pytest.mark.parametrize("grid,B,heads,Hkv,D", [((7, 10, 8), 1, 8, 4, 128), ((7, 10, 8), 1, 8, 4, 96), ((6, 9, 10), 1, 8, 4, 96), ((7, 9, 9), 1, 8, 4, 128), ((560,), 4, 8, 8, 64),
                                                 ((560,), 4, 8, 2, 64), ((2, 14, 20), 3, 8, 8, 64), ((6, 10, 12), 1, 12, 12, 112)])
def test_ragged_last_block_in_every_workgroup(grid, B, heads, Hkv, D):
    """more workgroups than compute units, so that some share a SIMD, with a last key block of 28 to 60 tokens: once, a valid key of it was stored as zeros by the
    workgroups that came second to their SIMD (its bit of the mask was taken by a 64-bit vector shift by the last register)"""
    N = math.prod(grid)
    _check(_make(B, N, N, heads, Hkv, D, H, grid))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("B", [1, 40])
def test_many_workgroups_of_four(B, dt):
    """enough tiles for four wavefronts a workgroup, on every way to the bias"""
    _check(_make(B, 260 if B > 1 else 4100, 260 if B > 1 else 300, 8, 4, 32, dt, (4100,), nb=16))
    _check(_make(B, 252, 252, 8, 8, 64, dt, (6, 7, 6), mask="empty" if B > 1 else None))
    _check(_make(B, 200, 200, 8, 8, 32, dt))


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("D", [96, 128])
@pytest.mark.parametrize("grid,nb,N", [((1003,), 32, 1000), ((8, 8, 8), None, 1000), ((10, 10, 10), None, 1000), (None, None, 1000)])
def test_wide_heads_by_workgroups_of_four(grid, nb, N, D, dt):
    """widths over 64 in enough tiles for four wavefronts a workgroup in every kernel (the registers that the width leaves differ by their number)"""
    _check(_make(4, N, N, 8, 8, D, dt, grid, nb=nb, mask="runs"))


@pytest.mark.gpu
@pytest.mark.parametrize("grid,B,Nq,Nk,heads,Hkv,D,nb,q0,mask", [((5, 5, 5), 1, 125, 125, 8, 8, 64, None, 0, None), ((500,), 2, 500, 500, 4, 2, 128, 32, 0, "runs"),
                                                                   ((40, 40), 1, 300, 1600, 2, 2, 32, 12, 100, "random"), (None, 1, 700, 700, 2, 1, 96, None, 0, None),
                                                                   ((3000,), 3, 1, 3000, 8, 2, 64, 32, 2999, "random"), ((6, 7, 8), 2, 336, 336, 4, 4, 8, None, 0, None)])
def test_f32_is_f32(grid, B, Nq, Nk, heads, Hkv, D, nb, q0, mask):
    """the Euclidean norm of the error, where independent roundings add as squares.  A score sums D <= 128 products one after another: sqrt(128) * 2^-24 of partial sums of
    order 3, 2e-6 of error, and so much relative error in a probability; products with v, dout, q, k add as much again, and dP - delta cancels up to a few times.  1e-5 and
    3e-5 of the norm leave a factor of a few; operands of 11 bits would be off by sqrt(128) * 2^-12 / 3 = 1e-3"""
    c = _make(B, Nq, Nk, heads, Hkv, D, F, grid, nb=nb, q0=q0, mask=mask)
    got, want = _run(c), _reference(c)
    for n in got:
        w = want[n][0]
        off = float((got[n].double() - w).norm() / w.norm())
        assert off <= (1e-5 if n in ("out", "dv") else 3e-5), (n, off)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid", [(300,), (5, 6, 10), (40, 40), None])
@pytest.mark.parametrize("Nq", [1, 300])
def test_masked_keys_may_hold_anything(grid, Nq, dt):
    c = _make(2, Nq, 300, 4, 2, 64, dt, grid, mask="random")
    clean = _run(c)
    bad = {n: c[n].clone() for n in ("k", "v")}
    for n, x in (("k", float("nan")), ("v", float("inf"))):
        bad[n][~c["mask"]] = x
    got = _run(c, **bad)
    for n in got:
        assert torch.equal(got[n], clean[n]), n
    as_bytes = _run(c, mask=c["mask"].to(torch.uint8) * 3)
    assert torch.equal(as_bytes["out"], clean["out"])


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("low", [float("-inf"), "lowest"])
@pytest.mark.parametrize("grid,Nq", [((150,), 150), ((5, 5, 6), 150), ((50, 50), 150), ((150,), 1)])
def test_excluded_entries(grid, Nq, low, dt):
    """entries of -inf and of the type's lowest value take their pairs out; a query all of whose pairs are out gives 0 and no gradient"""
    c = _make(1, Nq, 150, 2, 2, 32, dt, grid, nb=10, q0=150 - Nq)
    c["table"][3:7, 0] = torch.finfo(dt).min if low == "lowest" else low
    c["table"][:, 1] = torch.finfo(dt).min if low == "lowest" else low
    c["buckets"][::7] = -1                      # no bias there: those pairs stay
    c["buckets"][1::7] = 10
    _check(c)
    c["buckets"] = c["buckets"].clamp(0, 9)
    got = _run(c)
    assert float(got["out"][:, :, 1].abs().max()) == 0 and all(torch.isfinite(t).all() for t in got.values())
    assert float(got["dtable"][:, 1].abs().max()) == 0 and float(got["dq"][:, :, 1].abs().max()) == 0
    _check(c)


@pytest.mark.gpu
@BOTH
def test_large_scores(dt):
    """scores over hundreds of log2 units: the reference that moves only when a block exceeds it by 2^8 stays exact.  (A score of size 300 carries 300 * 2^-24
    * 16 of accumulated error in f32: within U)"""
    c = _make(1, 300, 300, 2, 2, 64, dt, (300,), nb=8)
    c["q"] = c["q"] * 6
    c["table"] = c["table"] * 30
    _check(c)


@pytest.mark.gpu
@BOTH
def test_views_read_in_place(dt):
    """packed (B, N, 3, H, D) projections, heads-first storage, keys broadcast over the batch, misaligned rows"""
    from passion_amd import ops
    c = _make(2, 100, 100, 4, 4, 32, dt, (4, 5, 5))
    want = _run(c)
    packed = torch.stack([c["q"], c["k"], c["v"]], 2).cuda().requires_grad_()
    out = ops.rel_attention(*packed.unbind(2), c["table"].cuda(), c["grid"])
    (g,) = torch.autograd.grad(out, packed, c["dout"].cuda())
    assert torch.equal(out, want["out"]) and all(torch.equal(g[:, :, i], want[n]) for i, n in enumerate(("dq", "dk", "dv")))
    heads_first = {n: c[n].cuda().transpose(1, 2).contiguous().transpose(1, 2) for n in "qkv"}
    got = _run(c, **heads_first)
    assert all(torch.equal(got[n], want[n]) for n in want)
    wide = torch.zeros(2, 100, 4, 33, dtype=dt, device="cuda")
    wide[..., 1:] = c["q"].cuda()
    got = _run(c, q=wide[..., 1:], dout=c["dout"].transpose(1, 2).contiguous().transpose(1, 2))
    assert all(torch.equal(got[n], want[n]) for n in want)
    one = {n: c[n][:1].expand(2, -1, -1, -1) for n in "kv"}
    k1 = c["k"][:1].cuda().requires_grad_()
    out = ops.rel_attention(c["q"].cuda(), k1.expand(2, -1, -1, -1), one["v"].cuda(), c["table"].cuda(), c["grid"])
    full = _run(c, **one)
    assert torch.equal(out, full["out"])
    (gk,) = torch.autograd.grad(out, k1, c["dout"].cuda())
    near(gk, full["dk"].double().sum(0, keepdim=True), 2.0 ** -8, "dk of a broadcast key")


@pytest.mark.gpu
@BOTH
def test_strides_of_dimensions_of_one(dt):
    """a batch of one sliced out of odd rows, one token out of wider ones, one head out of a larger tensor: strides that no step takes may be anything"""
    from passion_amd import ops
    c = _make(1, 100, 100, 8, 8, 64, dt)
    want = _run(c)
    cut = {}
    for n in ("q", "k", "v", "dout"):
        store = torch.zeros(3, 100 * 512 + 3, dtype=dt, device="cuda")
        store[0, :51200] = c[n].cuda().view(-1)
        cut[n] = store[:, :51200].unflatten(1, (100, 8, 64))[0:1]
        assert cut[n].stride(0) == 51203
    got = _run(c, **cut)
    assert all(torch.equal(got[n], want[n]) for n in want)
    c = _make(1, 1, 1, 8, 8, 64, dt)
    want = _run(c)
    for width in (516, 1 << 24):
        wide = {n: torch.as_strided(c[n].cuda().view(-1), (1, 1, 8, 64), (width + 1, width + 3, 64, 1)) for n in ("q", "k", "v")}
        got = _run(c, **wide)
        assert all(torch.equal(got[n], want[n]) for n in want)
    c = _make(2, 40, 40, 1, 1, 32, dt)
    want = _run(c)
    one = {n: torch.as_strided(c[n].cuda().view(-1), (2, 40, 1, 32), (1280, 32, 33, 1)) for n in ("q", "k", "v")}
    got = _run(c, **one)
    assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.gpu
@pytest.mark.parametrize("grid", [(5, 5, 5), (125,), (70, 70)])
def test_table_types_meet_either_operand_type(grid):
    for dt, tdt in ((F, H), (H, F)):
        c = _make(2, 125, 125, 4, 4, 64, dt, grid, table_dt=tdt)
        _check(c)
        assert _run(c)["dtable"].dtype == tdt


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid,Nq", [((6, 6, 6), 216), ((500,), 500), ((40, 40), 500), ((500,), 2)])
def test_repeats_and_streams(grid, Nq, dt):
    Nk = max(Nq, 216)
    c = _make(3, Nq, Nk, 8, 2, 64, dt, grid, nb=None if grid == (6, 6, 6) else 32, mask="random")
    a = _run(c)
    for _ in range(3):
        b = _run(c)
        assert all(torch.equal(a[n], b[n]) for n in a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(c)
    torch.cuda.synchronize()
    assert all(torch.equal(a[n], b[n]) for n in a)


@pytest.mark.gpu
@pytest.mark.parametrize("grid,Nq,Nk", [((6, 6, 6), 216, 216), ((300,), 300, 300), ((40, 40), 64, 500), ((5000,), 1, 5000)])
def test_captured_and_replayed(grid, Nq, Nk):
    from passion_amd import ops
    q0 = Nk - Nq if grid != (6, 6, 6) else 0
    sets = []
    for s in range(3):
        c = _make(2, Nq, Nk, 8, 2, 64, H, grid, nb=24, q0=q0, mask="random", seed=s)
        sets.append([c[n].cuda() for n in ("q", "k", "v", "dout", "table", "mask", "buckets")])
    statics = [t.clone() for t in sets[0]]

    def step(q, k, v, dout, table, mask, buckets):
        ins = [t.detach().requires_grad_() for t in (q, k, v, table)]
        out = ops.rel_attention(*ins, grid, buckets, mask, q_start=q0)
        return (out, *torch.autograd.grad(out, ins, dout))

    replayed(lambda: step(*statics), statics, sets, step)


@pytest.mark.gpu
def test_two_captured_graphs_share_nothing():
    """two graphs with split forwards, replayed in turn and on two streams at once"""
    from passion_amd import ops
    cs = [[t.cuda() for t in (c["q"], c["k"], c["v"], c["table"], c["buckets"])] for c in (_make(2, 1, 4000, 8, 2, 64, H, (4000,), nb=32, q0=3999, seed=s) for s in (1, 2))]
    call = lambda c: ops.rel_attention(*c[:4], (4000,), c[4], q_start=3999)
    with torch.no_grad():
        want = [call(c) for c in cs]
        torch.cuda.synchronize()
        graphs, outs = [], []
        for c in cs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(call(c))
            graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cs]
    for _ in range(5):
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.gpu
@pytest.mark.parametrize("grid", [(3, 4, 4), (48,)])
def test_gradient_against_differences(grid):
    """f32, central differences with step 1e-2 along a random direction: third-derivative terms of 1e-4 and 2^-24 * sum / step of rounding, against 1 % of the slope's size"""
    from passion_amd import ops
    c = {n: t.cuda() if torch.is_tensor(t) else t for n, t in _make(2, 48, 48, 4, 2, 32, F, grid).items()}
    f = lambda t: (ops.rel_attention(t["q"], t["k"], t["v"], t["table"], grid).double() * c["dout"].double()).sum()
    leaves = {n: c[n].clone().requires_grad_() for n in ("q", "k", "v", "table")}
    grads = dict(zip(leaves, torch.autograd.grad(f(leaves), list(leaves.values()))))
    g = torch.Generator(device="cuda").manual_seed(3)
    for n in leaves:
        way = torch.randn(c[n].shape, generator=g, device="cuda")
        with torch.no_grad():
            quotient = float(f({**c, n: c[n] + 1e-2 * way}) - f({**c, n: c[n] - 1e-2 * way})) / 2e-2
        assert abs(quotient - float((grads[n] * way).sum())) < 1e-2 * float(grads[n].norm()), n


@pytest.mark.gpu
def test_far_end_of_a_long_cache():
    """keys and values whose element offsets pass 2^31: only the last ones take part; the same as on a short copy of them"""
    from passion_amd import ops
    Nk, Hkv, D = (1 << 22) + 77, 8, 64
    k, v = (torch.zeros(1, Nk, Hkv, D, dtype=H, device="cuda") for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    for t in (k, v):
        t[:, -100:] = torch.randn(1, 100, Hkv, D, generator=g, device="cuda").to(H)
    q = torch.randn(1, 1, Hkv, D, generator=g, device="cuda").to(H)
    mask = torch.zeros(1, Nk, dtype=torch.bool, device="cuda")
    mask[:, -100:] = True
    got = ops.rel_attention(q, k, v, key_mask=mask)
    want = ops.rel_attention(q, k[:, -100:].contiguous(), v[:, -100:].contiguous())
    assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid,B,Nq,Nk,heads,Hkv,D,nb,q0,mask", [((1,), 2, 300, 700, 2, 1, 16, None, 0, "random"), ((2, 2), 1, 1000, 257, 2, 2, 32, None, 3, None),
                                                                   ((1, 3, 2), 3, 130, 900, 4, 4, 64, 4, 1, "runs"), ((4, 4, 4), 1, 700, 300, 1, 1, 40, None, 30, "empty"),
                                                                   ((5, 13), 1, 300, 300, 2, 1, 8, None, 7, None), ((3,), 2, 2, 1000, 2, 2, 16, None, 4, None),
                                                                   ((3, 9), 2, 1000, 20, 2, 2, 16, 9, 0, "random")])
def test_many_copies_of_few_cells(grid, B, Nq, Nk, heads, Hkv, D, nb, q0, mask, dt):
    """grids smaller than a tile: a pass of the table's sums takes several copies of the cells, and the copies fold afterwards"""
    _check(_make(B, Nq, Nk, heads, Hkv, D, dt, grid, nb=nb, q0=q0, mask=mask))


@pytest.mark.gpu
@pytest.mark.parametrize("cells", [1, 2, 3])
def test_the_table_s_gradient_of_a_long_sequence_over_few_cells(cells):
    """50000 tokens over one cell are 2.5e9 (query copy, key copy) pairs: once, they were counted in 32 bits and keys were read before their start.  Tolerance as above,
    the 64-bit sums taken in ranges of queries"""
    from passion_amd import ops
    N, D = 50000, 8
    c = {n: t.cuda() if torch.is_tensor(t) else t for n, t in _make(1, N, N, 1, 1, D, H, (cells,)).items()}
    table = c["table"].clone().requires_grad_()
    (got,) = torch.autograd.grad(ops.rel_attention(c["q"], c["k"], c["v"], table, (cells,)), table, c["dout"])
    q, k, v, do = (c[n][0, :, 0].double() for n in ("q", "k", "v", "dout"))
    u, cell = U[H], torch.arange(N, device="cuda") % cells
    want, room = (torch.zeros(2 * cells - 1, 1, dtype=torch.float64, device="cuda") for _ in range(2))
    step = 1200                                       # a multiple of the cells
    for a in range(0, N, step):
        rows = slice(a, min(N, a + step))
        off = cell[rows, None] - cell[None] + cells - 1
        p = torch.softmax(q[rows] @ k.t().contiguous() * c["scale"] + c["table"][:, 0].double()[off], 1)
        dp = do[rows] @ v.t().contiguous()
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        err = u * ds.abs() + p * (do[rows].abs() * u * (p @ v.abs() + (p @ v).abs())).sum(1, keepdim=True)
        for x in range(2 * cells - 1):
            at = off == x
            want[x] += ds[at].sum()
            room[x] += err[at].sum() / u
    near(got, want, u, "dtable", room=room)


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid,B,N,heads,D,nb", [((700,), 2, 700, 4, 64, 32), ((9, 9, 9), 1, 729, 4, 32, None), ((5, 5, 5), 4, 250, 4, 64, None), ((40, 40), 1, 1600, 2, 128, 12)])
def test_a_frozen_table_pays_nothing_for_its_gradient(grid, B, N, heads, D, nb, dt):
    """table without requires_grad: the other gradients bit for bit the same, and no memory for the partial sums (an eighth of a byte for every score of a 1D
    raster's heads, four bytes for every pair of a grid's cells)"""
    from passion_amd import ops
    c = _make(B, N, N, heads, heads, D, dt, grid, nb=nb, mask="random")
    want = _run(c)
    on = {n: c[n].cuda() for n in ("q", "k", "v", "dout", "table", "mask")}
    ins = [on[n].requires_grad_() for n in ("q", "k", "v")]
    buckets = None if nb is None else c["buckets"].cuda()
    peak = {}
    for learned in (True, False):
        table = on["table"].clone().requires_grad_(learned)
        out = ops.rel_attention(*ins, table, grid, buckets, on["mask"], c["scale"])
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        stats = lambda which: torch.cuda.memory_stats()["requested_bytes.all." + which]        # (what is counted as allocated includes whole cached blocks, up to 1 MB more)
        before = stats("current")
        grads = torch.autograd.grad(out, ins + [table] * learned, on["dout"])
        torch.cuda.synchronize()
        peak[learned] = stats("peak") - before
        assert all(torch.equal(g, want[n]) for n, g in zip(("dq", "dk", "dv"), grads))
        del out, grads
    slab = B * heads * N * N / 8 if len(grid) == 1 else 4 * heads * min(N, math.prod(grid)) ** 2
    assert peak[True] - peak[False] >= 0.9 * slab


@pytest.mark.gpu
def test_more_query_rows_than_a_launch_has_sixteenths_of_its_threads():
    """2^25 + 100 queries of 8 heads against 200 keys: the pass over out and dout before the backward takes 16 threads a row, past 2^32 in one launch.  All queries but the
    last hundred are 0 with a gradient of 0, so the gradients are those of the short call"""
    from passion_amd import ops
    N, n = (1 << 25) + 100, 100
    c = {k: v.cuda() if torch.is_tensor(v) else v for k, v in _make(1, n, 200, 8, 8, 8, H, seed=5).items()}
    wide = {m: torch.zeros(1, N, 8, 8, dtype=H, device="cuda") for m in ("q", "dout")}
    for m in wide:
        wide[m][:, -n:] = c[m]
    long = [t.requires_grad_() for t in (wide["q"], c["k"].clone(), c["v"].clone())]
    out = ops.rel_attention(*long)
    dq, dk, dv = torch.autograd.grad(out, long, wide["dout"])
    assert not bool(dq[:, :-n].any())
    want = _reference(c)
    for name, got in (("out", out[:, -n:]), ("dq", dq[:, -n:]), ("dk", dk), ("dv", dv)):
        near(got, want[name][0], U[H], name, room=want[name][1])


@pytest.mark.gpu
def test_more_offsets_than_a_launch_has_sixteenths_of_its_threads():
    """a line of 2^27 + 1 places, 200 tokens on it: the expansion of the buckets and the sums by offset run over 2^28 + 1 offsets; the same as on a line of 300"""
    from passion_amd import ops
    L, n = (1 << 27) + 1, 300
    c = {k: v.cuda() if torch.is_tensor(v) else v for k, v in _make(1, 200, 200, 1, 1, 16, H, (n,), nb=6, seed=6).items()}
    step = lambda grid, buckets: torch.autograd.grad(ops.rel_attention(*leaves, grid, buckets), leaves, c["dout"])
    leaves = [c[m].clone().requires_grad_() for m in ("q", "k", "v", "table")]
    want = step((n,), c["buckets"])
    buckets = torch.zeros(2 * L - 1, dtype=torch.int32, device="cuda")
    buckets[L - n:L + n - 1] = c["buckets"]
    got = step((L,), buckets)
    assert all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))
    near(got[3], want[3].double(), 2.0 ** -8, "dtable")


@pytest.mark.gpu
@BOTH
@pytest.mark.parametrize("grid,Nq,Nk,q0,nb", [((200, 200, 200), 300, 300, 0, 7), ((300, 4, 500), 130, 700, 597900, 64), ((30, 40, 50), 700, 90, 59500, None), ((5000,), 64, 64, 4970, 12),
                                              ((6, 7, 8), 40, 336, 320, None), ((6, 7, 8), 336, 41, 100, None), ((20, 30), 74, 600, 570, 9), ((20000003,), 100, 130, 40, 5)])
def test_few_tokens_of_a_large_grid(grid, Nq, Nk, q0, nb, dt):
    """queries on few of the cells, and such that go round the raster's end: the sums by offset walk the tokens' cells alone (once, all cells for every offset: 40 s over
    200^3 cells by count, hours at the largest grid that is taken)"""
    _check(_make(1, Nq, Nk, 2, 1, 16, dt, grid, nb=nb, q0=q0, mask="random"))


@pytest.mark.gpu
def test_no_tokens():
    from passion_amd import ops
    for B, Nq, Nk in ((0, 3, 3), (2, 0, 4), (2, 4, 0)):
        t = {n: torch.zeros(B, m, 2, 16, device="cuda", requires_grad=True) for n, m in (("q", Nq), ("k", Nk), ("v", Nk))}
        table = torch.zeros(9, 2, device="cuda", requires_grad=True)
        out = ops.rel_attention(t["q"], t["k"], t["v"], table, 5)
        assert out.shape == (B, Nq, 2, 16) and float(out.detach().abs().sum()) == 0
        out.sum().backward()
        assert float(table.grad.abs().sum()) == 0 and t["k"].grad.shape == t["k"].shape


@pytest.mark.gpu
def test_the_framework_s_attention_is_the_form_without_positions():
    """ops.attention on the packed projections and rel_attention without a table, both bf16: the same probabilities up to their roundings"""
    from passion_amd import ops
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(2, 300, 3 * 8 * 64, generator=g).to(H).cuda()
    a = ops.attention(qkv, 8, 0.125)
    b = ops.rel_attention(*qkv.view(2, 300, 3, 8, 64).unbind(2), scale=0.125)
    assert float((a.view_as(b).float() - b.float()).abs().max()) < 2.0 ** -6


def test_relative_buckets():
    from passion_amd import ops
    b, n = ops.relative_buckets(20, 8, 16)
    assert n == 8 and b.shape == (39,) and b.dtype == torch.int32
    mid = 19
    assert b[mid] == 0 and b[mid - 1] == 1 and b[mid + 1] == 5 and int(b.max()) == 7 and b[0] == 3
    assert (b[:mid + 1].flip(0).diff() >= 0).all() and (b[mid + 1:].diff() >= 0).all()
    b3, n3 = ops.relative_buckets((3, 1, 4), 4)
    one, _ = ops.relative_buckets(4, 4)
    assert n3 == 16 and b3.shape == (5 * 7,) and torch.equal(b3.view(5, 7)[2], one)
    for bad in ((0, 8), ((2, 2, 2, 2), 8), (5, 3), (5, 0)):
        with pytest.raises(ValueError):
            ops.relative_buckets(*bad)


def test_refusals():
    from passion_amd import _lib, ops
    q, k = torch.zeros(2, 5, 4, 16), torch.zeros(2, 7, 2, 16)
    t = torch.zeros(13, 4)
    ok = dict(q=q, k=k, v=k, table=t, grid=7)
    for change in (dict(v=k[:, :6]), dict(k=k[:1], v=k[:1]), dict(q=q.half()), dict(q=q.bfloat16()), dict(q=q[..., :12], k=k[..., :12], v=k[..., :12]), dict(k=k[:, :, :0], v=k[:, :, :0]),
                   dict(k=torch.zeros(2, 7, 3, 16), v=torch.zeros(2, 7, 3, 16)), dict(grid=None), dict(grid=8), dict(grid=(0, 7)), dict(grid=(1, 1, 1, 7)), dict(table=t[:, :3]),
                   dict(table=t.double()), dict(buckets=torch.zeros(12, dtype=torch.int32)), dict(buckets=torch.zeros(13)), dict(table=None, grid=None, buckets=torch.zeros(13).int()),
                   dict(key_mask=torch.ones(2, 5, dtype=torch.bool)), dict(key_mask=torch.ones(2, 7)), dict(q_start=-1), dict(q=q[0]), dict(grid=(2 ** 16, 2 ** 16))):
        with pytest.raises(ValueError):
            ops.rel_attention(**{**ok, **change})
    with pytest.raises(_lib.PassionHipError):
        ops.rel_attention(**ok)


def test_c_entry_refuses_on_the_host():
    import ctypes
    from passion_amd import _lib
    lib = _lib.load()
    S = (ctypes.c_int64 * 3)(1024, 64, 8)
    odd = (ctypes.c_int64 * 3)(1024, 63, 8)

    def fwd(q=256, sq=S, dt=0, B=1, Nq=4, Nk=4, H=2, Hkv=2, D=8, g=(1, 1, 4), q0=0, table=256, tdt=0, buckets=None, nb=7, out=256, ws=256):
        return lib.passion_rel_attn_fwd(q, sq, 256, S, 256, S, dt, B, Nq, Nk, H, Hkv, D, *g, q0, table, tdt, buckets, nb, None, 1.0, out, None, ws, None)

    for bad in (dict(dt=2), dict(B=0), dict(B=65536), dict(Nq=0), dict(Nk=0), dict(H=3), dict(D=12), dict(D=136), dict(g=(1, 0, 4)), dict(nb=6), dict(q0=-1), dict(tdt=5), dict(q=None),
                dict(out=None), dict(g=(40000, 40000, 1), buckets=256)):
        assert fwd(**bad) == -1003, bad
    assert fwd(q=260) == -1005 and fwd(sq=odd) == -1005 and fwd(ws=264) == -1005
    size = lambda *a: lib.passion_rel_attn_workspace_floats(*a)
    assert size(0, 0, 1, 4, 4, 2, 2, 12, 1, 1, 4, 0, 1, 0, 7) == -1003
    assert size(1, 1, 1, 400, 400, 2, 2, 64, 1, 1, 400, 0, 1, 0, 799) > 0


def test_strides_of_dimensions_of_one_on_the_host():
    """rows that are there to be read in place stay as they are; the C entry looks at no stride of a dimension of one (its next refusal is the missing workspace)"""
    import ctypes
    from passion_amd import _lib, ops
    t = torch.zeros(3, 100 * 512 + 3)[:, :51200].unflatten(1, (100, 8, 64))[0:1]
    if t.data_ptr() % 16 == 0:
        assert ops._rel_view(t).data_ptr() == t.data_ptr()
    odd = lambda n: torch.as_strided(torch.zeros(64 * 9 * 2), (n, 1, 1, 64), (67, 33, 5, 1))
    assert ops._rel_view(odd(1)).stride(0) == 67 and ops._rel_view(odd(2)).stride(0) == 64
    lib = _lib.load()
    fwd = lambda B, *strides: lib.passion_rel_attn_fwd(256, *[(ctypes.c_int64 * 3)(*strides), 256] * 2, (ctypes.c_int64 * 3)(*strides), 0, B, 64, 64, 1, 1, 64, 1, 1, 64, 0,
                                                       256, 0, None, 127, None, 1.0, 256, None, None, None)
    assert fwd(2, 51203, 64, 64) == -1005 and fwd(1, 51204, 65, 64) == -1005 and fwd(1, 51204, 1 << 24, 64) == -1005
    assert fwd(1, 51203, 64, 7) == -1003


def test_workspace_sizes_past_32_bits():
    """the partials of the table's gradient, counted on the host: products of batch, heads and lengths past 2^31"""
    from passion_amd import _lib
    size = lambda B, N, M, H, grid: _lib.load().passion_rel_attn_workspace_floats(1, 1, B, N, M, H, H, 8, *grid, 0, 1, 0, math.prod(2 * g - 1 for g in grid))
    assert size(40000, 33, 33, 60000, (1, 1, 40)) >= 40000 * 60000 * 2 * (64 + 32)                    # 1D: batch x heads x key tiles x (queries in blocks + 32)
    assert size(1, 1 << 22, 1 << 22, 1024, (4, 1, 1 << 20)) >= 1024 << 44                               # dense: heads x query cells x key cells
    assert size(1, 1 << 22, 10, 1024, (4, 1, 1 << 20)) >= (1024 << 22) * 64


def test_a_line_is_chosen_in_64_bits():
    """queries q_start .. q_start + Nq - 1 with a last one past 2^31 go round a line of 40 places: the sums of a line (about a float a query) are not theirs"""
    from passion_amd import _lib
    size = lambda q0: _lib.load().passion_rel_attn_workspace_floats(1, 1, 1, 1 << 30, 1, 1, 1, 8, 1, 1, 40, q0, 1, 0, 79)
    delta = 1 << 30
    assert delta < size(1 << 29) < delta + (1 << 25) and size(1 << 30) == size(1 << 29)


def test_workspace_without_the_table_s_gradient():
    from passion_amd import _lib
    size = lambda backward, grid, N, nb: _lib.load().passion_rel_attn_workspace_floats(1, backward, 1, N, N, 8, 8, 64, *grid, 0, 1, 1, nb)
    for grid, N, slab in (((20, 20, 20), 8000, 8 * 8000 * 8000), ((1, 1, 65536), 65536, 8 * 65536 * 65536 // 32)):
        assert size(1, grid, N, 32) >= slab
        offsets = math.prod(2 * g - 1 for g in grid)
        assert 0 < size(2, grid, N, 32) <= 8 * (offsets + N) + 256


def test_a_gradient_of_too_many_buckets_over_too_many_offsets_is_refused():
    """the last sum is a product of the two: at the largest sizes that are taken otherwise it would run for minutes.  Without the gradient, or with few buckets, the call goes on (to the next
    refusal: tensors that are not on a GPU)"""
    from passion_amd import _lib, ops
    lib = _lib.load()
    size = lambda backward, side, nb, heads=8: lib.passion_rel_attn_workspace_floats(1, backward, 1, 100, 100, heads, heads, 8, side, side, side, 0, 1, 1, nb)
    assert size(1, 400, 300) == -1003 and size(1, 200, 10 ** 6) == -1003
    assert size(2, 400, 300) > 0 and size(0, 400, 300) > 0 and size(1, 400, 256) > 0 and size(1, 200, 10 ** 4) > 0 and size(1, 20, 30000) > 0
    q = torch.zeros(1, 5, 2, 8)
    buckets = torch.zeros(1, dtype=torch.int32).expand(599 ** 3)
    for nb, learned in ((300, True), (300, False), (200, True)):
        table = torch.zeros(nb, 2, requires_grad=learned)
        with pytest.raises(ValueError if learned and nb == 300 else _lib.PassionHipError):
            ops.rel_attention(q, q, q, table, (300, 300, 300), buckets)
