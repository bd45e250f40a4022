"""ops.topk_distill (csrc/distill.hip) against the definition in 64 bits: class counts on both sides of every layout, odd rows that start anywhere, repeated
and missing indices, masked classes, and its refusals.

Tolerances: the log-sum-exp is a running f32 sum of V <= 130001 terms over at least 256 threads (at most 64 vectors of 8 a thread, 8 joins): below 600 additions
in sequence, 600 * 2^-24 = 3.6e-5 relative to the sum in the worst case and its square root, 1.5e-6, in the typical one; log2 of it and z carry 2^-24 of their
size (below 64 in these units): 4e-6.  The loss sums K shares of such terms: 5e-6 * T^2 * 64 with room.  The gradient g T (q - p): q has the error of
exp2(z - lse), 1e-5 relative, p the same: 2e-5 of the largest share, and one rounding to its type."""
import pytest
import torch

from _op_util import near, replayed

F, H = torch.float32, torch.bfloat16


def _make(R, V, K, dt, seed=0, tdt=F, idt=torch.int64):
    g = torch.Generator().manual_seed(seed)
    s = (3 * torch.randn(R, V, generator=g)).to(dt)
    t = (3 * torch.randn(R, K, generator=g)).to(tdt)
    i = torch.randint(0, V, (R, K), generator=g)
    return s, t, i.to(idt), torch.rand(R, generator=g)


def _reference(s, t, i, g, T):
    R, V = s.shape
    leaf = s.double().clone().requires_grad_()
    ok = (i >= 0) & (i < V) & (t != float("-inf"))
    live = ok.any(1)
    tv = torch.where(ok, t.double() / T, float("-inf"))
    tv = torch.where(live[:, None], tv, 0.0)
    p = torch.where(ok, torch.softmax(tv, 1), 0.0)
    clean = torch.where(live[:, None], leaf, 0.0)
    logq = torch.log_softmax(clean / T, 1).gather(1, i.long().clamp(0, V - 1))
    terms = torch.where(p > 0, p * (p.clamp(min=1e-300).log() - torch.where(p > 0, logq, 0.0)), 0.0)
    loss = T * T * terms.sum(1)
    (d,) = torch.autograd.grad((loss * g.double()).sum(), leaf)
    return loss.detach(), torch.where(live[:, None], d, 0.0)


def _run(s, t, i, g, T):
    from passion_amd import ops
    leaf = s.cuda().requires_grad_()
    loss = ops.topk_distill(leaf, t.cuda(), i.cuda(), T)
    (d,) = torch.autograd.grad(loss, leaf, g.cuda())
    with torch.no_grad():
        assert torch.equal(ops.topk_distill(leaf, t.cuda(), i.cuda(), T), loss)
    return loss, d


def _check(s, t, i, g, T):
    loss, d = _run(s, t, i, g, T)
    want, dw = _reference(s, t, i, g, T)
    off = (loss.double().cpu() - want).abs().max()
    assert float(off) <= 3.2e-4 * T * T + 2e-6 * float(want.abs().max()), (float(off), float(want.abs().max()))
    near(d, dw, 2e-5, "dlogits", room=(g.double() * T)[:, None].expand(dw.shape) * 1.0)
    assert d.dtype == s.dtype


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F, H])
@pytest.mark.parametrize("R,V,K", [(1, 1, 1), (5, 2, 2), (4097, 4, 2), (1000, 5, 3), (77, 8, 8), (33, 20, 7), (64, 104, 16), (50, 512, 64), (50, 511, 5), (9, 513, 4),
                                   (6, 1000, 1), (3, 4099, 33), (2, 32001, 64), (1100, 4100, 9), (1, 130001, 100)])
def test_sizes(R, V, K, dt):
    _check(*_make(R, V, K, dt), 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("tdt,idt", [(F, torch.int32), (H, torch.int64), (H, torch.int32)])
@pytest.mark.parametrize("V", [4, 100, 3001])
def test_teacher_types(V, tdt, idt):
    _check(*_make(40, V, 4, H, tdt=tdt, idt=idt), 4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [6, 700])
@pytest.mark.parametrize("T", [0.5, 1.0, 8.0])
def test_repeated_and_missing_entries(V, T):
    """the same class twice, entries out of range, rows without a teacher (whose logits may hold anything), teacher logits of -inf"""
    s, t, i, g = _make(64, V, 6, F, seed=4)
    i[0] = 3
    i[1, :3] = i[1, 3:].clone()
    i[2, 1:] = -1
    i[3, 2] = V
    i[4, 0] = -(2 ** 40)
    i[5, 4] = 2 ** 33 + 1
    i[6] = -1
    i[7] = -1
    s[7] = float("nan")
    t[8, 2:] = float("-inf")
    t[9] = float("-inf")
    t[10, 1] = torch.finfo(F).min
    i[11, 0] = -1
    t[11, 0] = float("nan")
    _check(s, t, i, g, T)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [7, 900])
def test_masked_classes(V):
    """student logits of -inf (classes that cannot occur) and of the type's lowest value: q = 0 there, and the gradient too"""
    s, t, i, g = _make(20, V, 2, F, seed=6)
    s[:, 0] = float("-inf")
    s[:, 1] = torch.finfo(F).min
    i = 2 + i % (V - 2)
    s[3, 2:] = 60 * s[3, 2:]
    loss, d = _run(s, t, i, g, 1.0)
    want, dw = _reference(s, t, i, g, 1.0)
    assert torch.allclose(loss.double().cpu(), want, rtol=2e-6, atol=1e-4)
    near(d, torch.nan_to_num(dw), 2e-5, "dlogits", room=g.double()[:, None].expand(dw.shape))
    assert float(d[:, :2].abs().max()) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F, H])
@pytest.mark.parametrize("T", [0.5, 1.0, 8.0])
@pytest.mark.parametrize("V", [3, 40, 500, 900, 4099, 40000])
def test_runs_of_masked_classes(V, T, dt):
    """whole runs of classes at their type's lowest value (a padded or restricted set of classes), as far as a row that holds nothing else (all classes alike) and a
    teacher's entries that do (all shares alike): log2(e) / T times that value is past the type's range below T = 1.44.  Same tolerances as ever: the differences of
    logits are exact or overflow to -inf, whose share is 0 on both sides"""
    s, t, i, g = _make(24, V, 2, dt, seed=11)
    s[:, V // 4:V // 2] = torch.finfo(dt).min
    s[5:9, : V - 1] = torch.finfo(dt).min
    s[9, 1:] = torch.finfo(dt).min
    s[10] = torch.finfo(dt).min
    i = V - 1 - i % max(1, V // 4)              # classes that every row but those few keeps
    i[5:9], i[9] = V - 1, 0
    t[11:13] = torch.finfo(F).min
    t[13, 0] = torch.finfo(F).min
    _check(s, t, i, g, T)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 3000])
def test_a_common_offset_of_a_row_costs_nothing(V):
    """softmax does not know it: logits of 1e5 and a little, exact in f32 as given"""
    s, t, i, g = _make(12, V, 3, F, seed=12)
    s[::2] += 1e5
    s[1::2] -= 1e5
    t += 3e4
    _check(s, t, i, g, 1.0)


@pytest.mark.gpu
def test_views_and_leading_shapes():
    """(B, D, H, W, C) voxels, transposed storage, a base that is not 16-byte aligned"""
    from passion_amd import ops
    s, t, i, g = _make(2 * 3 * 4 * 5, 9, 3, F, seed=8)
    want = _run(s, t, i, g, 2.0)
    a = s.cuda().view(2, 3, 4, 5, 9)
    turned = a.permute(4, 0, 1, 2, 3).contiguous().permute(1, 2, 3, 4, 0).detach().requires_grad_()
    loss = ops.topk_distill(turned, t.cuda().view(2, 3, 4, 5, 3), i.cuda().view(2, 3, 4, 5, 3), 2.0)
    assert loss.shape == (2, 3, 4, 5) and torch.equal(loss.view(-1), want[0])
    (d,) = torch.autograd.grad(loss, turned, g.cuda().view(2, 3, 4, 5))
    assert torch.equal(d.reshape(-1, 9), want[1])
    s, t, i, g = _make(5, 801, 3, H, seed=9)
    want = _run(s, t, i, g, 2.0)
    store = torch.empty(5 * 801 + 1, dtype=H, device="cuda")
    off = store[1:].view(5, 801)
    off.copy_(s)
    off = off.detach().requires_grad_()
    loss = ops.topk_distill(off, t.cuda(), i.cuda(), 2.0)
    assert torch.equal(loss, want[0]) and torch.equal(torch.autograd.grad(loss, off, g.cuda())[0], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("R,V,K", [(300, 4, 2), (40, 5001, 16)])
def test_captured_replayed_repeated_and_on_another_stream(R, V, K):
    from passion_amd import ops
    sets = [[v.cuda() for v in _make(R, V, K, H, seed=s)] for s in range(4)]
    statics = [t.clone() for t in sets[0]]

    def step(s, t, i, g):
        leaf = s.detach().requires_grad_()
        loss = ops.topk_distill(leaf, t, i, 2.0)
        return (loss, *torch.autograd.grad(loss, leaf, g))

    replayed(lambda: step(*statics), statics, sets, step)
    base = step(*sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*sets[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(base, other))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [12, 600])
def test_gradient_against_differences(V):
    """central differences of the f32 loss: step^2 third-derivative terms (1e-4) and 2^-24 * loss / step = 6e-4 at a loss of 100"""
    from passion_amd import ops
    s, t, i, g = (v.cuda() for v in _make(6, V, 4, F, seed=2))
    leaf = s.clone().requires_grad_()
    f = lambda x: (ops.topk_distill(x, t, i, 2.0).double() * g.double()).sum()
    (d,) = torch.autograd.grad(f(leaf), leaf)
    way = torch.randn(s.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    with torch.no_grad():
        quotient = float(f(s + 1e-2 * way) - f(s - 1e-2 * way)) / 2e-2
    assert abs(quotient - float((d * way).sum())) < 1e-2 * float(d.norm())


@pytest.mark.gpu
def test_the_whole_distribution_is_the_kl_of_the_framework():
    """K = V: the same loss as the framework's KL over whole class distributions up to its clamps (1e-8 in oracle terms) and its mean over classes"""
    from passion_amd import ops
    from passion_amd.utils import criterions
    g = torch.Generator().manual_seed(3)
    ls, lt = torch.randn(2, 4, 6, 6, 6, generator=g).cuda(), torch.randn(2, 4, 6, 6, 6, generator=g).cuda()
    want = criterions.temp_kl_loss_bs(ls, lt, temp=4.0)
    v, i = lt.permute(0, 2, 3, 4, 1).sort(-1, descending=True)
    got = ops.topk_distill(ls.permute(0, 2, 3, 4, 1), v, i, 4.0).mean((1, 2, 3)) / 4
    assert torch.allclose(got, want.view(-1), rtol=1e-4)


@pytest.mark.gpu
def test_no_rows():
    from passion_amd import ops
    s = torch.zeros(0, 10, device="cuda", requires_grad=True)
    loss = ops.topk_distill(s, torch.zeros(0, 3, device="cuda"), torch.zeros(0, 3, dtype=torch.long, device="cuda"))
    loss.sum().backward()
    assert loss.shape == (0,) and s.grad.shape == (0, 10)


def test_refusals():
    from passion_amd import _lib, ops
    s, t, i = torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.long)
    for bad in ((s, t[:2], i, 1.0), (s, t, i[:, :1], 1.0), (s, t, i.float(), 1.0), (s.half(), t, i, 1.0), (s, t.half(), i, 1.0), (s, t, i, 0.0), (s, t, i, float("nan")),
                (s, t, i, float("inf")), (s, torch.zeros(3, 0), torch.zeros(3, 0, dtype=torch.long), 1.0),
                (s, torch.zeros(3, 1025), torch.zeros(3, 1025, dtype=torch.long), 1.0), (s[0], t, i, 1.0)):
        with pytest.raises(ValueError):
            ops.topk_distill(*bad)
    with pytest.raises(_lib.PassionHipError):
        ops.topk_distill(s, t, i)


def test_temperatures_past_f32_are_refused():
    """the kernels hold T^2 and log2(e) / T in f32: temperatures whose square or reciprocal leaves its normal range gave NaN or 0"""
    from passion_amd import _lib, ops
    s, t, i = torch.zeros(3, 8), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.long)
    for T in (1e-300, 1e-40, 1e-20, 2e19, 1e300):
        with pytest.raises(ValueError):
            ops.topk_distill(s, t, i, T)
    lib = _lib.load()
    for T in (1e-40, 1e-20, 2e19, float("inf"), float("nan"), -1.0):
        assert lib.passion_topk_distill_fwd(256, 0, 256, 0, 256, 0, 2, 8, 2, T, 256, None, None) == -1003
        assert lib.passion_topk_distill_bwd(264, 0, 256, 0, 256, 0, 2, 1000, 2, T, 256, 256, 256, None) == -1003


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1e-18, 1e18])
@pytest.mark.parametrize("V", [9, 700])
def test_the_extreme_temperatures(V, T):
    """logits in proportion to T: the loss is T^2 times that of T = 1"""
    s, t, i, g = _make(6, V, 3, F, seed=3)
    _check(s * T, t * T, i, g, T)


def test_c_entry_refuses_on_the_host():
    from passion_amd import _lib
    lib = _lib.load()
    assert lib.passion_topk_distill_max_k() == 1024
    fwd = lambda R, V, K, T, dt=0: lib.passion_topk_distill_fwd(256, dt, 256, 0, 256, 0, R, V, K, T, 256, None, None)
    assert fwd(0, 8, 2, 1.0) == -1003 and fwd(2, 0, 2, 1.0) == -1003 and fwd(2, 8, 1025, 1.0) == -1003 and fwd(2, 8, 2, 0.0) == -1003 and fwd(2, 8, 2, 1.0, 2) == -1003
    assert lib.passion_topk_distill_bwd(264, 0, 256, 0, 256, 0, 2, 1000, 2, 1.0, 256, 256, 256, None) == -1005
