"""The token operators together, as a training step uses them: norm -> attention with a relative position bias over two modalities' grids, one sample with a
modality missing -> gated residual and the next norm -> MLP -> residual -> class head -> distillation from a teacher's top logits; loss and every gradient against the same
step in 64 bits on the CPU.

Tolerance: f32 throughout.  Four operators and four library products (f32 accumulation over at most 64 terms) in a row, each off by below 1e-5 of its largest value
(their own tests), conditioning of order ten through two norms: 1e-3 of a gradient's largest value leaves a factor of ten."""
import math

import pytest
import torch

from _op_util import near

GRID, MODS, B, C, HEADS, CLASSES, K = (3, 4, 5), 2, 2, 64, 4, 23, 5


def _params(seed=0):
    g = torch.Generator().manual_seed(seed)
    w = lambda *s: torch.randn(*s, generator=g) / math.sqrt(s[-1])
    N = math.prod(GRID) * MODS
    nd = math.prod(2 * n - 1 for n in GRID)
    p = dict(qkv=w(3 * C, C), proj=w(C, C), up=w(2 * C, C), down=w(C, 2 * C), head=w(CLASSES, C), table=0.5 * torch.randn(nd, HEADS, generator=g), scale=0.5 + 0.1 * torch.randn(C, generator=g),
             gate=torch.randn(B, 1, C, generator=g))
    for i in range(4):
        p[f"w{i}"], p[f"b{i}"] = 1 + 0.2 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)
    x = torch.randn(B, N, C, generator=g)
    teacher = 3 * torch.randn(B, N, CLASSES, generator=g)
    mask = torch.ones(B, N, dtype=torch.bool)
    mask[1, :math.prod(GRID)] = False
    return p, x, teacher, mask


def _step(p, x, teacher, mask, ops):
    """ops: the framework's, or None for the definition in the tensors' own type"""
    F = torch.nn.functional
    N = x.shape[1]
    if ops is not None:
        norm = lambda i: _ln(p, i)
        step = lambda r, h, post, pre, gate=None, scale=None: ops.residual_norm(r, h, post, pre, gate, scale)
    else:
        def norm(i):
            return lambda t: F.layer_norm(t, (C,), p[f"w{i}"], p[f"b{i}"])

        def step(r, h, post, pre, gate=None, scale=None):
            h = h if post is None else post(h)
            h = h if gate is None else h * gate
            r = r + (h if scale is None else h * scale)
            return r, pre(r)
    r, y = step(x, torch.zeros_like(x), None, norm(0))
    q, k, v = (y @ p["qkv"].t()).view(B, N, 3, HEADS, C // HEADS).unbind(2)
    if ops is not None:
        a = ops.rel_attention(q, k, v, p["table"], GRID, key_mask=mask)
    else:
        cell = torch.stack(torch.meshgrid(*[torch.arange(n) for n in GRID], indexing="ij"), -1).view(-1, 3).repeat(MODS, 1)
        d = cell[:, None] - cell[None] + torch.tensor(GRID) - 1
        off = (d[..., 0] * (2 * GRID[1] - 1) + d[..., 1]) * (2 * GRID[2] - 1) + d[..., 2]
        s = torch.einsum("bihd,bjhd->bhij", q, k) * (C // HEADS) ** -0.5 + p["table"][off].permute(2, 0, 1)
        a = torch.einsum("bhij,bjhd->bihd", s.masked_fill(~mask[:, None, None], -math.inf).softmax(-1), v)
    r, y = step(r, a.reshape(B, N, C) @ p["proj"].t(), norm(1), norm(2), p["gate"], p["scale"])
    _, y = step(r, F.gelu(y @ p["up"].t()) @ p["down"].t(), None, norm(3))
    logits = y @ p["head"].t()
    top, at = teacher.topk(K, -1)
    at = at.masked_fill(~mask[..., None], -1)                     # missing tokens have no teacher
    if ops is not None:
        rows = ops.topk_distill(logits, top, at, 2.0)
    else:
        t = torch.softmax(top / 2, -1)
        rows = 4 * (t * (t.log() - torch.log_softmax(logits / 2, -1).gather(-1, at.clamp(min=0)))).sum(-1) * mask
    return rows.sum() / mask.sum()


@pytest.mark.gpu
def test_a_training_step_of_the_operators_together():
    from passion_amd import ops
    p, x, teacher, mask = _params()
    exact = {n: t.double().requires_grad_() for n, t in p.items()}
    xe = x.double().requires_grad_()
    want = _step(exact, xe, teacher.double(), mask, None)
    gw = dict(zip([*exact, "x"], torch.autograd.grad(want, [*exact.values(), xe])))
    on = {n: torch.nn.Parameter(t.cuda()) for n, t in p.items()}
    xg = x.cuda().requires_grad_()
    loss = _step(on, xg, teacher.cuda(), mask.cuda(), ops)
    got = dict(zip([*on, "x"], torch.autograd.grad(loss, [*on.values(), xg])))
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-4 * abs(float(want.detach()))
    for n in gw:
        near(got[n], gw[n], 1e-3, "d" + n)


@pytest.mark.gpu
def test_the_step_under_bf16_and_an_optimizer_repeats():
    """bf16 tokens with an f32 residual stream: two runs of three optimizer steps give the same parameters bit for bit"""
    from passion_amd import ops
    _, x, teacher, mask = _params()
    ends = []
    for _ in range(2):
        p, *_r = _params()
        on = {n: torch.nn.Parameter(t.cuda()) for n, t in p.items()}
        opt = torch.optim.SGD(on.values(), lr=1e-2)
        for _ in range(3):
            cast = {n: t.bfloat16() if n in ("qkv", "proj", "up", "down", "head", "table", "gate") else t for n, t in on.items()}
            r, y = ops.residual_norm(x.cuda(), torch.zeros_like(x).cuda().bfloat16(), None, _ln(on, 0))
            q, k, v = (y @ cast["qkv"].t()).view(B, -1, 3, HEADS, C // HEADS).unbind(2)
            a = ops.rel_attention(q, k, v, cast["table"], GRID, key_mask=mask.cuda())
            r, y = ops.residual_norm(r, a.reshape(B, -1, C) @ cast["proj"].t(), _ln(on, 1), _ln(on, 2), cast["gate"], on["scale"])
            top, at = teacher.cuda().topk(K, -1)
            loss = ops.topk_distill(y @ cast["head"].t(), top, at.int(), 2.0).mean()
            opt.zero_grad()
            loss.backward()
            opt.step()
        ends.append([t.detach().clone() for t in on.values()])
    assert all(torch.equal(a, b) for a, b in zip(*ends)) and all(torch.isfinite(t).all() for t in ends[0])


def _ln(p, i):
    m = torch.nn.LayerNorm(C)
    del m.weight, m.bias
    m.weight, m.bias = p[f"w{i}"], p[f"b{i}"]
    return m


@pytest.mark.gpu
def test_topk_distill_loss_bs_on_volumes():
    """NCDHW volumes: K = C is the framework's KL up to its clamps; voxels without a teacher leave it"""
    from passion_amd.utils import criterions
    g = torch.Generator().manual_seed(1)
    ls, lt = torch.randn(2, 4, 4, 6, 8, generator=g).cuda().requires_grad_(), torch.randn(2, 4, 4, 6, 8, generator=g).cuda()
    v, i = lt.topk(4, 1)
    a, b = criterions.topk_distill_loss_bs(ls, v, i, 4.0), criterions.temp_kl_loss_bs(ls, lt, temp=4.0)
    assert a.shape == b.shape == (2, 1) and torch.allclose(a, b, rtol=1e-4)
    ga, gb = (torch.autograd.grad(t.sum(), ls)[0] for t in (a, b))
    assert float((ga - gb).abs().max()) < 1e-4 * float(gb.abs().max())
    i = i.clone()
    i[:, :, 0] = -1
    (ga,) = torch.autograd.grad(criterions.topk_distill_loss_bs(ls, v[:, :2], i[:, :2], 4.0).sum(), ls)
    assert float(ga[:, :, 0].abs().max()) == 0 and float(ga[:, :, 1:].abs().max()) > 0
