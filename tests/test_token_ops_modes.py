"""The token operators under the modes of torch that follow the calls of its dispatcher: forward-mode derivatives, traces, exported graphs, torch.func.  Their kernels are
launched outside it, so such a call would lose its tangent or leave a graph without the kernel; it is refused.  Shown on the CPU where the operators launch nothing (no
keys, no rows), and on the GPU through the public entry points."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx


def _calls(device, rows):
    """name -> (call of one tensor, the tensor)"""
    from passion_amd import _lib, ops
    host = _lib.token_ops()
    q, k = torch.ones(1, 3, 2, 8, device=device), torch.ones(1, rows, 2, 8, device=device)
    x, s = torch.ones(rows, 16, device=device), torch.ones(rows, 5, device=device)
    tv, ti = torch.ones(rows, 2, device=device), torch.zeros(rows, 2, dtype=torch.long, device=device)
    if device == "cpu":
        return {"rel_attention": (lambda t: host.rel_attention(t, k, k, None, None, None, [1, 1, 1, 0, 0], 1.0), q),
                "residual_norm": (lambda t: host.residual_norm(t, x, None, None, None, None, None, None, [0, 0, 0, 1, rows], [0.0, 0.0])[0], x.clone()),
                "topk_distill": (lambda t: host.topk_distill(t, tv, ti, 1.0), s)}
    return {"rel_attention": (lambda t: ops.rel_attention(t, k, k), q), "residual_norm": (lambda t: ops.residual_norm(t, x), x.clone()),
            "topk_distill": (lambda t: ops.topk_distill(t, tv, ti), s)}


NAMES = pytest.mark.parametrize("name", ["rel_attention", "residual_norm", "topk_distill"])


def _modes(f, t):
    def dual():
        with fwd.dual_level():
            f(fwd.make_dual(t, torch.ones_like(t)))

    yield "forward-mode", dual
    yield "jvp", lambda: torch.func.jvp(f, (t,), (torch.ones_like(t),))
    yield "vmap", lambda: torch.vmap(f)(t[None])
    yield "func.grad", lambda: torch.func.grad(lambda a: f(a).sum())(t)
    yield "jit.trace", lambda: torch.jit.trace(f, (t,), check_trace=False)
    for how in ("real", "fake", "symbolic"):
        yield "make_fx " + how, lambda: make_fx(f, tracing_mode=how)(t)


def _all_refused(f, t):
    f(t)
    for need in (False, True):
        leaf = t.clone().requires_grad_(need)
        for mode, call in _modes(f, leaf):
            with pytest.raises(Exception):
                call()
                raise_if_reached(mode)
    f(t)


def raise_if_reached(mode):
    pytest.fail(mode + " went through")


@NAMES
def test_refused_on_the_host(name):
    _all_refused(*_calls("cpu", 0)[name])


@pytest.mark.gpu
@NAMES
def test_refused_through_the_public_entry_points(name):
    _all_refused(*_calls("cuda", 4)[name])


@pytest.mark.gpu
def test_checkpointing_inference_mode_and_hooks_are_served():
    """what stays inside the dispatcher or above it goes on as before"""
    from torch.utils.checkpoint import checkpoint
    for f, t in _calls("cuda", 4).values():
        t = torch.randn(t.shape, generator=torch.Generator().manual_seed(0)).cuda()
        want = f(t)
        with torch.inference_mode():
            assert torch.equal(f(t), want)
        a, b = t.clone().requires_grad_(), t.clone().requires_grad_()
        f(a).sum().backward()
        out = checkpoint(f, b, use_reentrant=False)
        seen = []
        out.register_hook(seen.append)
        out.sum().backward()
        assert torch.equal(out, want) and torch.equal(a.grad, b.grad) and len(seen) == 1
