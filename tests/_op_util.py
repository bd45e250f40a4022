"""helpers of the token-operator tests: tolerances by type, capture and replay"""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # one rounding: torch.finfo(t).eps / 2, relative to the value


def near(got, want, rel, what, room=None):
    """|got - want| <= one rounding of got's type + rel * (room, or the largest wanted value), element by element"""
    got = got.detach()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    w = want.double().to(got.device)
    scale = w.abs().amax() if room is None else room.double().to(got.device)
    off = (got.double() - w).abs() - HALF[got.dtype] * w.abs() - rel * scale
    worst = float(off.max()) if off.numel() else -1.0
    assert torch.isfinite(got).all(), what
    assert worst <= 0, f"{what}: over its tolerance by {worst:.3e} (largest value {float(w.abs().max()):.3e})"


def replayed(fn, statics, fresh, eager):
    """capture fn() -> tuple of tensors over the static inputs, then replay on `fresh` input sets with the program's own eager work between the
    replays; every replay has to equal the eager result bit for bit"""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = fn()
    for new in fresh:
        want = [t.clone() for t in eager(*new)]
        for s, n in zip(statics, new):
            s.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
        torch.zeros(1 << 20, device="cuda").add_(1)
        torch.cuda.synchronize()
