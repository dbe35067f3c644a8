"""The 64-bit formulas that the kernels are held to, against differences of the loss and against autograd through the forward."""
import pytest
import torch

from attention_reference import forward, gradients

MASKS = [(0, -1, -1), (2, -1, 0), (2, 7, 2), (1, 5, 30)]
ADDITIONS = ["none", "cap", "alibi", "plane", "plane per head", "plane per sequence", "plane and cap", "alibi and cap"]
B, SQ, SK, HQ, HKV, D, SCALE = 2, 11, 17, 4, 2, 8, 0.45


def _problem(mask, add, seed):
    g = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, dout = normal(B, SQ, HQ, D), normal(B, SK, HKV, D), normal(B, SK, HKV, D), normal(B, SQ, HQ, D)
    shape = {"plane": (1, 1), "plane and cap": (1, 1), "plane per head": (1, HQ), "plane per sequence": (B, HQ)}.get(add)
    bias = normal(*shape, SQ, SK) if shape else None
    slopes = torch.rand(1, HQ, generator=g, dtype=torch.float64) if "alibi" in add else None
    return dout, normal(B, HQ, SQ), dict(q=q, k=k, v=v, bias=bias), dict(scale=SCALE, mask=mask, slopes=slopes, cap=1.5 if "cap" in add else 0.0), normal


def _loss(x, dout, dlse, kw):
    o, lse = forward(x["q"], x["k"], x["v"], bias=x["bias"], **kw)
    return (o * dout).sum() + (torch.where(torch.isneginf(lse), 0.0, lse) * dlse).sum()


def _formula(x, dout, dlse, kw):
    o, lse = forward(x["q"], x["k"], x["v"], bias=x["bias"], **kw)
    (dq, dk, dv, dt), _ = gradients(dout, x["q"], x["k"], x["v"], o, lse, bias=x["bias"], dlse=dlse, **kw)
    grads = dict(q=dq, k=dk, v=dv)
    if x["bias"] is not None:
        axes = [a for a in (0, 1) if x["bias"].shape[a] == 1]
        grads["bias"] = dt.sum(axes, keepdim=True) if axes else dt
    return grads


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("add", ADDITIONS)
@pytest.mark.parametrize("seed", [0, 1])
def test_differences_of_the_loss(mask, add, seed):
    """Each input moved by itself.  With a step of 1e-5 the quotient is off by h^2 / 6 of the third derivative (some 1e-10) and by the
    loss's rounding over h (some 1e-10 too); 1e-7 of |gradient| |direction| leaves room, and a gradient that is zero, has the wrong sign or
    misses a factor does not fit into it."""
    dout, dlse, x, kw, normal = _problem(mask, add, seed)
    grads, h = _formula(x, dout, dlse, kw), 1e-5
    for name, g in grads.items():
        along = normal(*g.shape)
        moved = [_loss({**x, name: x[name] + s * h * along}, dout, dlse, kw) for s in (1, -1)]
        slope, allowed = (moved[0] - moved[1]) / (2 * h), 1e-7 * g.norm() * along.norm()
        assert abs((g * along).sum() - slope) <= allowed, name
        # A zero or a wrong sign is off by the slope or more.  (The cosine between a gradient of n parts, 187 to 1496 here, and a random direction is
        # a normal number over sqrt(n): below 10 x 1e-7 for fewer than one direction in 30 000.)
        assert abs(slope) > 10 * allowed, f"{name}: this direction shows nothing"


@pytest.mark.parametrize("mask", [m for m in MASKS if m[0] != 1])  # (a row without keys has no derivative there)
@pytest.mark.parametrize("add", ADDITIONS)
def test_autograd_through_the_forward(mask, add):
    dout, dlse, x, kw, _ = _problem(mask, add, 2)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items() if t is not None}
    grads = _formula(x, dout, dlse, kw)
    want = torch.autograd.grad(_loss({**x, **leaves}, dout, dlse, kw), list(leaves.values()))
    for name, w in zip(leaves, want):
        # (sums of some hundred products in 64 bits)
        assert (grads[name] - w).abs().max() <= 1e-12 * w.abs().max(), name
