"""NaN and infinities in the backward pass: they stay out of what they are hidden from, and show in what they are part of."""
import pytest
import torch

from attention_reference import assert_within, forward, gradients
from flashck_b200 import _lib, ops

pytestmark = pytest.mark.gpu
NONE = (0, -1, -1)


@pytest.fixture(params=["tcgen05", "general"])
def instance(request):
    _lib.set_instance_param(0, "use_sm100_bwd", int(request.param == "tcgen05"))
    yield request.param
    _lib.set_instance_param(0, "use_sm100_bwd", 1)


def _problem(b, sq, sk, h, d, mask, dtype=torch.bfloat16, **more):
    q, dout = (torch.randn(b, sq, h, d, device="cuda").to(dtype) for _ in range(2))
    k, v = (torch.randn(b, sk, h, d, device="cuda").to(dtype) for _ in range(2))
    o, lse = forward(q, k, v, d ** -0.5, mask, **more)
    return dout, q, k, v, o.to(dtype), lse.float()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask", [(1, -1, 0), (3, 40, 3), (1, -1, 5)])  # top-left: the last keys are seen by no query
@pytest.mark.parametrize("sq,sk", [(100, 128), (100, 300), (130, 200), (1, 60)])
@pytest.mark.parametrize("add", ["none", "cap", "alibi", "bias"])
def test_keys_that_no_query_sees(d, mask, sq, sk, add, instance, device_ok):
    """Their K and V may hold anything: their gradients are zero, and the other keys' are what they are without them."""
    b, h = 2, 2
    more = dict(cap=dict(cap=4.0), alibi=dict(slopes=torch.rand(1, h, device="cuda") * 0.2),
                bias=dict(bias=torch.randn(1, h, sq, sk, device="cuda").bfloat16())).get(add, {})
    args = _problem(b, sq, sk, h, d, mask, **more)
    unseen = sq + mask[2]
    clean = [t.clone() for t in args]
    for t in clean[2:4]:
        t[:, unseen:] = 0
    want, bound = gradients(*clean, d ** -0.5, mask, **more)
    for t in args[2:4]:
        t[:, unseen:] = float("nan")
        t[:, unseen::3] = float("inf")
    _, dk, dv = ops.fmha_bwd(*args, mask_type=mask[0], window_size=mask[1:], bias=more.get("bias"), alibi_slopes=more.get("slopes"),
                             logits_soft_cap=more.get("cap", 0.0))
    assert not dk[:, unseen:].any() and not dv[:, unseen:].any()
    for n, x, w, e in (("dk", dk, want[1], bound[1]), ("dv", dv, want[2], bound[2])):
        assert_within(n, x, w, e)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("where", ["q", "lse"])
def test_a_nan_in_any_query_row_shows(d, where, instance, device_ok):
    """Sequence i has it in row i.  Its P are NaN, so all of dV and dK are, and the row's dQ; other rows' dQ are not."""
    n = 64
    dout, q, k, v, o, lse = _problem(n, n, 70, 1, d, NONE)
    rows = torch.arange(n, device="cuda")
    (q[:, :, 0, 0] if where == "q" else lse[:, 0])[rows, rows] = float("nan")
    dq, dk, dv = ops.fmha_bwd(dout, q, k, v, o, lse)
    assert torch.isnan(dv).all() and torch.isnan(dk).all()
    hit = torch.isnan(dq).all(-1)[..., 0]
    assert torch.equal(hit, torch.eye(n, dtype=torch.bool, device="cuda")) and torch.isfinite(dq[~hit]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_a_nan_in_any_key_shows(d, instance, device_ok):
    n = 64
    dout, q, k, v, o, lse = _problem(n, 70, n, 1, d, NONE)
    rows = torch.arange(n, device="cuda")
    k[rows, rows, 0, 0] = float("nan")
    dq, dk, dv = ops.fmha_bwd(dout, q, k, v, o, lse)
    assert torch.isnan(dq).all()
    hit = torch.isnan(dv).all(-1)[..., 0]
    assert torch.equal(hit, torch.eye(n, dtype=torch.bool, device="cuda")) and torch.isfinite(dv[~hit]).all()
    assert torch.equal(torch.isnan(dk).all(-1)[..., 0], hit) and torch.isfinite(dk[~hit]).all()
