"""Calls without a token whose positions have several axes: an image or video batch that happens to be empty."""
import pytest
import torch

from flashck_b200 import ops
from flashck_b200.ops import fmha
from flashck_b200.utils.enums import RopeEnum

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[False, True], ids=["binding", "python"])
def python(request, monkeypatch):
    if request.param:
        monkeypatch.setattr(fmha, "_NATIVE", False)


def _tensors(*lead, hq=4, hkv=2, d=64):
    return tuple(torch.zeros(*lead, h, d, device="cuda", dtype=torch.bfloat16) for h in (hq, hkv, hkv))


def _positions(*shape, dtype=torch.int32):
    return torch.zeros(shape, device="cuda", dtype=dtype)


T = dict(dtype=torch.bfloat16, device="cuda")


@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 7)])
@pytest.mark.parametrize("sections", [(8, 12, 12), (16, 16), (32,), None])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_rotary(python, lead, sections, dtype):
    q, k, _ = _tensors(*lead)
    t = torch.ones(9, 32, **T)
    axes = len(sections or (0,))
    pos = _positions(*((axes,) if axes > 1 else ()), *lead, dtype=dtype)
    for call in (ops.apply_rotary, ops.apply_rotary_autograd):
        y = call(q.requires_grad_(), k, pos, t, t, sections=sections)
        assert y[0].shape == q.shape and y[1].shape == k.shape
    y[0].sum().backward()
    assert q.grad.shape == q.shape


@pytest.mark.parametrize("packed", [False, True])
def test_append(python, packed):
    q, k, v = _tensors(*((0,) if packed else (2, 0)))
    parts = [x for _ in range(2) for x in ops.int4_cache(2, 16, 2, 64, group=32)]
    before = [x.clone() for x in parts]
    t, kw = torch.ones(9, 32, **T), {}
    if packed:
        kw = dict(zip(("cu_seqlens_q", "cu_seqlens_knew"), [torch.zeros(3, dtype=torch.int64, device="cuda")] * 2))
    y = ops.fmha_fwd_append_kv_int4(q, *parts, k, v, _positions(2), t, t, rope=RopeEnum.HALF_ROTATED, positions=_positions(3, *k.shape[:-2]),
                                    sections=(8, 12, 12), return_kv=True, **kw)
    assert [x.shape for x in y] == [x.shape for x in (q, k, v)] and all(torch.equal(a, b) for a, b in zip(before, parts))


@pytest.mark.parametrize("shape,sections", [((2, 0), (8, 12, 12)), ((0,), (16, 16)), ((0, 3), (8, 12, 12)), ((3, 1), (8, 12, 12))])
def test_positions_of_another_number_of_axes_are_refused(python, shape, sections):
    q, k, _ = _tensors(0)
    t = torch.ones(9, 32, **T)
    with pytest.raises(ValueError, match="positions"):
        ops.apply_rotary(q, k, _positions(*shape), t, t, sections=sections)
