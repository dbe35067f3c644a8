"""Windows that reach over everything, written as a large number: no window, on the same kernels."""
import pytest
import torch

from flashck_b200 import _lib, ops

pytestmark = pytest.mark.gpu
FAR = [2 ** 30 - 1, 2 ** 30, 2 ** 31, 2 ** 40, 2 ** 63 - 1]


@pytest.fixture(params=["tcgen05", "general"])
def instance(request):
    _lib.set_instance_param(0, "use_sm100_bwd", int(request.param == "tcgen05"))
    yield request.param
    _lib.set_instance_param(0, "use_sm100_bwd", 1)


@pytest.mark.parametrize("far", FAR)
@pytest.mark.parametrize("mask_type,left,right", [(2, "far", 0), (2, 20, "far"), (1, "far", 7), (3, "far", "far"), (2, "far", -1)])
@pytest.mark.parametrize("sq,sk", [(200, 330), (300, 40)])
def test_windows_without_an_end(far, mask_type, left, right, sq, sk, instance, device_ok):
    q, k, v, dout = (torch.randn(2, n, 2, 64, device="cuda").bfloat16() for n in (sq, sk, sk, sq))
    window, plain = (tuple(end if x == "far" else x for x in (left, right)) for end in (far, -1))
    o, lse = ops.fmha_fwd(q, k, v, mask_type=mask_type, window_size=plain, return_lse=True)
    want = ops.fmha_bwd(dout, q, k, v, o, lse, mask_type=mask_type, window_size=plain)
    got = ops.fmha_bwd(dout, q, k, v, o, lse, mask_type=mask_type, window_size=window)
    assert _lib.get_instance_param(0, "last_bwd_instance") == int(instance == "tcgen05")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
