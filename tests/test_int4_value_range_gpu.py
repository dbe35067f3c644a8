"""Values far from 1, in all groups together: their scales pass what a half or the weights' reference alone could hold."""
import pytest
import torch

import int4_reference as ref
from flashck_b200 import _lib, ops
from test_int4_group_scales_gpu import _bound

pytestmark = pytest.mark.gpu


def _hold(tokens, n, hq, hkv, d, group, factor, splits=0):
    """factor [n]: what the tokens' scales and least values are multiplied by."""
    g, t, four = torch.Generator("cuda").manual_seed(3), torch.bfloat16, []
    for i in range(2):
        c, sc, lo = ref.quantise(torch.randn(n, hkv, d, generator=g, device="cuda").to(t), group)
        params = torch.stack([sc, lo], -1)
        four += [ref.pack(c), (params * factor[:, None, None, None] if i else params).to(t)]
    q = torch.randn(tokens, hq, d, generator=g, device="cuda").to(t)
    o, lse = ops.fmha_fwd_splitkv_int4(q[None], *(x[None].contiguous() for x in four), seqlen_k=torch.tensor([n], dtype=torch.int32, device="cuda"),
                                       num_splits=splits, return_lse=True)
    want, want_lse, bound, lse_bound = _bound(q, *four, d ** -0.5, (0, -1, -1))
    ref.assert_within("o", o[0], want, bound + 2.0 ** -133)  # (half of bf16's least step)
    assert ((lse[0] - want_lse).abs() <= lse_bound).all() and _lib.device_status() == 0


SHAPES = [(1, 4, 1, 128, 128), (1, 8, 1, 64, 64), (3, 8, 2, 128, 128), (5, 4, 1, 64, 64), (1, 4, 1, 128, 32), (2, 4, 1, 64, 32), (5, 8, 2, 128, 64)]


@pytest.mark.parametrize("tokens,hq,hkv,d,group", SHAPES)
@pytest.mark.parametrize("power", [-116, -100, -80, -60, 60, 100, 108, 114, 122])
def test_values_of_any_magnitude(tokens, hq, hkv, d, group, power):
    _hold(tokens, 500, hq, hkv, d, group, torch.full((500,), 2.0 ** power, dtype=torch.float64, device="cuda"))


@pytest.mark.parametrize("tokens,hq,hkv,d,group", SHAPES)
@pytest.mark.parametrize("low,high", [(-116, -60), (-90, 10), (-20, 80), (60, 122)])
@pytest.mark.parametrize("splits", [0, 1])
def test_values_that_grow_and_shrink_along_the_keys(tokens, hq, hkv, d, group, low, high, splits):
    f = 2.0 ** torch.linspace(low, high, 700, dtype=torch.float64, device="cuda")
    _hold(tokens, 700, hq, hkv, d, group, f, splits)
    _hold(tokens, 700, hq, hkv, d, group, f.flip(0), splits)
