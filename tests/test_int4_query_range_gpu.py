"""Queries far from 1 over keys as far the other way: scores of the usual size."""
import pytest
import torch

import int4_reference as ref
from flashck_b200 import _lib, ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-110, -60, 60, 101, 104, 110, 114, 118])
@pytest.mark.parametrize("d,group,hq", [(128, 128, 4), (128, 32, 8), (64, 64, 8), (64, 32, 16)])
def test_queries_of_any_magnitude(power, d, group, hq):
    g = torch.Generator("cuda").manual_seed(1)
    n, t = 200, torch.bfloat16
    four = []
    for i in range(2):
        c, sc, lo = ref.quantise(torch.randn(n, 1, d, generator=g, device="cuda").to(t), group)
        four += [ref.pack(c), (torch.stack([sc, lo], -1) * (1.0 if i else 2.0 ** -power)).to(t)]
    q = (torch.randn(1, hq, d, generator=g, device="cuda") * 2.0 ** power).to(t)
    assert torch.isfinite(q).all() and (four[1].abs().amax() > 0)
    o, lse = ops.fmha_fwd_splitkv_int4(q[None], *(x[None].contiguous() for x in four), seqlen_k=torch.tensor([n], dtype=torch.int32, device="cuda"),
                                       return_lse=True)
    want, want_lse, bound, lse_bound = ref.attend(q, *four, d ** -0.5, (0, -1, -1))
    ref.assert_within("o", o[0], want, bound)
    assert ((lse[0] - want_lse).abs() <= lse_bound).all()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("scale", [2.0 ** -40, 30.0, 2.0 ** 20])
def test_scales_of_any_size(scale):
    """The same with the caller's scale: what the queries lose goes to it."""
    g = torch.Generator("cuda").manual_seed(2)
    n, d, t = 90, 64, torch.bfloat16
    four = []
    for _ in range(2):
        c, sc, lo = ref.quantise(torch.randn(n, 1, d, generator=g, device="cuda").to(t), 64)
        four += [ref.pack(c), torch.stack([sc, lo], -1).to(t)]
    q = (torch.randn(1, 8, d, generator=g, device="cuda") * d ** -0.5 / scale).to(t)
    o = ops.fmha_fwd_splitkv_int4(q[None], *(x[None].contiguous() for x in four), seqlen_k=torch.tensor([n], dtype=torch.int32, device="cuda"), scale=scale)
    want, _, bound, _ = ref.attend(q, *four, scale, (0, -1, -1))
    ref.assert_within("o", o[0], want, bound)
