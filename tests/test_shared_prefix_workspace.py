"""The workspace of decode over a shared prefix: its size is the call's own, whatever the instance parameters are when it is asked for."""
import pytest
import torch

from attention_reference import assert_within, forward, half_step
from flashck_b200 import _lib

SETTINGS = [("use_sm100_splitkv", 0), ("split_item_cost", 1), ("split_item_cost", 60)]


def _size(prefix, page, batch, sq, hq, hkv, d, group=0):
    return _lib.lib().FlashckSharedPrefixWorkspace(prefix, page, 16, batch, sq, sq if group else 0, hq, hkv, d, group, 4)


@pytest.fixture(params=SETTINGS, ids=[f"{k}={v}" for k, v in SETTINGS])
def setting(request):
    key, value = request.param
    before = _lib.get_instance_param(2, key)
    yield lambda: _lib.set_instance_param(2, key, value)
    _lib.set_instance_param(2, key, before)


@pytest.mark.parametrize("sizes", [
    (131072, 64, 32, 1, 64, 8, 128), (131072, 64, 257, 1, 64, 8, 128), (5000, 16, 40, 1, 8, 2, 64), (300, 16, 700, 1, 4, 1, 64),
    (8192, 16, 64, 1, 32, 8, 128), (2000, 0, 48, 4, 8, 2, 64), (100, 16, 2, 1, 4, 2, 64), (9000, 0, 3, 7, 12, 4, 128), (700, 48, 40, 1, 8, 2, 64),
])
def test_size_does_not_follow_the_instance_parameters(sizes, setting):
    asked = _size(*sizes)
    setting()
    assert _size(*sizes) == asked


@pytest.mark.parametrize("page", [16, 48, 80, 128])
@pytest.mark.parametrize("prefix", [1, 33, 500, 9000])
@pytest.mark.parametrize("batch,hq,hkv", [(32, 64, 8), (5, 8, 1), (400, 4, 1), (3, 3, 1)])
def test_a_page_size_without_a_table_needs_no_more(page, prefix, batch, hq, hkv):
    """A call without a table is not paged, whatever page size came with it: it fits what was asked for with that page size."""
    assert _size(prefix, page, batch, 1, hq, hkv, 64) >= _size(prefix, 0, batch, 1, hq, hkv, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("b,tokens", [(5, 1), (40, 1), (3, 4)])
def test_a_workspace_sized_before_a_setting_changed(b, tokens, setting, device_ok):
    """Behind the bytes that were asked for nothing is written, and the result is the formula's."""
    hq, hkv, d, prefix, cap, dtype = 8, 1, 64, 4000, 24, torch.bfloat16
    q = torch.randn(b, tokens, hq, d, device="cuda", dtype=dtype)
    kp, vp = (torch.randn(prefix, hkv, d, device="cuda", dtype=dtype) for _ in range(2))
    k, v = (torch.randn(b, cap, hkv, d, device="cuda", dtype=dtype) for _ in range(2))
    sl = torch.full((b,), cap, dtype=torch.int32, device="cuda")
    lib = _lib.lib()
    n = lib.FlashckSharedPrefixWorkspace(prefix, 0, 0, b, tokens, 0, hq, hkv, d, 0, 4)
    setting()
    room = torch.full((n + (64 << 20),), 0x5A, dtype=torch.uint8, device="cuda")  # (more than any setting asked for at these sizes)
    o, lse = torch.empty_like(q), torch.empty(b, hq, tokens, device="cuda")
    rc = lib.FmhaFwdSharedPrefix(*(t.data_ptr() for t in (q, kp, vp, k, v, o, lse, room)), 0, 0, sl.data_ptr(), 0, prefix, 0, prefix, 0, b, 0, cap,
                                 b, tokens, 0, hq, hkv, d, d, 0.0, 0, torch.cuda.current_stream().cuda_stream, 4)
    assert rc == 0, _lib.last_error()
    assert (room[n:] == 0x5A).all()
    whole = [torch.cat([p.expand(b, -1, -1, -1), x], dim=1) for p, x in ((kp, k), (vp, v))]
    want, want_lse = forward(q, *whole, d ** -0.5, (0, -1, -1))
    spread, _ = forward(q, whole[0], whole[1].abs(), d ** -0.5, (0, -1, -1))
    u = half_step(dtype)
    # P rounded where it meets V, fp32 sums of d terms in S, the exponential to 2^-18, O rounded once
    e = d * 2.0 ** -24 * q.double().abs().amax() * whole[0].double().abs().sum(-1).amax() * d ** -0.5 + 2.0 ** -18
    assert_within("o", o, want, (u + e) * spread + u * want.abs())
    assert ((lse - want_lse).abs() <= e + 2.0 ** -20 * (1 + want_lse.abs())).all()
