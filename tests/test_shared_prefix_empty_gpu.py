"""Own caches that hold nothing yet: contiguous ones of capacity 0, as a block table without columns."""
import pytest
import torch

from attention_reference import assert_within, forward, half_step
from flashck_b200 import ops
from flashck_b200.ops import fmha

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("prefix", [0, 40, 700])
@pytest.mark.parametrize("tokens,packed", [(1, False), (4, False), (2, True)])
@pytest.mark.parametrize("causal", [True, False])
def test_contiguous_caches_of_capacity_0(monkeypatch, native, d, prefix, tokens, packed, causal, device_ok):
    if not native:
        monkeypatch.setattr(fmha, "_NATIVE", False)
    b, hq, hkv, dtype = 3, 8, 2, torch.bfloat16
    q = torch.randn(b, tokens, hq, d, device="cuda", dtype=dtype)
    kp, vp = (torch.randn(prefix, hkv, d, device="cuda", dtype=dtype) for _ in range(2))
    empty = torch.empty(b, 0, hkv, d, device="cuda", dtype=dtype)
    kw = dict(seqlen_k=torch.zeros(b, dtype=torch.int32, device="cuda"), causal=causal, return_lse=True)
    if packed:
        kw.update(cu_seqlens_q=torch.arange(b + 1, device="cuda") * tokens, max_seqlen_q=tokens)
    o, lse = ops.fmha_fwd_shared_prefix(q.flatten(0, 1) if packed else q, kp, vp, empty, empty, **kw)
    if packed:
        o, lse = o.view_as(q), lse.view(hq, b, tokens).transpose(0, 1)
    if not prefix:
        assert not o.any() and torch.isneginf(lse).all()
        return
    k, v = (t.expand(b, -1, -1, -1).contiguous() for t in (kp, vp))
    want, want_lse = forward(q, k, v, d ** -0.5, (0, -1, -1))
    spread, _ = forward(q, k, v.abs(), d ** -0.5, (0, -1, -1))
    u = half_step(dtype)
    # P rounded where it meets V, fp32 sums of d terms in S, the exponential to 2^-18, O rounded once
    e = d * 2.0 ** -24 * q.double().abs().amax() * kp.double().abs().sum(-1).amax() * d ** -0.5 + 2.0 ** -18
    assert_within("o", o, want, (u + e) * spread + u * want.abs())
    assert ((lse - want_lse).abs() <= e + 2.0 ** -20 * (1 + want_lse.abs())).all()
