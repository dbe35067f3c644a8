"""Sums over many keys of a 4-bit cache: weights that are equal and exact, so that nothing but the sums of the codes can be off."""
import pytest
import torch

from flashck_b200 import _lib, ops

pytestmark = pytest.mark.gpu
KEYS, HEADS, FIRST = 65536, 8, 64


def _cache(batch, d, group):
    """Keys of zero; values with codes 1..15, scale 2^-6 for a sequence's first 64 keys and 2^-6 (1 + 1023 / 1024) for the rest, least value -8
    scales.  Returns the parts, the block table and the 64-bit mean of the values over the keys, [batch, heads, d]."""
    g = torch.Generator("cuda").manual_seed(d + group)
    pages, groups = batch * KEYS // 64, d // group
    codes = torch.randint(1, 16, (pages, 64, HEADS, d), generator=g, device="cuda", dtype=torch.uint8)
    scale = torch.full((batch, KEYS), 2.0 ** -6 * (1 + 1023 / 1024), device="cuda")
    scale[:, :FIRST] = 2.0 ** -6
    vp = torch.stack([scale, -8 * scale], -1).view(pages, 64, 1, 1, 2).expand(-1, -1, HEADS, groups, -1).to(torch.float16).contiguous()
    vc = codes[..., ::2] | codes[..., 1::2] << 4
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    kept = torch.empty_like(vc), torch.empty_like(vp)
    for x, y in zip(kept, (vc, vp)):
        x[table.long()] = y
    u = codes.view(batch, KEYS, HEADS, d)
    first, rest = (x.sum(1, dtype=torch.int64) - 8 * x.shape[1] for x in (u[:, :FIRST], u[:, FIRST:]))
    want = (first.double() * scale[0, 0].double() + rest.double() * scale[0, -1].double()) / KEYS
    k = torch.zeros_like(vc), torch.zeros_like(vp)
    return (*k, *kept), table.view(batch, -1), want


@pytest.mark.parametrize("d,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("tokens,heads_per_kv", [([1], 4), ([1], 8), ([1], 16), ([3], 8), ([1, 4], 4), ([2, 4], 4)],
                         ids=["4 rows", "8 rows", "16 rows", "24 rows", "4 and 16 rows", "8 and 16 rows"])
def test_sums_of_many_keys_keep_their_bits(d, group, tokens, heads_per_kv):
    """One split: a warp sums up to 65536 keys.

    Bounds.  With q = 0 all weights p are equal, and the reference of a warp, set at its first keys, makes its weights p s 2^4 there and 2^4 (1 +
    1023 / 1024) behind them, halves both; p (m + 8 s) is 0.  A sum of w u is a multiple of 2^-6; over 256 keys it is below 256 * 32 * 15 = 2^16.9,
    and what is left of 65536 keys less 8 w each is a walk of 4.4 * 32 * 256 = 2^15.2: below 2^18 together, 24 bits, which 32-bit sums hold
    exactly, cut off or not.  So even channels are off by the output's rounding (2^-11, or 2^-25 below its normal numbers), and by 2^-17 of
    themselves for exponential, quotient and merge.  Odd channels come from sums of w (16 u' + u), below 2^21 + 2^19.3, whose cut off products lose up
    to 17 * 2^-2 for 16 keys: over 16, against 16 keys of weight 32, 17 / 4 / 16 / 512 of a scale.  Uncentred, the even sums of half of the keys
    pass 2^23, and cuts of half a unit for 16 keys are 2^-10 of 512 already, on one side."""
    parts, table, want = _cache(len(tokens), d, group)
    packed = len(set(tokens)) > 1
    q = torch.zeros(sum(tokens), HEADS * heads_per_kv, d, device="cuda", dtype=torch.float16)
    kw = dict(cu_seqlens_q=torch.tensor([0] + tokens, device="cuda").cumsum(0), max_seqlen_q=max(tokens)) if packed else {}
    o = ops.fmha_fwd_splitkv_int4(q if packed else q.view(len(tokens), -1, *q.shape[1:]), *parts, seqlen_k=torch.full((len(tokens),), KEYS, device="cuda", dtype=torch.int32),
                                  block_table=table, num_splits=1, **kw)
    o, scale, row = o.view(sum(tokens), HEADS, heads_per_kv, d).double(), 2.0 ** -5, 0
    for s, t in enumerate(tokens):
        off = o[row: row + t] - want[s][None, :, None]
        row += t
        assert (off.abs() <= (2.0 ** -11 + 2.0 ** -17) * want[s][None, :, None].abs() + 2.0 ** -25)[..., ::2].all(), \
            f"sequence {s}: even channels off by {(off[..., ::2].abs().max() / scale).item():.3g} of a scale, {(off[..., ::2].mean() / scale).item():.3g} in the mean"
        assert (off[..., 1::2].abs() <= (2.0 ** -11 + 2.0 ** -17) * want[s][None, :, None, 1::2].abs() + 17 / 4 / 16 / 512 * scale + 2.0 ** -25).all(), \
            f"sequence {s}: odd channels off by {(off[..., 1::2].abs().max() / scale).item():.3g} of a scale"
    assert _lib.device_status() == 0
