"""Values whose groups of channels have scales far apart, against 64 bits: each channel by its own group's scales."""
import pytest
import torch

import int4_reference as ref
from flashck_b200 import _lib, ops

pytestmark = pytest.mark.gpu


def _bound(q, kc, kp, vc, vp, scale, mask):
    """(o, its bound, lse, its bound) as ref.attend has them, but for what a weight loses below a half's normal numbers, which counts by the scales of
    the channel's own group: 8 n 2^-24 of the largest p s there.  (Summed up anew: a bound of all groups does not go back to a small one's.)"""
    o, lse, _, lse_bound = ref.attend(q, kc, kp, vc, vp, scale, mask)
    n, hq, d = kc.shape[0], q.shape[1], q.shape[2]
    per, bound = hq // kc.shape[1], torch.zeros_like(o)
    k = ref.values(kc, kp)
    ks, vs, kl, vl = (p[..., i].double().repeat_interleave(d // p.shape[-2], -1) for i in (0, 1) for p in (kp, vp))
    seen = ref.visible(q.shape[0], n, mask, q.device)
    for h in range(hq):
        kh = h // per
        x = torch.where(seen, q[:, h].double() @ k[:, kh].T * scale, -torch.inf)
        any_ = seen.any(-1)
        p = torch.where(any_[:, None], torch.exp(x - torch.where(any_, torch.logsumexp(x, -1), 0)[:, None]), 0)
        size = (q[:, h].double().abs() @ (kl[:, kh].abs() + 15 * ks[:, kh]).T * abs(scale)).masked_fill(~seen, 0).amax(-1)
        e = 2.0 ** -20 * (size + 1) + 2.0 ** -22 * torch.where(seen, x, 0).abs().amax(-1)
        top = (p[:, :, None] * vs[None, :, kh]).amax(1)
        bound[:, h] = ref.half_step(q.dtype) * o[:, h].abs() * 1.01 + 2.0 ** -11 * (p @ (8 * vs[:, kh])) + 8 * n * 2.0 ** -24 * top + \
            (3 * e[:, None] + 2.0 ** -18) * (p @ (vl[:, kh].abs() + 15 * vs[:, kh]))
    return o, lse, bound, lse_bound


def _hold(tokens, lens, hq, hkv, d, group, dtype, factor, mask=(2, -1, 0), queries=1.0, splits=0):
    """factor(tokens of a sequence) -> [tokens, groups]: what a token's scales and least values of each group are multiplied by."""
    g = torch.Generator("cuda").manual_seed(5)
    caps, sequences = max(lens), []
    parts = [torch.zeros(len(lens), caps, hkv, d // 2, dtype=torch.uint8, device="cuda"), torch.zeros(len(lens), caps, hkv, d // group, 2, dtype=dtype, device="cuda")]
    parts += [x.clone() for x in parts]
    for s, n in enumerate(lens):
        four = []
        for i in range(2):
            c, sc, lo = ref.quantise(torch.randn(n, hkv, d, generator=g, device="cuda").to(dtype), group)
            params = torch.stack([sc, lo], -1)
            if i:
                params = params * factor(n)[:, None, :, None]
            four += [ref.pack(c), params.to(dtype)]
        for part, x in zip(parts, four):
            part[s, :n] = x
        sequences.append(four)
    qs = [(torch.randn(t, hq, d, generator=g, device="cuda") * queries).to(dtype) for t in tokens]
    packed = len(set(tokens)) > 1
    kw = dict(cu_seqlens_q=torch.tensor([0] + tokens, device="cuda").cumsum(0), max_seqlen_q=max(tokens)) if packed else {}
    o, lse = ops.fmha_fwd_splitkv_int4(torch.cat(qs) if packed else torch.stack(qs), *parts, seqlen_k=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                                       mask_type=mask[0], window_size=mask[1:], num_splits=splits, return_lse=True, **kw)
    row = 0
    for s, t in enumerate(tokens):
        got, got_lse = (o[row: row + t], lse[:, row: row + t]) if packed else (o[s], lse[s])
        row += t
        want, want_lse, bound, lse_bound = _bound(qs[s], *sequences[s], d ** -0.5, mask)
        ref.assert_within(f"o of sequence {s}", got, want, bound)
        seen = ~torch.isneginf(want_lse)
        assert torch.equal(torch.isneginf(got_lse), ~seen) and ((got_lse - want_lse).abs()[seen] <= lse_bound[seen]).all()
    assert _lib.device_status() == 0


SHAPES = [(128, 64), (128, 32), (64, 32)]
ROWS = [([1, 1], 8, 2), ([1, 1], 16, 2), ([1, 4], 8, 2), ([5, 5], 8, 2)]


@pytest.mark.parametrize("tokens,hq,hkv", ROWS)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("power", [-12, -20, -28, -60])
def test_a_group_of_small_scales(d, group, tokens, hq, hkv, power):
    groups = d // group
    small = 2.0 ** torch.linspace(0, power, groups, device="cuda")
    _hold(tokens, [700, 300], hq, hkv, d, group, torch.bfloat16, lambda n: small.expand(n, -1))


@pytest.mark.parametrize("tokens,hq,hkv", ROWS)
@pytest.mark.parametrize("d,group", SHAPES)
@pytest.mark.parametrize("splits", [0, 1])
def test_groups_whose_scales_cross(d, group, tokens, hq, hkv, splits):
    """One group's scales grow by 2^40 along the keys, the other ones' shrink: with few tokens in sight they are far apart both ways."""
    def factor(n):
        up = 2.0 ** torch.linspace(-40, 0, n, device="cuda")
        return torch.stack([up if k % 2 else up.flip(0) for k in range(d // group)], -1)
    _hold(tokens, [900, 450], hq, hkv, d, group, torch.bfloat16, factor, queries=3.0, splits=splits)


@pytest.mark.parametrize("tokens,hq,hkv", ROWS)
@pytest.mark.parametrize("d,group", SHAPES)
def test_the_weight_decides_with_the_scale(d, group, tokens, hq, hkv):
    """Groups with large scales only at keys of small weight, zero scales among the rest."""
    def factor(n, least):
        f = torch.full((n, d // group), least, device="cuda")
        f[:, 0] = 1
        f[n // 2: n // 2 + 3, -1] = 1.0
        f[: n // 4, -1] = 0
        return f
    for dtype, least in ((torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -26)):
        _hold(tokens, [512, 260], hq, hkv, d, group, dtype, lambda n: factor(n, least), mask=(2, 100, 0), queries=6.0)
