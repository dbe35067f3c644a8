"""The 4-bit cache, the rotation and attention over such a cache, stated in 64 bits channel by channel (group by group) for the tests."""
import torch

from attention_reference import assert_within, half_step, visible  # noqa: F401


def quantise(x, group):
    """codes [..., d] as integers, scale and least value [..., d / group] of x [..., d]; each comparison decided in 64 bits."""
    parts = x.double().unflatten(-1, (-1, group))
    lo, hi = parts.amin(-1), parts.amax(-1)
    scale = ((hi - lo) / 15).float().to(x.dtype).double()
    r = (parts.float() - lo.float()[..., None]).double()  # (the difference is one of 32 bits)
    codes = torch.zeros_like(r)
    for i in range(15):  # passes i + 1/2 if above it, or on it with an odd code below
        edge = (i + 0.5) * scale[..., None]
        codes += ((r > edge) | ((r == edge) & (i % 2 == 1))) & (scale[..., None] > 0)
    return codes.flatten(-2).long(), scale, lo


def pack(codes):
    return (codes[..., ::2] + 16 * codes[..., 1::2]).to(torch.uint8)


def unpack(codes):
    c = codes.long()
    return torch.stack([c % 16, c // 16], -1).flatten(-2)


def values(codes, params):
    """What packed codes [..., d / 2] and params [..., groups, 2] stand for, in 64 bits."""
    u = unpack(codes).double().unflatten(-1, (params.shape[-2], -1))
    return (params[..., 1:].double() + params[..., :1].double() * u).flatten(-2)


def rotate(x, cos, sin, at, pair_axis, interleaved, inverse=False):
    """x [tokens, heads, d] turned by positions at [axes, tokens]: products and sums rounded to 32 bits one by one, the result to x's type."""
    half = cos.shape[1]
    y = x.clone()
    for i in range(half):
        pos = at[pair_axis[i]].long()
        inside = (pos >= 0) & (pos < cos.shape[0])
        c, s = (torch.where(inside, t[pos.clamp(0, cos.shape[0] - 1), i].float(), torch.nan)[:, None] for t in (cos, sin))
        if inverse:
            s = -s
        p, r = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., p].float(), x[..., r].float()
        y[..., p] = (a * c - b * s).to(x.dtype)
        y[..., r] = (a * s + b * c).to(x.dtype)
    return y


def attend(q, kc, kp, vc, vp, scale, mask):
    """q [t, hq, d] over a sequence's codes and params [n, hkv, ...] -> (o [t, hq, d], lse [hq, t], bound of o's error, bound of lse's).

    The bounds, without a constant from a measurement (u: half a step of the output's type).  Scores: the codes' products are summed in 32
    bits, cut off (2^-23 each of up to d / 16 + 2 steps), q's halves are exact to 2^-24 of the row's largest, and x - R is a difference of 32
    bits: in all below e = 2^-20 of the largest sum of magnitudes, 2^-20 of 1, and 2^-22 of the score itself.  Weights p s are rounded to
    halves (2^-11), or to 2^-25 where they are below 2^-14 with the largest above 1/2 (its own p s then counts 2^-24); they meet codes less 8.
    The rest of O (sums in 32 bits, cut off at each of the few steps between two centrings) is below 2^-18 of the sum of magnitudes."""
    t, hq, d = q.shape
    n, hkv = kc.shape[:2]
    u, g = half_step(q.dtype), hq // hkv
    o, lse = torch.zeros(t, hq, d, dtype=torch.float64, device=q.device), torch.full((hq, t), -torch.inf, dtype=torch.float64, device=q.device)
    bound, lse_bound = torch.zeros_like(o), torch.zeros_like(lse)
    if n == 0:
        return o, lse, bound, lse_bound
    k, v = values(kc, kp), values(vc, vp)
    ks, vs = (p[..., 0].double().repeat_interleave(d // p.shape[-2], -1) for p in (kp, vp))
    kl, vl = (p[..., 1].double().repeat_interleave(d // p.shape[-2], -1) for p in (kp, vp))
    seen = visible(t, n, mask, q.device)
    for h in range(hq):
        kh = h // g
        x = torch.where(seen, q[:, h].double() @ k[:, kh].T * scale, -torch.inf)
        size = (q[:, h].double().abs() @ (kl[:, kh].abs() + 15 * ks[:, kh]).T * abs(scale)).masked_fill(~seen, 0).amax(-1)
        any_ = seen.any(-1)
        e = 2.0 ** -20 * (size + 1) + 2.0 ** -22 * torch.where(seen, x, 0).abs().amax(-1)
        l = torch.logsumexp(x, -1)
        p = torch.where(any_[:, None], torch.exp(x - torch.where(any_, l, 0)[:, None]), 0)
        zero = lambda a: torch.where(seen.any(0)[:, None], a, 0.0)  # noqa: E731  (what no row sees may be anything)
        o[:, h] = p @ zero(v[:, kh])
        all_, eight = p @ zero(vl[:, kh].abs() + 15 * vs[:, kh]), p @ zero(8 * vs[:, kh])
        top = (p[:, :, None] * zero(vs[:, kh])[None]).amax(1)
        few = 8 * n * 2.0 ** -24 * top.amax(-1, keepdim=True)
        bound[:, h] = u * o[:, h].abs() * 1.01 + 2.0 ** -11 * eight + few + (3 * e[:, None] + 2.0 ** -18) * all_
        lse[h] = l
        lse_bound[h] = torch.where(any_, e + 2.0 ** -20 * (1 + torch.where(any_, l, 0).abs()), 0)
    return o, lse, bound, lse_bound
