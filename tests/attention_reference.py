"""Attention and its gradients in 64 bits, and bounds on what roundings may do to them."""
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def visible(sq, sk, mask, device):
    """``mask``: (mask_type, left, right) as the C ABI has it."""
    kind, left, right = mask
    i, j = torch.arange(sq, device=device)[:, None], torch.arange(sk, device=device)[None]
    seen = torch.ones(sq, sk, dtype=torch.bool, device=device)
    if kind:
        i = i + (sk - sq if kind == 2 else 0)
        if left >= 0:
            seen &= j >= i - left
        if right >= 0:
            seen &= j <= i + right
    return seen


def _scores(q, k, scale, mask, bias, slopes, cap):
    """q [b, h, sq, d], k [b, h, sk, d] in 64 bits -> (scores, -inf where hidden; derivative of the cap)."""
    x = (q @ k.transpose(2, 3)) * scale
    slope = torch.ones_like(x)
    if cap > 0:
        t = torch.tanh(x / cap)
        x, slope = cap * t, 1 - t * t
    sq, sk = x.shape[2:]
    if bias is not None:
        x = x + bias.double()
    if slopes is not None:
        away = (torch.arange(sq, device=x.device)[:, None] + sk - sq - torch.arange(sk, device=x.device)[None]).abs()
        x = x - slopes.double()[:, :, None, None] * away
    return x.masked_fill(~visible(sq, sk, mask, x.device), -torch.inf), slope


def _heads_first(t, hq):
    t = t.double().transpose(1, 2)
    return t.repeat_interleave(hq // t.shape[1], dim=1)


def forward(q, k, v, scale, mask, bias=None, slopes=None, cap=0.0):
    """BSHD -> (o [b, sq, hq, d], lse [b, hq, sq]) in 64 bits; rows that see nothing: o = 0, lse = -inf."""
    hq = q.shape[2]
    x, _ = _scores(_heads_first(q, hq), _heads_first(k, hq), scale, mask, bias, slopes, cap)
    lse = torch.logsumexp(x, dim=-1) if x.shape[-1] else x.new_full(x.shape[:-1], -torch.inf)
    p = torch.where(torch.isneginf(lse)[..., None], 0.0, torch.exp(x - lse.masked_fill(torch.isneginf(lse), 0.0)[..., None]))
    return (p @ _heads_first(v, hq)).transpose(1, 2).contiguous(), lse


def gradients(dout, q, k, v, o, lse, scale, mask, bias=None, slopes=None, cap=0.0, dlse=None):
    """(dq, dk, dv, dT) and the bounds of their errors, all in 64 bits; dT is [b, hq, sq, sk].

    The bounds count, for inputs of half step u: P and dS rounded to the element type where they enter a product (u each), the
    result rounded once (u), sums of d fp32 terms (d 2^-24 of the sum of magnitudes) in S, dP and D, and 2^-18 for the
    exponential (the polynomial of the tcgen05 kernels is good to 2.7e-6 = 2^-18.5); the soft cap's tanh is good to 2^-21 of the cap."""
    hq, hkv, d, u = q.shape[2], k.shape[2], q.shape[3], half_step(q.dtype)
    qd, kd, vd = (_heads_first(t, hq) for t in (q, k, v))
    do, od = _heads_first(dout, hq), _heads_first(o, hq)
    x, slope = _scores(qd, kd, scale, mask, bias, slopes, cap)
    lse = lse.double()[..., None]
    p = torch.where(torch.isneginf(lse) | torch.isneginf(x), 0.0, torch.exp(x - lse.masked_fill(torch.isneginf(lse), 0.0)))
    delta = (do * od).sum(-1, keepdim=True)
    if dlse is not None:
        delta = delta - dlse.double()[..., None]
    dt = p * (do @ vd.transpose(2, 3) - delta)
    ds = dt * slope

    def grouped(t):
        return t.unflatten(1, (hkv, hq // hkv)).sum(2).transpose(1, 2)

    dv, dk, dq = grouped(p.transpose(2, 3) @ do), grouped(ds.transpose(2, 3) @ qd) * scale, (ds @ kd).transpose(1, 2) * scale
    sums = d * 2.0 ** -24
    # relative error of a P: what the sum in S moves the exponent by, the exponential itself; the largest additions in fp32
    big = x.masked_fill(torch.isneginf(x), 0.0).abs() + lse.masked_fill(torch.isneginf(lse), 0.0).abs()
    e = sums * scale * (qd.abs() @ kd.abs().transpose(2, 3)) + 2.0 ** -18 + 2.0 ** -22 * big + (cap * 2.0 ** -21 + 2.0 ** -12 if cap else 0.0)
    mag = do.abs() @ vd.abs().transpose(2, 3) + (do * od).abs().sum(-1, keepdim=True)
    e_dt = e * dt.abs() + 2 * sums * p * mag
    tiny = torch.finfo(q.dtype).smallest_normal * u if q.dtype == torch.float16 else 0.0  # (fp16: half the spacing of its subnormals)
    b_dv = grouped((p * (e + u) + tiny).transpose(2, 3) @ do.abs())
    e_ds = e_dt + u * ds.abs() + tiny
    b_dk = grouped(e_ds.transpose(2, 3) @ qd.abs()) * scale
    b_dq = (e_ds @ kd.abs()).transpose(1, 2) * scale
    bounds = [b + u * t.abs() + tiny for b, t in ((b_dq, dq), (b_dk, dk), (b_dv, dv))] + [e_dt]
    return (dq, dk, dv, dt), bounds


def assert_within(name, got, want, bound):
    got = got.double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{name}: {int((over > 0).sum())} of {over.numel()} beyond the bound, worst by {over.max().item():.3g}"
