"""Rotary embedding of queries and keys by itself, with positions along one or several axes (C symbol ``FmhaRotary``).

Decode and append turn their rows as they write the cache (:func:`fmha_fwd_append_kv`, :func:`fmha_fwd_append_kv_int4`); prefill and
training turn them before the attention, here.  Images and video have a position along time, height and width for each token, and each
axis turns its own pairs of a head.
"""
from __future__ import annotations

import functools
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib
from ..utils.enums import RopeEnum
from . import fmha as _f
from .gradients import _ON_DEFAULT_STREAM, _mark_leaves, _same_device

__all__ = ["apply_rotary", "apply_rotary_autograd"]

_MAX_AXES = 4


@functools.lru_cache(maxsize=256)
def _pair_axes(sections: Optional[Tuple[int, ...]], interleaved: bool, half: int, axes: int) -> Optional[bytes]:
    """The axis of each of the ``half`` pairs, or None where there is one axis."""
    if not 1 <= axes <= _MAX_AXES:
        raise ValueError(f"positions must have 1 to {_MAX_AXES} axes, got {axes}")
    if sections is None:
        if axes != 1:
            raise ValueError(f"positions along {axes} axes need sections")
        return None
    if len(sections) != axes or min(sections) < 0 or sum(sections) != half:
        raise ValueError(f"sections must be {axes} numbers of pairs that sum to rotary_dim / 2 = {half}, got {sections}")
    if not interleaved:
        return bytes(a for a, n in enumerate(sections) for _ in range(n))
    left, order = list(sections), []
    while len(order) < half:  # dealt out in turn to the axes that have pairs left
        for a in range(axes):
            if left[a]:
                left[a] -= 1
                order.append(a)
    return bytes(order)


def _tables(cos: torch.Tensor, sin: torch.Tensor, dtype: torch.dtype, rotary_dim: Optional[int]) -> Tuple[int, int]:
    """(rotary_dim, rows) of the tables ``[positions, rotary_dim / 2]``."""
    for n, t in (("rotary_cos", cos), ("rotary_sin", sin)):
        if t is None:
            raise TypeError(f"{n} must be a torch.Tensor")
        _f._check_cuda(n, t, dtype)
        if t.dim() != 2:
            _f._refuse(n, t, "2 dimensions [positions, rotary_dim / 2]")
    if cos.shape != sin.shape or (rotary_dim is not None and int(rotary_dim) != 2 * cos.shape[1]):
        raise ValueError(f"the rotary tables must be [positions, rotary_dim / 2], got {tuple(cos.shape)} and {tuple(sin.shape)}")
    return 2 * cos.shape[1], cos.shape[0]


def _as_positions(positions: torch.Tensor, tokens: int, sections: Optional[Sequence[int]] = None) -> Tuple[torch.Tensor, int]:
    """(positions int32 [axes, tokens], axes).  Positions of no token have as many axes as there are sections."""
    if positions is None or not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be a torch.Tensor")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must have dtype torch.int32 or torch.int64, got {positions.dtype}")
    # (the kernels hold 32 bits: what lies behind them is outside every table, and must not come back to it)
    p = _f._as_i32("positions", positions.clamp(-1, 2 ** 31 - 1) if positions.dtype == torch.int64 and positions.is_cuda else positions)
    axes = p.numel() // tokens if tokens else 1 if sections is None else len(sections)
    if p.numel() != axes * tokens or axes < 1 or (axes > 1 and p.shape[0] != axes):
        _f._refuse("positions", positions, f"{tokens} positions, or [axes, ...] of them")
    return p, axes


def _rotary(q, k, positions, cos, sin, sections, interleaved_sections, rope, inverse):
    rope = int(rope)
    native = _f._native()
    if native:
        r = native._call_rotary(q, k, positions, cos, sin, sections, interleaved_sections, rope, inverse)
        if r is not None:
            return r if r.__class__ is not int else _lib.check(r, "FmhaRotary")
    if q is None:
        raise TypeError("q must be a torch.Tensor")
    _f._check_cuda("q", q)
    code = _f._dtype_code(q)
    _f._check_cuda("k", k, q.dtype)
    if q.dim() < 3:
        _f._refuse("q", q, "3 dimensions or more [..., heads, hdim]")
    lead, (hq, d) = q.shape[:-2], q.shape[-2:]
    if k is not None and (k.dim() != q.dim() or k.shape[:-2] != lead or k.shape[-1] != d):
        raise ValueError(f"inconsistent shapes q{tuple(q.shape)} k{tuple(k.shape)}")
    tokens = 1
    for n in lead:
        tokens *= n
    if rope not in (int(RopeEnum.INTERLEAVED), int(RopeEnum.HALF_ROTATED)):
        raise ValueError("rope must be RopeEnum.INTERLEAVED or RopeEnum.HALF_ROTATED")
    pos, axes = _as_positions(positions, tokens, sections)
    rotary_dim, rows = _tables(cos, sin, q.dtype, None)
    if rotary_dim > d:
        raise ValueError(f"the rotary tables turn {rotary_dim} columns of heads of {d}")
    pairs = _pair_axes(None if sections is None else tuple(int(n) for n in sections), bool(interleaved_sections), rotary_dim // 2, axes)
    _same_device(q, k=k, positions=pos, rotary_cos=cos, rotary_sin=sin)
    q_out = torch.empty_like(q)
    k_out = torch.empty_like(k) if k is not None else None
    with _f._on(q.device):
        rc = _lib.lib().FmhaRotary(_f._ptr(q), _f._ptr(q_out), _f._ptr(k), _f._ptr(k_out), _f._ptr(pos), _f._ptr(cos), _f._ptr(sin), pairs,
                                   axes, tokens, hq, k.shape[-2] if k is not None else 0, d, rotary_dim, rows, rope, int(bool(inverse)),
                                   _f._stream(), code)
    _lib.check(rc, "FmhaRotary")
    return q_out, k_out


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary_cos: torch.Tensor, rotary_sin: torch.Tensor, *,
                 sections: Optional[Sequence[int]] = None, interleaved_sections: bool = False, rope: int = RopeEnum.HALF_ROTATED,
                 inverse: bool = False):
    """Rotary embedding of q ``[..., hq, d]`` and k ``[..., hkv, d]`` (or None), which have the same tokens.  Returns new tensors
    ``(q, k)``.

    positions: int32 or int64, one per token, or ``[axes, ...]`` of them (up to 4 axes) with ``sections``: the number of pairs of a head that
    turn with each axis, summing to ``rotary_dim / 2``; one run per axis, or with ``interleaved_sections`` dealt out in turn.
    rotary_cos / rotary_sin ``[positions, rotary_dim / 2]`` in q's dtype, as in :func:`fmha_fwd_append_kv`; the channels behind
    ``rotary_dim`` are copied.  A position outside the tables turns by NaN.  ``inverse`` turns the other way, which is the gradient."""
    return _rotary(q, k, positions, rotary_cos, rotary_sin, sections, interleaved_sections, rope, inverse)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, options):
        ctx.save_for_backward(positions, cos, sin)
        ctx.options = options
        ctx.set_materialize_grads(False)
        return _rotary(q, k, positions, cos, sin, *options, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        if torch.cuda.is_current_stream_capturing() and any(n.metadata.get(_ON_DEFAULT_STREAM) for n, _ in ctx.next_functions if n is not None):
            raise RuntimeError("this backward pass is being captured, but an input's gradient belongs to a graph that was recorded on the default "
                               "stream and still lives: release that graph's outputs, or record it on a side stream")
        dq, dk = (g if g is None or not need else g.contiguous() for g, need in zip((dq, dk), ctx.needs_input_grad))
        dq, dk = (g if need else None for g, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is not None:
            dq, dk = _rotary(dq, dk, *ctx.saved_tensors, *ctx.options, True)
        elif dk is not None:
            dk, _ = _rotary(dk, None, *ctx.saved_tensors, *ctx.options, True)
        return dq, dk, None, None, None, None


def apply_rotary_autograd(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, rotary_cos: torch.Tensor, rotary_sin: torch.Tensor,
                          *, sections: Optional[Sequence[int]] = None, interleaved_sections: bool = False,
                          rope: int = RopeEnum.HALF_ROTATED):
    """:func:`apply_rotary` as a function that autograd differentiates with respect to q and k (the tables are constants).  About captured
    backward passes see :func:`fmha_autograd`."""
    for n, t in (("rotary_cos", rotary_cos), ("rotary_sin", rotary_sin)):
        if isinstance(t, torch.Tensor) and t.requires_grad:
            raise ValueError(f"{n} is a constant: its gradient is not computed")
    held = _mark_leaves(q, k) if torch.is_grad_enabled() else None  # noqa: F841
    return _Rotary.apply(q, k, positions, rotary_cos, rotary_sin, (None if sections is None else tuple(sections), interleaved_sections, rope))
