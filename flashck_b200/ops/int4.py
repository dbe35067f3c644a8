"""Serving from a key/value cache held in 4 bits: its write, decode over it, and its way back to 16-bit keys and values.

A group of 32, 64 or 128 neighbouring channels of one token's head is held as ``lo + scale * code``: lo the group's least value, scale
``(greatest - lo) / 15`` in the model's dtype, code 0..15 the nearest, ties to even.  A cache is a pair of tensors (:func:`int4_cache`):
codes uint8 ``[pages, page, hkv, d / 2]``, byte j with channel 2j in its low and 2j + 1 in its high half, and params
``[pages, page, hkv, d / group, 2]`` = (scale, lo) in the model's dtype; or ``[b_cache, capacity, ...]`` of both without a block table.
Against a 16-bit cache it takes 17 / 64 (group 128) to 5 / 16 (group 32) of the bytes, which is what decode is bound by.

A page id outside the pools is not followed, nor a ``cache_batch_idx`` outside the block table or the contiguous rows: reads take zeros there,
writes are skipped and reported (:func:`_lib.device_status`).
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from .. import _lib
from ..utils.enums import RopeEnum
from . import fmha as _f
from .rotary import _as_positions, _pair_axes, _tables

__all__ = ["int4_cache", "fmha_fwd_append_kv_int4", "fmha_fwd_splitkv_int4", "fmha_read_kv_int4"]


def int4_cache(pages: int, page: int, hkv: int, d: int, *, group: int = 0, dtype: torch.dtype = torch.bfloat16,
               device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes, params)`` of ``pages`` pages of ``page`` tokens (or of rows and their capacity), holding zeros.  group 0: a whole head."""
    group = int(group) or d
    if d not in (64, 128) or group not in (32, 64, 128) or group > d:
        raise ValueError(f"a 4-bit cache has heads of 64 or 128 channels in groups of 32, 64 or 128, got {d} in groups of {group}")
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"attention supports torch.float16 and torch.bfloat16, got {dtype}")
    return (torch.zeros(pages, page, hkv, d // 2, dtype=torch.uint8, device=device),
            torch.zeros(pages, page, hkv, d // group, 2, dtype=dtype, device=device))


def _same_device(device: torch.device, **tensors: Optional[torch.Tensor]) -> None:
    for n, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{n} must be on {device} like the other tensors, got {t.device}")


class _Cache:
    """The checked parts of a cache: sizes and what the C calls take of them."""

    def __init__(self, k_cache, k_params, v_cache, v_params, seqlen_k, block_table, cache_batch_idx, dtype, device, paged_unit):
        for n, t, dt in (("k_cache", k_cache, torch.uint8), ("k_params", k_params, dtype), ("v_cache", v_cache, torch.uint8),
                         ("v_params", v_params, dtype), ("seqlen_k", seqlen_k, None)):
            if t is None:
                raise TypeError(f"{n} must be a torch.Tensor")
            _f._check_cuda(n, t, dt)
        if k_cache.dim() != 4 or k_cache.shape[3] not in (32, 64):
            _f._refuse("k_cache", k_cache, "shape [pages, page, hkv, d / 2] with d 64 or 128")
        self.pool, self.page, self.hkv, half = k_cache.shape
        self.d = 2 * half
        if k_params.dim() != 5 or k_params.shape[:3] != k_cache.shape[:3] or k_params.shape[4] != 2 or \
                k_params.shape[3] not in (1, 2, 4) or self.d // k_params.shape[3] < 32:
            _f._refuse("k_params", k_params, f"shape {tuple(k_cache.shape[:3])} + [d / group, 2] with groups of 32, 64 or 128 channels")
        if v_cache.shape != k_cache.shape or v_params.shape != k_params.shape:
            raise ValueError(f"inconsistent shapes k{tuple(k_cache.shape)} {tuple(k_params.shape)} v{tuple(v_cache.shape)} {tuple(v_params.shape)}")
        self.group = self.d // k_params.shape[3]
        for n, t in (("k_cache", k_cache), ("k_params", k_params), ("v_cache", v_cache), ("v_params", v_params)):
            if t.data_ptr() % 16:
                raise ValueError(f"{n} must start at a multiple of 16 bytes")
        self.seqlen = _f._as_i32("seqlen_k", seqlen_k)
        self.batch = self.seqlen.numel()
        if self.seqlen.dim() != 1 or self.batch < 1:
            _f._refuse("seqlen_k", seqlen_k, "one dimension and an entry for each sequence")
        self.table = _f._as_i32("block_table", block_table) if block_table is not None else None
        self.index = _f._as_i64("cache_batch_idx", cache_batch_idx) if cache_batch_idx is not None else None
        self.bt_stride = 0
        if self.table is not None:
            if self.table.dim() != 2 or self.table.shape[1] < 1 or (self.index is None and self.table.shape[0] < self.batch):
                _f._refuse("block_table", self.table, f"a row for each of the {self.batch} sequences and a column for their pages")
            self.bt_stride = self.table.shape[1]
            if self.page % paged_unit:
                raise ValueError(f"pages must have a multiple of {paged_unit} tokens, got {self.page}")
        elif self.index is None and self.pool < self.batch:
            _f._refuse("k_cache", k_cache, f"a row for each of the {self.batch} sequences")
        if self.index is not None and self.index.numel() < self.batch:
            _f._refuse("cache_batch_idx", self.index, f"{self.batch} entries")
        _same_device(device, k_cache=k_cache, k_params=k_params, v_cache=v_cache, v_params=v_params, seqlen_k=self.seqlen,
                     block_table=self.table, cache_batch_idx=self.index)
        if self.table is not None and self.index is not None:
            # The kernels do not know how many rows the table has: the rows are picked here, and one that is not there has no page.
            table, index = self.table, self.index.flatten()[:self.batch]
            there = (index >= 0) & (index < table.shape[0])
            picked = table[index.clamp(0, table.shape[0] - 1)] if table.shape[0] else table.new_empty(self.batch, self.bt_stride)
            self.table, self.index = torch.where(there[:, None], picked, -1), None


def fmha_fwd_append_kv_int4(q: Optional[torch.Tensor], k_cache: torch.Tensor, k_params: torch.Tensor, v_cache: torch.Tensor,
                            v_params: torch.Tensor, knew: torch.Tensor, vnew: torch.Tensor, seqlen_k: torch.Tensor,
                            rotary_cos: Optional[torch.Tensor] = None, rotary_sin: Optional[torch.Tensor] = None, *,
                            rope: int = RopeEnum.INTERLEAVED, rotary_dim: Optional[int] = None, positions: Optional[torch.Tensor] = None,
                            sections: Optional[Sequence[int]] = None, interleaved_sections: bool = False,
                            block_table: Optional[torch.Tensor] = None, cache_batch_idx: Optional[torch.Tensor] = None,
                            cu_seqlens_q: Optional[torch.Tensor] = None, cu_seqlens_knew: Optional[torch.Tensor] = None,
                            return_kv: bool = False):
    """RoPE on the queries and the new keys, and the write of the new keys and values in 4 bits (C symbol ``FmhaFwdAppendKVInt4``).

    As :func:`fmha_fwd_append_kv`, to a cache of :func:`int4_cache`: ``seqlen_k`` counts the cached tokens *before* the append, q, knew,
    vnew are ``[b, n, h, d]`` or packed with ``cu_seqlens_*``, a token that does not fit is skipped and reported.  Two things differ: q is
    left as it is and the turned queries are returned, and tokens may have ``positions`` of their own, ``[axes, ...]`` of the new tokens
    with ``sections`` as in :func:`apply_rotary` (the queries are the last new tokens of their sequence); without them token j of a
    sequence is at ``seqlen_k + j``.

    Returns the turned q (None if q is None); with ``return_kv`` also the values that the cache now holds for the new keys and values, like
    knew and vnew.  Rows that belong to no sequence are zero."""
    rope = int(rope)
    native = _f._native()
    if native and cache_batch_idx is None:
        r = native._call_append_kv_int4(q, k_cache, k_params, v_cache, v_params, knew, vnew, seqlen_k, rotary_cos, rotary_sin, rope, rotary_dim,
                                        positions, sections, interleaved_sections, block_table, cu_seqlens_q, cu_seqlens_knew, return_kv)
        if r is not None:
            return r if r.__class__ is not int else _lib.check(r, "FmhaFwdAppendKVInt4")
    if knew is None or vnew is None:
        raise TypeError("knew and vnew must be torch.Tensors")
    _f._check_cuda("knew", knew)
    code = _f._dtype_code(knew)
    _f._check_cuda("vnew", vnew, knew.dtype)
    _f._check_cuda("q", q, knew.dtype)
    c = _Cache(k_cache, k_params, v_cache, v_params, seqlen_k, block_table, cache_batch_idx, knew.dtype, knew.device, 1)
    group_mode = cu_seqlens_knew is not None
    cu_n = _f._as_i64("cu_seqlens_knew", cu_seqlens_knew) if group_mode else None
    if q is not None and (cu_seqlens_q is not None) != group_mode:
        raise ValueError("cu_seqlens_q and cu_seqlens_knew go together")
    cu_q = _f._as_i64("cu_seqlens_q", cu_seqlens_q) if group_mode and q is not None else None
    dims = 3 if group_mode else 4
    if knew.dim() != dims or knew.shape[-2:] != (c.hkv, c.d) or vnew.shape != knew.shape or (not group_mode and knew.shape[0] != c.batch):
        raise ValueError(f"knew and vnew must be {'[total_new' if group_mode else f'[{c.batch}, n'}, {c.hkv}, {c.d}], got {tuple(knew.shape)} "
                         f"and {tuple(vnew.shape)}")
    if q is not None and (q.dim() != dims or q.shape[-1] != c.d or (not group_mode and q.shape[0] != c.batch)):
        _f._refuse("q", q, f"{dims} dimensions, {c.d} columns like knew, and a row for each sequence")
    for n, t in (("cu_seqlens_knew", cu_n), ("cu_seqlens_q", cu_q)):
        if t is not None and t.numel() != c.batch + 1:
            _f._refuse(n, t, f"{c.batch + 1} entries")
    tokens = knew.shape[0] if group_mode else knew.shape[0] * knew.shape[1]
    axes, pairs, pos, rows = 1, None, None, 0
    if rope:
        if rotary_cos is None or rotary_sin is None:
            raise ValueError("rotary_cos / rotary_sin are required unless rope == RopeEnum.NONE")
        rotary_dim, rows = _tables(rotary_cos, rotary_sin, knew.dtype, rotary_dim)
        if positions is not None:
            pos, axes = _as_positions(positions, tokens, sections)
        pairs = _pair_axes(None if sections is None else tuple(int(n) for n in sections), bool(interleaved_sections), rotary_dim // 2, axes)
    elif positions is not None or sections is not None:
        raise ValueError("positions and sections need a rotation (rope)")
    _same_device(knew.device, q=q, vnew=vnew, rotary_cos=rotary_cos, rotary_sin=rotary_sin, positions=pos, cu_seqlens_q=cu_q, cu_seqlens_knew=cu_n)
    q_out = torch.empty_like(q) if q is not None else None
    held = (torch.empty_like(knew), torch.empty_like(vnew)) if return_kv else (None, None)
    with _f._on(knew.device):
        rc = _lib.lib().FmhaFwdAppendKVInt4(
            _f._ptr(q), _f._ptr(q_out), _f._ptr(k_cache), _f._ptr(k_params), _f._ptr(knew), _f._ptr(v_cache), _f._ptr(v_params), _f._ptr(vnew),
            _f._ptr(held[0]), _f._ptr(held[1]), _f._ptr(c.seqlen), _f._ptr(cu_q), _f._ptr(cu_n), _f._ptr(pos), _f._ptr(rotary_cos),
            _f._ptr(rotary_sin), pairs, _f._ptr(c.table), _f._ptr(c.index), c.batch, (q.shape[0] if group_mode else q.shape[1]) if q is not None else 0,
            knew.shape[0] if group_mode else knew.shape[1], q.shape[-2] if q is not None else 0, c.hkv, c.d, c.group, axes, int(rotary_dim or 0),
            rows, rope, c.bt_stride, c.page, c.pool, _f._stream(), code)
    _lib.check(rc, "FmhaFwdAppendKVInt4")
    return (q_out, *held) if return_kv else q_out


def _split_depth(batch: int, rows: int, hkv: int, sm_count: int = 148) -> int:
    """Workspace depth for :func:`fmha_fwd_splitkv_int4` where the caller leaves it open, for ``rows`` query rows per kv head (``seqlen_q * hq / hkv``).

    As :func:`default_num_splits`, but no more than the grid can use: its CTAs are shared out over the groups of kv heads (up to 8 together) and the
    tiles of 16 rows, and a sequence cut among those that remain touches one piece more than there are.  (One sequence of 2048 queries of 32 / 8
    heads: 34 MB of workspace where 128 splits take 4.3 GB.)"""
    heads = next(n for n in (8, 4, 2, 1) if hkv % n == 0)
    ctas = sm_count // (-(-rows // 16) * (hkv // heads))
    return 1 if ctas <= 1 else min(_f.default_num_splits(batch, sm_count), ctas + 1)


def fmha_fwd_splitkv_int4(q: torch.Tensor, k_cache: torch.Tensor, k_params: torch.Tensor, v_cache: torch.Tensor, v_params: torch.Tensor, *,
                          seqlen_k: torch.Tensor, block_table: Optional[torch.Tensor] = None, cache_batch_idx: Optional[torch.Tensor] = None,
                          cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: int = 0, num_splits: int = 0,
                          scale: Optional[float] = None, causal: bool = False, window_size: Sequence[int] = (-1, -1),
                          mask_type: Optional[int] = None, return_lse: bool = False):
    """Split-KV attention (decode) over a 4-bit cache, followed by the combine (C symbol ``FmhaFwdSplitKVInt4``).

    As :func:`fmha_fwd_splitkv`: q ``[b, sq, hq, d]``, or packed ``[total_q, hq, d]`` with ``cu_seqlens_q``; a cache of :func:`int4_cache`,
    paged (pages of a multiple of 16 tokens) with ``block_table`` int32 ``[b, pages_per_seq]``, or contiguous; ``seqlen_k`` int32 ``[b]``,
    the new tokens among them.  Keys and values count as exactly ``lo + scale * code``; the softmax's weights are rounded to 11 bits on their way to
    the values (of P times scale; sums are 32-bit), and of a query row what is below 2^-34 of its largest magnitude is dropped.  Any number of query
    rows is taken, but the cache is read once per 16 rows of a kv head (``sq * hq / hkv``): a chunk of a prompt goes through
    :func:`fmha_read_kv_int4` and :func:`fmha_fwd_var_len`.  There are no ALiBi slopes.

    Returns o like q (and LSE fp32 ``[b, hq, sq]`` / ``[hq, total_q]``); packed rows that belong to no sequence hold nothing of meaning."""
    native = _f._native()
    if native and cache_batch_idx is None:
        r = native._call_splitkv_int4(q, k_cache, k_params, v_cache, v_params, seqlen_k, block_table, cu_seqlens_q, max_seqlen_q, num_splits, scale,
                                      causal, window_size, mask_type, return_lse)
        if r is not None:
            return r if r.__class__ is not int else _lib.check(abs(r), "FmhaFwdSplitKVInt4" if r > 0 else "FmhaFwdSplitKVCombine")
    if q is None:
        raise TypeError("q must be a torch.Tensor")
    _f._check_cuda("q", q)
    code = _f._dtype_code(q)
    c = _Cache(k_cache, k_params, v_cache, v_params, seqlen_k, block_table, cache_batch_idx, q.dtype, q.device, 16)
    group_mode = cu_seqlens_q is not None
    cu_q = _f._as_i64("cu_seqlens_q", cu_seqlens_q) if group_mode else None
    if q.dim() != (3 if group_mode else 4) or q.shape[-1] != c.d or (not group_mode and q.shape[0] != c.batch):
        _f._refuse("q", q, f"shape {'[total_q' if group_mode else f'[{c.batch}, sq'}, hq, {c.d}]")
    if group_mode and cu_q.numel() != c.batch + 1:
        _f._refuse("cu_seqlens_q", cu_q, f"{c.batch + 1} entries")
    if q.data_ptr() % 16:
        raise ValueError("q must start at a multiple of 16 bytes")
    hq, sq = q.shape[-2], q.shape[-3]
    if hq % c.hkv if c.hkv else True:
        raise ValueError(f"the number of query heads ({hq}) must be a multiple of the kv heads ({c.hkv})")
    _same_device(q.device, cu_seqlens_q=cu_q)
    max_sq = min(int(max_seqlen_q) or sq, sq) if group_mode else sq
    mt, wl, wr = _f._mask(causal, window_size, mask_type)
    o = torch.empty_like(q)
    lse = torch.empty((hq, sq) if group_mode else (c.batch, hq, sq), dtype=torch.float32, device=q.device) if return_lse else None
    if q.numel() == 0:
        return (o, lse) if return_lse else o
    if c.pool == 0 or c.page == 0:
        raise ValueError("the cache has no room")
    splits = int(num_splits) if num_splits and num_splits > 0 else _split_depth(c.batch, max_sq * (hq // c.hkv), c.hkv)
    lse_acc, o_acc = _f.splitkv_workspace(q, c.d, splits, cu_q)
    lib = _lib.lib()
    with _f._on(q.device):
        rc = lib.FmhaFwdSplitKVInt4(_f._ptr(q), _f._ptr(k_cache), _f._ptr(k_params), _f._ptr(v_cache), _f._ptr(v_params), _f._ptr(lse_acc),
                                    _f._ptr(o_acc), _f._ptr(cu_q), _f._ptr(c.seqlen), _f._ptr(c.table), _f._ptr(c.index), c.batch, sq, max_sq, hq,
                                    c.hkv, c.d, c.group, splits, c.bt_stride, c.page, c.pool, float(scale or 0.0), wl, wr, mt, _f._stream(), code)
        _lib.check(rc, "FmhaFwdSplitKVInt4")
        rc = lib.FmhaFwdSplitKVCombine(_f._ptr(lse_acc), _f._ptr(o_acc), _f._ptr(o), None, 1 if group_mode else c.batch, sq, hq, c.d, sq, splits,
                                       _f._stream(), _f._ptr(lse), code)
    _lib.check(rc, "FmhaFwdSplitKVCombine")
    return (o, lse) if return_lse else o


def fmha_read_kv_int4(k_cache: torch.Tensor, k_params: torch.Tensor, v_cache: torch.Tensor, v_params: torch.Tensor, seqlen_k: torch.Tensor, *,
                      block_table: Optional[torch.Tensor] = None, cache_batch_idx: Optional[torch.Tensor] = None,
                      cu_seqlens_k: Optional[torch.Tensor] = None, total_k: Optional[int] = None, max_seqlen_k: Optional[int] = None):
    """A 4-bit cache read back as keys and values of the model's dtype (C symbol ``FmhaReadKVInt4``): what a prefill over cached tokens takes.

    With ``cu_seqlens_k`` (int64 ``[b+1]``) and ``total_k`` packed ``[total_k, hkv, d]``, as :func:`fmha_fwd_var_len` takes them; with
    ``max_seqlen_k`` instead ``[b, max_seqlen_k, hkv, d]``.  Rows that are no token of a sequence are zero.  Returns ``(k, v)``."""
    native = _f._native()
    if native and cache_batch_idx is None:
        r = native._call_read_kv_int4(k_cache, k_params, v_cache, v_params, seqlen_k, block_table, cu_seqlens_k, total_k, max_seqlen_k)
        if r is not None:
            return r if r.__class__ is not int else _lib.check(r, "FmhaReadKVInt4")
    if k_params is None:
        raise TypeError("k_params must be a torch.Tensor")
    _f._check_cuda("k_params", k_params)
    code = _f._dtype_code(k_params)
    c = _Cache(k_cache, k_params, v_cache, v_params, seqlen_k, block_table, cache_batch_idx, k_params.dtype, k_params.device, 1)
    packed = cu_seqlens_k is not None
    if packed != (total_k is not None) or packed == (max_seqlen_k is not None):
        raise ValueError("a packed result takes cu_seqlens_k and total_k, the other one max_seqlen_k")
    cu = _f._as_i64("cu_seqlens_k", cu_seqlens_k) if packed else None
    if packed and cu.numel() != c.batch + 1:
        _f._refuse("cu_seqlens_k", cu, f"{c.batch + 1} entries")
    tokens = int(total_k if packed else max_seqlen_k)
    if tokens < 0:
        raise ValueError("the number of tokens must not be negative")
    _same_device(k_params.device, cu_seqlens_k=cu)
    shape = (tokens, c.hkv, c.d) if packed else (c.batch, tokens, c.hkv, c.d)
    k, v = (torch.empty(shape, dtype=k_params.dtype, device=k_params.device) for _ in range(2))
    with _f._on(k_params.device):
        rc = _lib.lib().FmhaReadKVInt4(_f._ptr(k_cache), _f._ptr(k_params), _f._ptr(v_cache), _f._ptr(v_params), _f._ptr(k), _f._ptr(v),
                                       _f._ptr(c.seqlen), _f._ptr(cu), _f._ptr(c.table), _f._ptr(c.index), c.batch, tokens, c.hkv, c.d, c.group,
                                       c.bt_stride, c.page, c.pool, _f._stream(), code)
    _lib.check(rc, "FmhaReadKVInt4")
    return k, v
