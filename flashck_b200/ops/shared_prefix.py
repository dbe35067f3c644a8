"""Decode for a batch whose sequences share a long prefix: a system prompt, a document, the prompt of a group of samples.

:func:`fmha_fwd_splitkv` over a block table whose first pages are the same for every sequence gives the same result, and reads
those pages once per sequence.  Here they are read once per 128 query rows of a kv head (C symbol ``FmhaFwdSharedPrefix``)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from . import fmha as _f
from .gradients import _same_device

__all__ = ["fmha_fwd_shared_prefix"]


def fmha_fwd_shared_prefix(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                           seqlen_k: torch.Tensor, prefix_len: Optional[int] = None, prefix_table: Optional[torch.Tensor] = None,
                           block_table: Optional[torch.Tensor] = None, cu_seqlens_q: Optional[torch.Tensor] = None, max_seqlen_q: int = 0,
                           scale: Optional[float] = None, causal: bool = False, return_lse: bool = False):
    """Attention of a few new tokens per sequence over a shared prefix and each sequence's own keys.

    q ``[b, sq, hq, d]``, or packed ``[total_q, hq, d]`` with ``cu_seqlens_q``.  The prefix: ``k_prefix/v_prefix`` ``[n, hkv, d]``, or
    pools ``[pages, page, hkv, d]`` with ``prefix_table`` int32, its pages in order; ``prefix_len`` tokens of it count (with a table it
    has to be given, and may end inside a page).  The own caches, as in :func:`fmha_fwd_splitkv`: contiguous
    ``[b, capacity, hkv, d]``, or pools with ``block_table`` int32 ``[b, pages_per_seq]`` (a slice of columns of a longer table will
    do); ``seqlen_k`` int32 ``[b]`` counts own keys, the new tokens among them, and may be 0.  ``causal``: query i of a sequence
    sees the whole prefix and its own keys up to ``seqlen_k - sq + i``.

    Returns o like q (and LSE ``[b, hq, sq]`` / ``[hq, total_q]``); packed rows that belong to no sequence are not written."""
    native = _f._native()
    if native:
        r = native._call_shared_prefix(q, k_prefix, v_prefix, k_cache, v_cache, seqlen_k, prefix_len, prefix_table, block_table, cu_seqlens_q,
                                       max_seqlen_q, scale, causal, return_lse)
        if r is not None:
            return r if r.__class__ is not int else _lib.check(r, "FmhaFwdSharedPrefix")
    for n, t in (("q", q), ("k_prefix", k_prefix), ("v_prefix", v_prefix), ("k_cache", k_cache), ("v_cache", v_cache), ("seqlen_k", seqlen_k)):
        if t is None:
            raise TypeError(f"{n} must be a torch.Tensor")
        _f._check_cuda(n, t, q.dtype if n not in ("q", "seqlen_k") else None)
    code = _f._dtype_code(q)
    sl = _f._as_i32("seqlen_k", seqlen_k)
    batch, group = sl.numel(), cu_seqlens_q is not None
    cu_q = _f._as_i64("cu_seqlens_q", cu_seqlens_q) if group else None
    if q.dim() != (3 if group else 4):
        raise ValueError(f"q must be [b, sq, hq, d], or [total_q, hq, d] with cu_seqlens_q, got shape {tuple(q.shape)}")
    if group and cu_q.numel() != batch + 1:
        _f._refuse("cu_seqlens_q", cu_q, f"{batch + 1} entries")
    if not group and q.shape[0] != batch:
        _f._refuse("seqlen_k", sl, f"{q.shape[0]} entries")
    sq, hq, d = q.shape[-3:]
    hkv = k_cache.shape[-2] if k_cache.dim() == 4 else 0
    # the prefix
    table = prefix_table is not None
    if k_prefix.dim() != (4 if table else 3) or k_prefix.shape[-2:] != (hkv, d) or v_prefix.shape != k_prefix.shape:
        raise ValueError(f"the prefix must be {'pools [pages, page' if table else '[n'}, {hkv}, {d}], got k{tuple(k_prefix.shape)} v{tuple(v_prefix.shape)}")
    if table:
        if prefix_len is None:
            raise ValueError("a paged prefix needs prefix_len")
        prefix_table = _f._as_i32("prefix_table", prefix_table)
        page = k_prefix.shape[1]
        if prefix_table.dim() != 1 or prefix_table.numel() * page < prefix_len:
            _f._refuse("prefix_table", prefix_table, f"the {-(-prefix_len // max(page, 1))} pages of the prefix")
    elif prefix_len is not None and prefix_len > k_prefix.shape[0]:
        _f._refuse("k_prefix", k_prefix, f"{prefix_len} tokens")
    prefix_len = k_prefix.shape[0] if prefix_len is None else int(prefix_len)
    if prefix_len < 0:
        raise ValueError("prefix_len must not be negative")
    # the own caches
    if k_cache.dim() != 4 or k_cache.shape[-1] != d or v_cache.shape != k_cache.shape:
        raise ValueError(f"inconsistent shapes q{tuple(q.shape)} k{tuple(k_cache.shape)} v{tuple(v_cache.shape)}")
    stride = 0
    if block_table is not None:
        if not block_table.is_cuda:
            raise ValueError("block_table must be a CUDA tensor")
        if block_table.dim() != 2 or block_table.shape[0] != batch:
            _f._refuse("block_table", block_table, f"a row for each of the {batch} sequences")
        if block_table.dtype != torch.int32:
            block_table = block_table.to(torch.int32)
        if block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("the entries of a row of block_table must be contiguous")
        stride = block_table.stride(0) if batch > 1 else block_table.shape[1]
        if stride < block_table.shape[1]:
            raise ValueError("the rows of block_table must not overlap")
    elif k_cache.shape[0] != batch:
        _f._refuse("k_cache", k_cache, f"a row for each of the {batch} sequences")
    _same_device(q, k_prefix=k_prefix, v_prefix=v_prefix, k_cache=k_cache, v_cache=v_cache, seqlen_k=sl, prefix_table=prefix_table,
                 block_table=block_table, cu_seqlens_q=cu_q)
    o = torch.empty_like(q)
    lse = torch.empty((hq, sq) if group else (batch, hq, sq), dtype=torch.float32, device=q.device) if return_lse else None
    lib, max_sq = _lib.lib(), int(max_seqlen_q)
    p_page = k_prefix.shape[1] if table else 0
    page = k_cache.shape[1] if block_table is not None else 0
    with _f._on(q.device):
        need = lib.FlashckSharedPrefixWorkspace(prefix_len, p_page, page, batch, sq, max_sq, hq, hkv, d, int(group), code) if hkv else 16
        if need < 0:
            _lib.check(1, "FmhaFwdSharedPrefix")
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
        rc = lib.FmhaFwdSharedPrefix(_f._ptr(q), _f._ptr(k_prefix), _f._ptr(v_prefix), _f._ptr(k_cache), _f._ptr(v_cache), _f._ptr(o),
                                     _f._ptr(lse), _f._ptr(workspace), _f._ptr(prefix_table), _f._ptr(block_table), _f._ptr(sl),
                                     _f._ptr(cu_q), prefix_len, p_page, k_prefix.shape[0], page, k_cache.shape[0], stride,
                                     0 if page else k_cache.shape[1], batch, sq, max_sq, hq, hkv, d, d, float(scale or 0.0), int(causal),
                                     _f._stream(), code)
    _lib.check(rc, "FmhaFwdSharedPrefix")
    return (o, lse) if return_lse else o
