"""Gradients of the attention forward, and the forward as a differentiable function.

:func:`fmha_bwd` / :func:`fmha_bwd_var_len` take dO and what the forward took and gave (Q, K, V, O, LSE) and return the
gradients; they are the C symbol ``FmhaBwd`` and involve no autograd.  :func:`fmha_autograd` / :func:`fmha_autograd_var_len`
are ``fmha_fwd`` / ``fmha_fwd_var_len`` as functions that autograd differentiates through.  The reference has no backward
pass; names and arguments follow the forward's.

Every gradient is summed in a fixed order, so that equal calls give equal bits.  P and dS are rounded to the element type
where they enter a product (as P is in the forward); in fp16, dS below 6e-8 is lost, as usual without a loss scale.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import _lib
from . import fmha as _f

__all__ = ["fmha_bwd", "fmha_bwd_var_len", "fmha_autograd", "fmha_autograd_var_len"]


def _same_device(q: torch.Tensor, **tensors: Optional[torch.Tensor]) -> None:
    for n, t in tensors.items():
        if t is not None and t.device != q.device:
            raise ValueError(f"{n} must be on {q.device} like q, got {t.device}")


def _qkv(q, k, v, dims: int, layout: str) -> None:
    for n, t in (("q", q), ("k", k), ("v", v)):
        if t is None:
            raise TypeError(f"{n} must be a torch.Tensor")
        _f._check_cuda(n, t, getattr(q, "dtype", None))
        if t.dim() != dims:
            raise ValueError(f"{n} must be {layout}, got shape {tuple(t.shape)}")


def _shaped(name: str, t: Optional[torch.Tensor], shape, dtype: torch.dtype) -> None:
    _f._check_cuda(name, t, dtype)
    if t is not None and t.shape != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _gradients(dout, q, k, v, o, lse, cu_q, cu_k, batch, sq, sk, max_sq, max_sk, scale, causal, window_size, mask_type, bias,
               alibi_slopes, logits_soft_cap, dlse, return_dbias):
    """The checks that both forms share, the outputs, and the C call."""
    hq, d = q.shape[-2:]
    hkv = k.shape[-2]
    group = cu_q is not None
    if k.shape[-1] != d or v.shape != k.shape:
        raise ValueError(f"inconsistent shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    lse_shape = (hq, sq) if group else (batch, hq, sq)
    _shaped("dout", dout, q.shape, q.dtype)
    _shaped("o", o, q.shape, q.dtype)
    _shaped("lse", lse, lse_shape, torch.float32)
    _shaped("dlse", dlse, lse_shape, torch.float32)
    if lse is None or dout is None or o is None:
        raise ValueError("the backward pass needs dout and the forward's o and lse (return_lse=True)")
    code = _f._dtype_code(q)
    mt, wl, wr = _f._mask(causal, window_size, mask_type)
    bias_buf, bias_enum, bias_rank = _f._bias_args(q, bias, alibi_slopes, 1 if group and bias is not None else batch, hq, sq, sk)
    if return_dbias and bias is None:
        raise ValueError("return_dbias needs a bias tensor")
    _same_device(q, dout=dout, k=k, v=v, o=o, lse=lse, dlse=dlse, bias=bias_buf, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    # (packed: the bias plane has elements that belong to no sequence)
    dbias = (torch.zeros_like if group else torch.empty_like)(bias) if return_dbias else None
    delta = torch.empty_like(lse)
    with _f._on(q.device):
        rc = _lib.lib().FmhaBwd(_f._ptr(dout), _f._ptr(q), _f._ptr(k), _f._ptr(v), _f._ptr(bias_buf), _f._ptr(o), _f._ptr(lse),
                                _f._ptr(dlse), _f._ptr(dq), _f._ptr(dk), _f._ptr(dv), _f._ptr(dbias), _f._ptr(delta), _f._ptr(cu_q),
                                _f._ptr(cu_k), batch, sq, sk, hq, hkv, d, d, max_sq, max_sk, float(scale or 0.0), wl, wr, mt,
                                _f._stream(), code, bias_enum, bias_rank, float(logits_soft_cap))
    _lib.check(rc, "FmhaBwd")
    return (dq, dk, dv, dbias) if return_dbias else (dq, dk, dv)


def fmha_bwd(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor, *,
             scale: Optional[float] = None, causal: bool = False, window_size: Sequence[int] = (-1, -1),
             mask_type: Optional[int] = None, bias: Optional[torch.Tensor] = None, alibi_slopes: Optional[torch.Tensor] = None,
             logits_soft_cap: float = 0.0, dlse: Optional[torch.Tensor] = None, return_dbias: bool = False):
    """Gradients of :func:`fmha_fwd` (C symbol ``FmhaBwd``).

    dout and o ``[b, sq, hq, d]``, q, k, v and the options as the forward had them, lse fp32 ``[b, hq, sq]`` -> ``(dq, dk, dv)``,
    with ``return_dbias`` the bias tensor's gradient as a fourth.  ``dlse``: the gradient of the LSE where it was used too."""
    native = _f._native()
    if native and bias is None and alibi_slopes is None and not return_dbias:
        r = native._call_backward(dout, q, k, v, o, lse, None, None, 0, 0, scale, causal, window_size, mask_type, logits_soft_cap, dlse)
        if r is not None:
            return r if r.__class__ is not int else _lib.check(r, "FmhaBwd")
    _qkv(q, k, v, 4, "[batch, seqlen, heads, hdim]")
    b, sq = q.shape[:2]
    if k.shape[0] != b:
        raise ValueError(f"inconsistent shapes q{tuple(q.shape)} k{tuple(k.shape)} v{tuple(v.shape)}")
    return _gradients(dout, q, k, v, o, lse, None, None, b, sq, k.shape[1], 0, 0, scale, causal, window_size, mask_type, bias,
                      alibi_slopes, logits_soft_cap, dlse, return_dbias)


def fmha_bwd_var_len(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                     cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, max_seqlen_q: int = 0, max_seqlen_k: int = 0, *,
                     scale: Optional[float] = None, causal: bool = False, window_size: Sequence[int] = (-1, -1),
                     mask_type: Optional[int] = None, bias: Optional[torch.Tensor] = None,
                     alibi_slopes: Optional[torch.Tensor] = None, logits_soft_cap: float = 0.0,
                     dlse: Optional[torch.Tensor] = None, return_dbias: bool = False):
    """Gradients of :func:`fmha_fwd_var_len`: packed ``[total, heads, d]`` tensors, lse ``[hq, total_q]``, int64 ``[b+1]`` starts.

    ``max_seqlen_*`` bound the longest sequences (0: the packed totals).  Rows that belong to no sequence get zeros; elements
    of the bias gradient outside the sequences' blocks too."""
    native = _f._native()
    if native and bias is None and alibi_slopes is None and not return_dbias and cu_seqlens_q is not None:
        r = native._call_backward(dout, q, k, v, o, lse, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal, window_size,
                                  mask_type, logits_soft_cap, dlse)
        if r is not None:
            return r if r.__class__ is not int else _lib.check(r, "FmhaBwd")
    _qkv(q, k, v, 3, "packed [total_tokens, heads, hdim]")
    cu_q, cu_k = _f._as_i64("cu_seqlens_q", cu_seqlens_q), _f._as_i64("cu_seqlens_k", cu_seqlens_k)
    if cu_q.numel() != cu_k.numel() or cu_q.numel() < 2:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must both have batch + 1 entries")
    return _gradients(dout, q, k, v, o, lse, cu_q, cu_k, cu_q.numel() - 1, q.shape[0], k.shape[0], int(max_seqlen_q),
                      int(max_seqlen_k), scale, causal, window_size, mask_type, bias, alibi_slopes, logits_soft_cap, dlse, return_dbias)


# A leaf's gradient is accumulated on the stream where its node was made (by the first graph that uses the leaf), for as long as a
# graph holds the node.  Where that is the default stream, a captured backward pass would make it wait for the capture, which
# ends the process.  The node carries a mark, and the captured pass is refused.
_ON_DEFAULT_STREAM = "flashck_b200: made on the default stream"


def _mark_leaves(*tensors: Optional[torch.Tensor]) -> list:
    """The nodes of the leaves among the tensors, marked; they have to be held until the graph holds them."""
    leaves = [t for t in tensors if t is not None and t.is_cuda and t.is_leaf and t.requires_grad]
    nodes = [torch.autograd.graph.get_gradient_edge(t).node for t in leaves]
    native = _f._native()
    for t, n in zip(leaves, nodes):
        if native:
            n.metadata[_ON_DEFAULT_STREAM] = native._accumulates_on_default_stream(t)
        else:  # what made the node cannot be asked: the first call here that meets it is taken for it
            n.metadata.setdefault(_ON_DEFAULT_STREAM, torch.cuda.current_stream(t.device).cuda_stream == 0)
    return nodes


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias, alibi_slopes, cu_q, cu_k, max_sq, max_sk, options):
        if cu_q is None:
            o, lse = _f.fmha_fwd(q, k, v, return_lse=True, bias=bias, alibi_slopes=alibi_slopes, **options)
        else:
            cu_q, cu_k = _f._as_i64("cu_seqlens_q", cu_q), _f._as_i64("cu_seqlens_k", cu_k)
            o, lse = _f.fmha_fwd_var_len(q, k, v, cu_q, cu_k, max_sq or q.shape[0], max_sk, return_lse=True, bias=bias,
                                         alibi_slopes=alibi_slopes, **options)
            with _f._on(q.device):
                _lib.check(_lib.lib().FmhaZeroOutside(_f._ptr(o), _f._ptr(lse), _f._ptr(cu_q), cu_q.numel() - 1, *o.shape, _f._stream(),
                                                      _f._dtype_code(o)), "FmhaZeroOutside")
        ctx.save_for_backward(q, k, v, bias, alibi_slopes, cu_q, cu_k, o, lse)
        ctx.max_sq, ctx.max_sk, ctx.options = max_sq, max_sk, options
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v, bias, alibi_slopes, cu_q, cu_k, o, lse = ctx.saved_tensors
        if dout is None and dlse is None:
            return (None,) * 10
        if torch.cuda.is_current_stream_capturing() and any(n.metadata.get(_ON_DEFAULT_STREAM) for n, _ in ctx.next_functions if n is not None):
            raise RuntimeError("this backward pass is being captured, but an input's gradient belongs to a graph that was recorded on the default "
                               "stream and still lives: release that graph's outputs, or record it on a side stream")
        dout = torch.zeros_like(o) if dout is None else dout.contiguous()
        if dout.data_ptr() % 16:
            dout = dout.clone()
        more = dict(bias=bias, alibi_slopes=alibi_slopes, dlse=None if dlse is None else dlse.contiguous(),
                    return_dbias=bias is not None and ctx.needs_input_grad[3], **ctx.options)
        g = (fmha_bwd(dout, q, k, v, o, lse, **more) if cu_q is None else
             fmha_bwd_var_len(dout, q, k, v, o, lse, cu_q, cu_k, ctx.max_sq, ctx.max_sk, **more))
        wanted = [x if need else None for x, need in zip(g, ctx.needs_input_grad)]
        return tuple(wanted + [None] * (10 - len(wanted)))


def _differentiable(q, k, v, bias, alibi_slopes, cu_q, cu_k, max_sq, max_sk, return_lse, options):
    if alibi_slopes is not None and alibi_slopes.requires_grad:
        raise ValueError("alibi_slopes are constants: their gradient is not computed")
    held = _mark_leaves(q, k, v, bias) if torch.is_grad_enabled() else None  # noqa: F841
    o, lse = _Attention.apply(q, k, v, bias, alibi_slopes, cu_q, cu_k, max_sq, max_sk, options)
    return (o, lse) if return_lse else o


def fmha_autograd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None, causal: bool = False,
                  window_size: Sequence[int] = (-1, -1), mask_type: Optional[int] = None, return_lse: bool = False,
                  bias: Optional[torch.Tensor] = None, alibi_slopes: Optional[torch.Tensor] = None, logits_soft_cap: float = 0.0):
    """:func:`fmha_fwd` as a function that autograd differentiates: same arguments and results, with gradients for q, k, v and
    the bias tensor, through the output and (``return_lse``) the LSE.

    A backward pass in a CUDA graph: capture the whole step after a warm-up on a side stream, or call :func:`fmha_bwd` in the
    capture.  A captured pass is refused while a graph of the same leaves that was recorded on the default stream lives."""
    return _differentiable(q, k, v, bias, alibi_slopes, None, None, 0, 0, return_lse,
                           dict(scale=scale, causal=causal, window_size=tuple(window_size), mask_type=mask_type, logits_soft_cap=logits_soft_cap))


def fmha_autograd_var_len(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                          max_seqlen_q: int, max_seqlen_k: int = 0, *, scale: Optional[float] = None, causal: bool = False,
                          window_size: Sequence[int] = (-1, -1), mask_type: Optional[int] = None, return_lse: bool = False,
                          bias: Optional[torch.Tensor] = None, alibi_slopes: Optional[torch.Tensor] = None,
                          logits_soft_cap: float = 0.0):
    """:func:`fmha_fwd_var_len` as a function that autograd differentiates (see :func:`fmha_autograd`).  Rows of the output
    and entries of the LSE that belong to no sequence are zero."""
    return _differentiable(q, k, v, bias, alibi_slopes, cu_seqlens_q, cu_seqlens_k, int(max_seqlen_q), int(max_seqlen_k), return_lse,
                           dict(scale=scale, causal=causal, window_size=tuple(window_size), mask_type=mask_type, logits_soft_cap=logits_soft_cap))
