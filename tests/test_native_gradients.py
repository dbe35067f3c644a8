"""The compiled backward and shared-prefix calls against the Python of ops: the same bits, and what they cannot check is left to it."""
import pytest
import torch

from flashck_b200 import ops
from flashck_b200.ops import fmha


def _t(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", dtype=dtype)


def _both(monkeypatch, call):
    """(results through the binding and through Python, whether the binding took the call)"""
    native, taken = fmha._native(), []
    assert native, "the binding has not been built"

    class Spy:
        def __getattr__(self, name):
            def f(*a):
                r = getattr(native, name)(*a)
                if name in ("_call_backward", "_call_shared_prefix"):
                    taken.append(r is not None)
                return r
            return f

    out = []
    for binding in (Spy(), False):
        with monkeypatch.context() as m:
            m.setattr(fmha, "_NATIVE", binding)
            try:
                r = call()
                out.append(r if isinstance(r, tuple) else (r,))
            except (RuntimeError, ValueError, TypeError) as e:
                out.append((type(e), str(e)))
    return out, taken


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) if isinstance(x, torch.Tensor) else x == y for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("kw,native", [
    ({}, True), ({"causal": True}, True), ({"window_size": (20, 3)}, True), ({"scale": 0.5, "logits_soft_cap": 10.0}, True),
    ({"scale": 1}, False), ({"window_size": [20, 3]}, False), ({"mask_type": 7}, False), ({"logits_soft_cap": -1.0}, True),
])
@pytest.mark.parametrize("packed", [False, True])
def test_backward(monkeypatch, kw, native, packed):
    q, k, v, dout = _t(2, 70, 4, 64), _t(2, 90, 2, 64), _t(2, 90, 2, 64), _t(2, 70, 4, 64)
    o, lse = ops.fmha_fwd(q, k, v, return_lse=True)
    if packed:
        cu_q, cu_k = torch.tensor([0, 30, 140], device="cuda"), torch.tensor([0, 80, 180], device="cuda")
        q, k, v, dout = (x.flatten(0, 1) for x in (q, k, v, dout))
        o, lse = ops.fmha_fwd_var_len(q, k, v, cu_q, cu_k, 110, 100, return_lse=True)
        call = lambda: ops.fmha_bwd_var_len(dout, q, k, v, o, lse, cu_q, cu_k, 110, 100, **kw)  # noqa: E731
    else:
        call = lambda: ops.fmha_bwd(dout, q, k, v, o, lse, dlse=torch.ones_like(lse), **kw)  # noqa: E731
    (a, b), taken = _both(monkeypatch, call)
    assert _same(a, b) and taken == [native]


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["lse", "dtype", "strided", "heads", "o", "hdim"])
def test_backward_refuses_alike(monkeypatch, form):
    q, k, lse = _t(1, 8, 4, 64), _t(1, 8, 2, 64), torch.zeros(1, 4, 8, device="cuda")
    o, dout = torch.zeros_like(q), torch.zeros_like(q)
    if form == "lse":
        lse = lse[..., :7].contiguous()
    elif form == "dtype":
        o = o.half()
    elif form == "strided":
        dout = dout.transpose(1, 2)
    elif form == "heads":
        k = _t(1, 8, 3, 64)
    elif form == "o":
        o = o[:, :7].contiguous()
    else:
        q, k, o, dout = (x[..., :32].contiguous() for x in (q, k, o, dout))
    (a, b), _ = _both(monkeypatch, lambda: ops.fmha_bwd(dout, q, k, k, o, lse))
    assert _same(a, b) and isinstance(a[0], type) and issubclass(a[0], Exception)


@pytest.mark.gpu
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("slice_of", [False, True])
def test_shared_prefix(monkeypatch, paged, packed, slice_of):
    b = 3
    q = _t(5, 4, 64) if packed else _t(b, 1, 4, 64)
    cu = torch.tensor([0, 1, 3, 5], device="cuda") if packed else None
    sl = torch.tensor([3, 20, 17], dtype=torch.int32, device="cuda")
    if paged:
        k, v = _t(20, 16, 2, 64), _t(20, 16, 2, 64)
        ids = torch.randperm(20, device="cuda").to(torch.int32)
        table = ids[6:18].view(3, 4) if not slice_of else ids[3:18].view(3, 5)[:, 1:]
        call = lambda **kw: ops.fmha_fwd_shared_prefix(q, k, v, k, v, prefix_len=40, prefix_table=ids[:3].contiguous(), seqlen_k=sl,  # noqa: E731
                                                       block_table=table, cu_seqlens_q=cu, max_seqlen_q=2, causal=True, **kw)
    else:
        k, v, kp, vp = _t(b, 24, 2, 64), _t(b, 24, 2, 64), _t(50, 2, 64), _t(50, 2, 64)
        call = lambda **kw: ops.fmha_fwd_shared_prefix(q, kp, vp, k, v, prefix_len=41 if slice_of else None, seqlen_k=sl, cu_seqlens_q=cu,  # noqa: E731
                                                       causal=True, **kw)
    for kw in ({}, {"return_lse": True}, {"scale": 0.3}):
        (a, b_), taken = _both(monkeypatch, lambda: call(**kw))
        assert _same(a, b_) and taken == [not (paged and slice_of)]


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["prefix_len", "table", "seqlen", "cache", "page", "heads"])
def test_shared_prefix_refuses_alike(monkeypatch, form):
    q, k = _t(2, 1, 4, 64), _t(8, 16, 2, 64)
    kw = dict(prefix_len=40, prefix_table=torch.zeros(3, dtype=torch.int32, device="cuda"), seqlen_k=torch.ones(2, dtype=torch.int32, device="cuda"),
              block_table=torch.zeros(2, 2, dtype=torch.int32, device="cuda"))
    cache = k
    if form == "prefix_len":
        kw["prefix_len"] = None
    elif form == "table":
        kw["prefix_len"] = 49
    elif form == "seqlen":
        kw["seqlen_k"] = kw["seqlen_k"][:1].contiguous()
    elif form == "cache":
        kw["block_table"] = None
    elif form == "page":
        k = cache = _t(8, 8, 2, 64)
        kw["prefix_len"] = 24
    else:
        cache = _t(8, 16, 1, 64)
    (a, b), _ = _both(monkeypatch, lambda: ops.fmha_fwd_shared_prefix(q, k, k, cache, cache, **kw))
    assert _same(a, b) and isinstance(a[0], type) and issubclass(a[0], Exception)
