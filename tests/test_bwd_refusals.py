"""What the backward entry points refuse, without a GPU: the C symbol's checks come before any CUDA call."""
import pytest
import torch

from flashck_b200 import _lib, get_available_operations, ops
from flashck_b200.utils import get_operation_function

P = 4096  # an address that is never read: every call below is refused, or has nothing to do


def _call(**kw):
    a = dict(dout=P, q=P, k=P, v=P, bias=0, o=P, lse=P, dlse=0, dq=P, dk=P, dv=P, dbias=0, delta=P, cu_q=0, cu_k=0, batch=1, sq=4, sk=4,
             hq=2, hkv=2, d=64, dvh=64, max_q=0, max_k=0, scale=0.0, left=-1, right=-1, mask=0, stream=0, dtype=4, bias_enum=0, rank=0, cap=0.0)
    a.update(kw)
    return _lib.lib().FmhaBwd(*a.values()), _lib.last_error()


@pytest.mark.parametrize("change,code,said", [
    (dict(dtype=7), 2, "dtype"), (dict(dtype=1), 2, "dtype"), (dict(hq=3), 1, "multiple"), (dict(d=96, dvh=96), 2, "hdim"),
    (dict(dvh=128), 2, "hdim"), (dict(bias_enum=1), 1, "without a bias"), (dict(bias_enum=3, bias=P), 1, "bias_enum"),
    (dict(bias_enum=2, bias=P, rank=2), 1, "rank"), (dict(bias_enum=1, bias=P, rank=2, cu_q=P, cu_k=P), 1, "rank"),
    (dict(dbias=P), 1, "dbias"), (dict(cap=-1.0), 1, "cap"), (dict(sq=-1), 1, "negative"), (dict(max_k=-1), 1, "negative"),
    (dict(mask=4), 1, "mask"), (dict(cu_q=P), 1, "seqstart"), (dict(lse=0), 1, "null"), (dict(delta=0), 1, "null"), (dict(dv=0), 1, "null"),
    (dict(k=P + 8), 1, "16-byte"), (dict(dq=P + 2), 1, "16-byte"), (dict(batch=1 << 20, sq=1 << 12), 2, "2\\^31"),
])
def test_c_symbol_refuses(change, code, said):
    import re
    rc, text = _call(**change)
    assert rc == code and re.search(said, text), text


def test_nothing_to_do_is_no_error():
    assert _call(batch=0)[0] == 0
    assert _call(sq=0, sk=0, dout=0, q=0, k=0, v=0, o=0, lse=0, dq=0, dk=0, dv=0, delta=0)[0] == 0


@pytest.mark.parametrize("change,code,said", [
    (dict(dtype=1), 2, "dtype"), (dict(batch=-1), 1, "negative"), (dict(o=0), 1, "null"), (dict(cu=0), 1, "null"), (dict(o=P + 8), 2, "16-byte"),
    (dict(hq=1, dv=4), 2, "16-byte"), (dict(total=0, o=0), 0, ""),
])
def test_zero_outside_refuses(change, code, said):
    a = dict(o=P, lse=P, cu=P, batch=1, total=4, hq=2, dv=64, stream=0, dtype=4)
    a.update(change)
    assert _lib.lib().FmhaZeroOutside(*a.values()) == code and (code == 0 or said in _lib.last_error())


def test_functions_refuse_before_launch():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    lse = torch.zeros(1, 2, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.fmha_bwd(q, q, q, q, q, lse)
    with pytest.raises(ValueError, match="CUDA"):
        ops.fmha_bwd_var_len(q[0], q[0], q[0], q[0], q[0], lse[0], torch.zeros(2), torch.zeros(2))
    with pytest.raises(TypeError):
        ops.fmha_bwd(q, "q", q, q, q, lse)
    with pytest.raises(TypeError):
        ops.fmha_bwd(None, None, q, q, q, lse)
    with pytest.raises(ValueError, match="slopes"):
        ops.fmha_autograd(q, q, q, alibi_slopes=torch.ones(1, 2, requires_grad=True))


def test_registered():
    for name, fn in (("backward", ops.fmha_bwd), ("backward_var_len", ops.fmha_bwd_var_len), ("autograd", ops.fmha_autograd),
                     ("autograd_var_len", ops.fmha_autograd_var_len)):
        assert get_operation_function("fmha", name) is fn
    assert "fmha" in get_available_operations()
