"""What the 4-bit cache's functions and the rotation refuse, without a GPU: the C symbols' checks come before any CUDA call."""
import re

import pytest
import torch

from flashck_b200 import _lib, ops
from flashck_b200.ops import rotary
from flashck_b200.utils import get_operation_function

P = 4096  # an address that is never read


def _said(rc):
    return rc, _lib.last_error()


def _append(**kw):
    a = dict(q=P, q_out=P, kc=P, kp=P, knew=P, vc=P, vp=P, vnew=P, kh=0, vh=0, lens=P, cu_q=0, cu_n=0, pos=0, cos=P, sin=P, pair=None, tab=P, idx=0,
             batch=2, sq=1, n=1, hq=4, hkv=2, d=64, group=32, axes=1, width=64, rows=10, rope=2, stride=4, page=16, pool=8, stream=0, dtype=4)
    a.update(kw)
    return _said(_lib.lib().FmhaFwdAppendKVInt4(*a.values()))


def _attend(**kw):
    a = dict(q=P, kc=P, kp=P, vc=P, vp=P, lse=P, acc=P, cu=0, lens=P, tab=P, idx=0, batch=2, sq=1, max_q=0, hq=4, hkv=2, d=64, group=32, splits=2,
             stride=4, page=16, pool=8, scale=0.0, left=-1, right=-1, mask=0, stream=0, dtype=4)
    a.update(kw)
    return _said(_lib.lib().FmhaFwdSplitKVInt4(*a.values()))


def _read(**kw):
    a = dict(kc=P, kp=P, vc=P, vp=P, k=P, v=P, lens=P, cu=0, tab=P, idx=0, batch=2, tokens=5, hkv=2, d=64, group=32, stride=4, page=16, pool=8,
             stream=0, dtype=4)
    a.update(kw)
    return _said(_lib.lib().FmhaReadKVInt4(*a.values()))


def _rotary(**kw):
    a = dict(q=P, q_out=P, k=P, k_out=P, pos=P, cos=P, sin=P, pair=None, axes=1, tokens=5, hq=4, hkv=2, d=64, width=64, rows=10, rope=2, inverse=0,
             stream=0, dtype=4)
    a.update(kw)
    return _said(_lib.lib().FmhaRotary(*a.values()))


_CACHE = [(dict(dtype=7), 2, "dtype"), (dict(d=96), 2, "hdim"), (dict(d=128, group=16), 2, "groups"), (dict(group=48), 1, "divide"),
          (dict(kc=0), 1, "null"), (dict(vp=0), 1, "null"), (dict(lens=0), 1, "null"), (dict(kc=P + 4), 1, "16-byte"), (dict(vp=P + 8), 1, "16-byte"),
          (dict(batch=0), 1, "batch"), (dict(page=0), 1, "page"), (dict(pool=1 << 31), 1, "pool"), (dict(stride=-1), 1, "table")]


@pytest.mark.parametrize("call", [_append, _attend, _read])
@pytest.mark.parametrize("change,code,said", _CACHE)
def test_caches(call, change, code, said):
    rc, text = call(**change)
    assert rc in (1, 2) and (rc == code or change == dict(page=0)) and re.search(said, text), text


@pytest.mark.parametrize("change,code,said", [
    (dict(hq=3), 1, "multiple"), (dict(knew=0), 1, "null"), (dict(q_out=0), 1, "null"), (dict(cu_q=P), 1, "group mode"), (dict(n=-1), 1, "tokens"),
    (dict(rope=3), 1, "rope_type"), (dict(width=66), 1, "rotary_dim"), (dict(width=0), 1, "rotary_dim"), (dict(width=7), 1, "rotary_dim"),
    (dict(cos=0), 1, "tables"), (dict(pos=P, axes=5), 2, "axes"), (dict(pos=P, axes=0), 2, "axes"), (dict(pair=b"\1" * 32), 1, "turns with axis"),
])
def test_append(change, code, said):
    rc, text = _append(**change)
    assert rc == code and re.search(said, text), text


@pytest.mark.parametrize("change,code,said", [
    (dict(hq=3), 1, "multiple"), (dict(q=0), 1, "null"), (dict(lse=0), 1, "null"), (dict(q=P + 8), 1, "16-byte"), (dict(acc=P + 4), 1, "16-byte"),
    (dict(splits=0), 1, "num_splits"), (dict(mask=4), 1, "mask_type"), (dict(sq=0), 1, "rows"), (dict(cu=P), 1, "rows"), (dict(page=24), 2, "multiple of 16"),
    (dict(batch=8193), 2, "8192"), (dict(pool=0), 1, "pool"),
])
def test_attend(change, code, said):
    rc, text = _attend(**change)
    assert rc == code and re.search(said, text), text


@pytest.mark.parametrize("change,code,said", [(dict(tokens=-1), 1, "tokens"), (dict(k=0), 1, "null"), (dict(v=P + 8), 1, "16-byte")])
def test_read(change, code, said):
    rc, text = _read(**change)
    assert rc == code and re.search(said, text), text
    assert _read(tokens=0, k=0, v=0)[0] == 0


@pytest.mark.parametrize("change,code,said", [
    (dict(dtype=1), 2, "dtype"), (dict(d=60), 2, "hdim"), (dict(rope=0), 1, "rope_type"), (dict(rope=3), 1, "rope_type"), (dict(width=80), 1, "rotary_dim"),
    (dict(d=512, width=320), 1, "rotary_dim"), (dict(axes=5), 2, "axes"), (dict(q=0), 1, "null"), (dict(k_out=0), 1, "null"), (dict(pos=0), 1, "null"),
    (dict(cos=0), 1, "tables"), (dict(tokens=-1), 1, "sizes"), (dict(pair=b"\0" * 31 + b"\1"), 1, "turns with axis"), (dict(rows=-1), 1, "rows"),
])
def test_rotary(change, code, said):
    rc, text = _rotary(**change)
    assert rc == code and re.search(said, text), text
    assert _rotary(tokens=0, q=0, q_out=0, pos=0)[0] == 0


def test_functions_refuse_before_launch():
    c = [torch.zeros(2, 16, 2, 32, dtype=torch.uint8), torch.zeros(2, 16, 2, 2, 2, dtype=torch.bfloat16)] * 2
    q, lens, t = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32), torch.zeros(9, 32, dtype=torch.bfloat16)
    for call in (lambda: ops.fmha_fwd_splitkv_int4(q, *c, seqlen_k=lens), lambda: ops.fmha_read_kv_int4(*c, lens, max_seqlen_k=3),
                 lambda: ops.fmha_fwd_append_kv_int4(q, *c, q, q, lens, t, t), lambda: ops.apply_rotary(q, None, lens, t, t),
                 lambda: ops.apply_rotary_autograd(q, None, lens, t, t)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: ops.fmha_fwd_splitkv_int4(None, *c, seqlen_k=lens), lambda: ops.fmha_fwd_append_kv_int4(None, *c, None, None, lens),
                 lambda: ops.fmha_read_kv_int4(c[0], None, *c[2:], lens, max_seqlen_k=3), lambda: ops.apply_rotary(None, None, lens, t, t)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError, match="constant"):
        ops.apply_rotary_autograd(q, None, lens, t.clone().requires_grad_(), t)


def test_caches_are_made():
    codes, params = ops.int4_cache(3, 16, 2, 128, group=64, dtype=torch.float16, device="cpu")
    assert codes.shape == (3, 16, 2, 64) and codes.dtype == torch.uint8 and params.shape == (3, 16, 2, 2, 2) and params.dtype == torch.float16
    assert ops.int4_cache(1, 1, 1, 64, device="cpu")[1].shape == (1, 1, 1, 1, 2)
    for kw in (dict(d=96), dict(d=64, group=128), dict(d=128, group=16)):
        with pytest.raises(ValueError, match="groups"):
            ops.int4_cache(1, 16, 1, device="cpu", **kw)
    with pytest.raises(TypeError):
        ops.int4_cache(1, 16, 1, 64, dtype=torch.float32, device="cpu")


def test_pairs_and_their_axes():
    f = rotary._pair_axes
    assert f(None, False, 32, 1) is None
    assert f((2, 3, 1), False, 6, 3) == bytes([0, 0, 1, 1, 1, 2])
    assert f((3, 2, 1), True, 6, 3) == bytes([0, 1, 2, 0, 1, 0]) and f((0, 2), True, 2, 2) == bytes([1, 1])
    for args in ((None, False, 6, 2), ((2, 3), False, 6, 2), ((2, 3, 1), False, 6, 2), ((-1, 7), False, 6, 2), ((6,) * 5, False, 30, 5)):
        with pytest.raises(ValueError):
            f(*args)


def test_positions_and_tables_fit():
    f = rotary._as_positions
    for bad in (torch.zeros(5), "x", None):
        with pytest.raises(TypeError):
            f(bad, 5)
    with pytest.raises(ValueError, match="CUDA"):
        f(torch.zeros(5, dtype=torch.int32), 5)


def test_registered():
    for name, fn in (("append_kv_int4", ops.fmha_fwd_append_kv_int4), ("forward_splitkv_int4", ops.fmha_fwd_splitkv_int4),
                     ("read_kv_int4", ops.fmha_read_kv_int4), ("rotary", ops.apply_rotary), ("rotary_autograd", ops.apply_rotary_autograd)):
        assert get_operation_function("fmha", name) is fn
