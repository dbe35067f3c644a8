"""What decode over a shared prefix refuses, without a GPU: the C symbol's checks come before any CUDA call."""
import re

import pytest
import torch

from flashck_b200 import _lib, ops
from flashck_b200.nn import FlashAttention
from flashck_b200.utils import get_operation_function

P = 4096  # an address that is never read


def _call(**kw):
    a = dict(q=P, kp=P, vp=P, k=P, v=P, o=P, lse=0, ws=P, ptab=P, tab=P, lens=P, cu=0, prefix=100, p_page=16, p_pages=10, page=16, pages=10,
             stride=4, cap=0, batch=2, sq=1, max_q=0, hq=4, hkv=2, d=64, dv=64, scale=0.0, causal=1, stream=0, dtype=4)
    a.update(kw)
    return _lib.lib().FmhaFwdSharedPrefix(*a.values()), _lib.last_error()


@pytest.mark.parametrize("change,code,said", [
    (dict(dtype=7), 2, "dtype"), (dict(hq=3), 1, "multiple"), (dict(d=96, dv=96), 2, "hdim"), (dict(dv=128), 2, "hdim"),
    (dict(prefix=-1), 1, "negative"), (dict(cap=-1), 1, "negative"), (dict(q=0), 1, "null"), (dict(lens=0), 1, "null"), (dict(ws=0), 1, "null"),
    (dict(kp=0), 1, "null"), (dict(q=P + 8), 1, "16-byte"), (dict(ws=P + 4), 1, "16-byte"), (dict(p_page=8), 2, "multiple of 16"),
    (dict(page=24), 2, "multiple of 16"), (dict(pages=0), 1, "pages"), (dict(p_pages=1 << 30), 1, "pages"), (dict(stride=-1), 1, "stride"),
    (dict(tab=0, page=0, cap=1 << 30, batch=4), 2, "2\\^31"), (dict(causal=2), 1, "causal"), (dict(prefix=1 << 31), 2, "prefix_len"),
])
def test_c_symbol_refuses(change, code, said):
    rc, text = _call(**change)
    assert rc == code and re.search(said, text), text


def test_nothing_to_do_is_no_error():
    assert _call(batch=0)[0] == 0 and _call(sq=0)[0] == 0


def test_workspace_sizes():
    f = _lib.lib().FlashckSharedPrefixWorkspace
    assert f(100, 16, 16, 2, 1, 0, 4, 3, 64, 0, 4) == -1 and f(-1, 16, 16, 2, 1, 0, 4, 2, 64, 0, 4) == -1
    assert f(0, 16, 16, 2, 1, 0, 4, 2, 64, 0, 4) > 0
    assert f(5000, 16, 16, 2, 1, 0, 4, 2, 64, 0, 4) > f(0, 16, 16, 2, 1, 0, 4, 2, 64, 0, 4)


def test_functions_refuse_before_launch():
    q, k = torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16), torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.fmha_fwd_shared_prefix(q, k[0], k[0], k, k, seqlen_k=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError):
        ops.fmha_fwd_shared_prefix(None, k[0], k[0], k, k, seqlen_k=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="window"):
        FlashAttention(4, 64, 2, causal=True, window_size=(5, 0)).forward_shared_prefix(q, k[0], k[0], k, k, None)


def test_registered():
    assert get_operation_function("fmha", "forward_shared_prefix") is ops.fmha_fwd_shared_prefix
