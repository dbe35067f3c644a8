"""A block table without columns has no address: it must not be taken for a contiguous cache."""
import pytest
import torch

from flashck_b200 import ops
from flashck_b200.ops import fmha
from flashck_b200.utils.enums import RopeEnum

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("python", [False, True], ids=["binding", "python"])
def test_refused(monkeypatch, python):
    if python:
        monkeypatch.setattr(fmha, "_NATIVE", False)
    parts = [x for _ in range(2) for x in ops.int4_cache(3, 16, 2, 64, group=32)]
    before = [x.clone() for x in parts]
    x = torch.ones(2, 1, 2, 64, device="cuda", dtype=torch.bfloat16)
    lens, table = torch.ones(2, dtype=torch.int32, device="cuda"), torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    for call in (lambda: ops.fmha_fwd_append_kv_int4(None, *parts, x, x, lens, rope=RopeEnum.NONE, block_table=table),
                 lambda: ops.fmha_fwd_splitkv_int4(x, *parts, seqlen_k=lens, block_table=table),
                 lambda: ops.fmha_read_kv_int4(*parts, lens, block_table=table, max_seqlen_k=1)):
        with pytest.raises(ValueError, match="block_table"):
            call()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(parts, before))
