"""cache_batch_idx together with a block table: it picks the table's rows, and one that is not there has no pages."""
import pytest
import torch

from flashck_b200 import _lib, ops
from flashck_b200.utils.enums import RopeEnum

pytestmark = pytest.mark.gpu
OVERFLOW = 0x40000000  # FLASHCK_STATUS_APPEND_OVERFLOW


def _cache():
    g = torch.Generator("cuda").manual_seed(0)
    parts = [x for _ in range(2) for x in ops.int4_cache(20, 16, 2, 64, group=32)]
    table = torch.randperm(20, generator=g, device="cuda").to(torch.int32).view(5, 4)
    k, v = (torch.randn(5, 60, 2, 64, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    ops.fmha_fwd_append_kv_int4(None, *parts, k, v, torch.zeros(5, dtype=torch.int32, device="cuda"), rope=RopeEnum.NONE, block_table=table)
    return parts, table, torch.randn(3, 1, 4, 64, generator=g, device="cuda").to(torch.bfloat16)


def _all(parts, q, lens, **kw):
    return (*ops.fmha_fwd_splitkv_int4(q, *parts, seqlen_k=lens, return_lse=True, **kw), *ops.fmha_read_kv_int4(*parts, lens, max_seqlen_k=60, **kw))


@pytest.mark.parametrize("index", [[3, 0, 4], [2, 2, 1]])
def test_rows_are_picked(index):
    parts, table, q = _cache()
    index, lens = torch.tensor(index, device="cuda"), torch.tensor([60, 33, 1], dtype=torch.int32, device="cuda")
    got = _all(parts, q, lens, block_table=table, cache_batch_idx=index)
    assert all(torch.equal(a, b) for a, b in zip(got, _all(parts, q, lens, block_table=table[index].contiguous())))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("bad", [5, -1, 2 ** 40, -2 ** 40])
def test_rows_that_are_not_there_have_no_pages(bad):
    parts, table, q = _cache()
    index, lens = torch.tensor([3, bad, 4], device="cuda"), torch.tensor([60, 33, 1], dtype=torch.int32, device="cuda")
    o, lse, k, v = _all(parts, q, lens, block_table=table, cache_batch_idx=index)
    none = table[[3, 0, 4]]
    none[1] = -1
    assert all(torch.equal(a, b) for a, b in zip((o, lse, k, v), _all(parts, q, lens, block_table=none)))
    assert (k[1] == 0).all() and (v[1] == 0).all() and (o[1] == 0).all()
    before, new = [x.clone() for x in parts], torch.ones(3, 1, 2, 64, device="cuda", dtype=torch.bfloat16)
    ops.fmha_fwd_append_kv_int4(None, *parts, new, new, lens - 1, rope=RopeEnum.NONE, block_table=table, cache_batch_idx=index)
    assert _lib.device_status() & OVERFLOW
    ops.fmha_fwd_append_kv_int4(None, *before, new, new, lens - 1, rope=RopeEnum.NONE, block_table=none)
    assert _lib.device_status() & OVERFLOW
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(parts, before))


def test_a_table_without_rows():
    parts, table, q = _cache()
    o, lse, k, _ = _all(parts, q, torch.tensor([60, 33, 1], dtype=torch.int32, device="cuda"), block_table=table[:0].contiguous(),
                        cache_batch_idx=torch.zeros(3, dtype=torch.int64, device="cuda"))
    assert (o == 0).all() and (k == 0).all() and torch.isfinite(lse).all()
    assert _lib.device_status() == 0
