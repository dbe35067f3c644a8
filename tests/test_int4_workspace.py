"""The depth of the workspace of decode over a 4-bit cache where the caller leaves it open: what the kernel's grid can use, and no more."""
import pytest
import torch

from flashck_b200 import ops
from flashck_b200.ops import int4

SIZES = [(b, rows, hkv) for b in (1, 2, 7, 64, 300, 8192) for rows in (1, 4, 8, 9, 16, 17, 64, 2000, 300000) for hkv in (1, 2, 3, 8, 12, 40)]


def _touched(lens, ctas, depth):
    """Most splits that a sequence of `lens` tiles needs when `ctas` pieces are cut for a workspace of `depth` splits."""
    total = sum(lens)
    piece = max(1, -(-total // ctas), -(-max(lens) // (depth - 1)) if depth > 1 else total)
    before, most = 0, 0
    for n in lens:
        if n:
            most = max(most, (before + n - 1) // piece - before // piece + 1)
        before += n
    return most, piece


@pytest.mark.parametrize("batch,rows,hkv", SIZES)
def test_depth_is_what_the_grid_uses(batch, rows, hkv):
    depth, usual = int4._split_depth(batch, rows, hkv), ops.default_num_splits(batch)
    heads = max(n for n in (1, 2, 4, 8) if hkv % n == 0)
    ctas = max(1, 148 // (-(-rows // 16) * (hkv // heads)))
    assert 1 <= depth <= usual
    if depth < usual and batch <= 300:  # not less than the cut for the usual depth takes, which it leaves as it is
        for lens in ([1] * batch, [1000] * batch, [1 + 37 * i % 90 for i in range(batch)], [100000] + [1] * (batch - 1), [0] * (batch - 1) + [777]):
            if depth > 1:
                assert _touched(lens, ctas, depth)[1] == _touched(lens, ctas, usual)[1]
            else:
                assert ctas == 1
            assert _touched(lens, ctas, usual)[0] <= depth


@pytest.mark.parametrize("batch,rows,hkv", SIZES)
def test_the_binding_agrees(batch, rows, hkv):
    from flashck_b200.ops import fmha
    native = fmha._native()
    if not native:
        pytest.skip("no binding")
    assert native._split_depth(batch, rows, hkv) == int4._split_depth(batch, rows, hkv)


def test_many_rows_take_no_splits():
    assert int4._split_depth(1, 8192, 8) == 1 and int4._split_depth(1, 4, 8) == 128 and int4._split_depth(64, 4, 8) == 6


@pytest.mark.gpu
@pytest.mark.parametrize("python", [False, True], ids=["binding", "python"])
def test_a_chunk_of_a_prompt_takes_little_memory(monkeypatch, python):
    from flashck_b200.ops import fmha
    if python:
        monkeypatch.setattr(fmha, "_NATIVE", False)
    parts = [x for _ in range(2) for x in ops.int4_cache(1, 4096, 8, 64)]
    q = torch.randn(1, 2048, 32, 64, device="cuda").to(torch.bfloat16)
    lens = torch.full((1,), 2100, dtype=torch.int32, device="cuda")
    ops.fmha_fwd_splitkv_int4(q[:, :1].contiguous(), *parts, seqlen_k=lens)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    o = ops.fmha_fwd_splitkv_int4(q, *parts, seqlen_k=lens, causal=True)
    assert torch.cuda.max_memory_allocated() - before <= o.numel() * 2 + 2048 * 32 * 65 * 4 + (1 << 21)
    split = ops.fmha_fwd_splitkv_int4(q, *parts, seqlen_k=lens, causal=True, num_splits=9)
    assert torch.equal(o, split)
