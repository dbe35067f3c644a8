"""More packed sequences than the schedule by cost orders, with and without their longest one stated."""
import pytest
import torch

from attention_reference import assert_within, forward, gradients, half_step
from flashck_b200 import _lib, ops

pytestmark = pytest.mark.gpu
CAUSAL = (2, -1, 0)


def _packed(lens, hq, hkv, d, dtype=torch.bfloat16):
    total = sum(lens)
    q, dout = (torch.randn(total, hq, d, device="cuda").to(dtype) for _ in range(2))
    k, v = (torch.randn(total, hkv, d, device="cuda").to(dtype) for _ in range(2))
    cu = torch.tensor([0] + lens).cumsum(0).cuda()
    o, lse = ops.fmha_fwd_var_len(q, k, v, cu, cu, max(lens), max(lens), causal=True, return_lse=True)
    return (dout, q, k, v, o, lse), cu


def _blocks(call):
    """Blocks of every kernel that the call launches, from the graph that it is captured into."""
    from cuda.bindings import driver
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        held = call()
    raw = driver.CUgraph(graph.raw_cuda_graph())
    err, _, n = driver.cuGraphGetNodes(raw)
    err, nodes, n = driver.cuGraphGetNodes(raw, n)
    assert int(err) == 0
    grids = []
    for node in nodes[:n]:
        err, kind = driver.cuGraphNodeGetType(node)
        if kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, params = driver.cuGraphKernelNodeGetParams(node)
            assert int(err) == 0
            grids.append(params.gridDimX * params.gridDimY * params.gridDimZ)
    del held
    return grids


@pytest.mark.parametrize("longest", [False, True])
@pytest.mark.parametrize("n", [200, 257, 3000])
def test_the_grid_does_not_grow_with_the_sequences(n, longest, device_ok):
    """Tiles of the longest sequence times sequences would be millions of blocks where no length is stated."""
    lens = [i * 7 % 41 for i in range(n)]
    args, cu = _packed(lens, 4, 2, 64)
    stated = (max(lens),) * 2 if longest else (0, 0)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    grids = _blocks(lambda: ops.fmha_bwd_var_len(*args, cu, cu, *stated, causal=True))
    assert len(grids) == 2 and max(grids) <= sms, grids


@pytest.mark.parametrize("lens,hq,hkv,d", [
    ([i * 7 % 41 for i in range(3000)], 4, 2, 64),
    ([0] * 300 + [i * 37 % 300 for i in range(300)] + [0] * 300, 6, 2, 128),
    ([1000] + [1] * 400 + [513], 8, 8, 128),
    ([128] * 257, 2, 1, 64),
])
def test_lengths_that_are_not_stated(lens, hq, hkv, d, device_ok):
    args, cu = _packed(lens, hq, hkv, d)
    got = ops.fmha_bwd_var_len(*args, cu, cu, max(lens), max(lens), causal=True)
    assert _lib.get_instance_param(0, "last_bwd_instance") == 1
    for a, b in zip(got, ops.fmha_bwd_var_len(*args, cu, cu, causal=True)):
        assert torch.equal(a, b)
    assert _lib.get_instance_param(0, "last_bwd_instance") == 1
    at = cu.tolist()
    for i, n in enumerate(lens):
        if n and (i % 40 == 0 or n > 200 or i + 1 == len(lens)):
            rows = slice(at[i], at[i + 1])
            part = [t[None, rows] for t in args[:5]] + [args[5][None, :, rows]]
            want, bound = gradients(*part, d ** -0.5, CAUSAL)
            for name, x, w, e in zip(("dq", "dk", "dv"), got, want, bound):
                assert_within(f"{name} of sequence {i}", x[rows], w[0], e[0])


def test_a_dense_batch_of_many_sequences(device_ok):
    q, k, v, dout = (torch.randn(300, 40, h, 64, device="cuda").bfloat16() for h in (4, 2, 2, 4))
    o, lse = forward(q, k, v, 0.125, CAUSAL)
    args = (dout, q, k, v, o.bfloat16(), lse.float())
    want, bound = gradients(*args, 0.125, CAUSAL)
    for name, x, w, e in zip(("dq", "dk", "dv"), ops.fmha_bwd(*args, causal=True), want, bound):
        assert_within(name, x, w, e)


def _milliseconds(call):
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return sorted(times)[3]


@pytest.mark.parametrize("heads,planes,d", [(2, 1, 64), (2, 2, 128)])
def test_bias_gradient_of_many_sequences(heads, planes, d, device_ok):
    """The blocks of 500 sequences in one plane, with and without the longest one stated: the same bits, in about the same time
    (tiles of the whole plane, sequence by sequence, are some four million here)."""
    lens = [i * 7 % 41 for i in range(500)]
    total, cu = sum(lens), torch.tensor([0] + lens).cumsum(0).cuda()
    q, k, v, dout = (torch.randn(total, heads, d, device="cuda").bfloat16() for _ in range(4))
    bias = torch.randn(1, planes, total, total, device="cuda").bfloat16()
    o, lse = ops.fmha_fwd_var_len(q, k, v, cu, cu, max(lens), max(lens), return_lse=True, bias=bias)
    call = lambda *longest: ops.fmha_bwd_var_len(dout, q, k, v, o, lse, cu, cu, *longest, bias=bias, return_dbias=True)  # noqa: E731
    got = call()
    assert all(torch.equal(a, b) for a, b in zip(got, call(max(lens), max(lens))))
    at, outside = cu.tolist(), torch.ones_like(bias, dtype=torch.bool)
    for i, n in enumerate(lens):
        block = (slice(None), slice(None), slice(at[i], at[i + 1]), slice(at[i], at[i + 1]))
        outside[block] = False
        if n and i % 25 == 0:
            rows = block[2]
            part = [t[None, rows] for t in (dout, q, k, v, o)] + [lse[None, :, rows]]
            want, bound = gradients(*part, d ** -0.5, (0, -1, -1), bias=bias[block])
            w, e = (t.sum(1, keepdim=True) if planes == 1 else t for t in (want[3], bound[3]))
            assert_within(f"dbias of sequence {i}", got[3][block], w, e + half_step(bias.dtype) * w.abs() + 2.0 ** -25)
    assert not got[3][outside].any()
    assert _milliseconds(call) <= 2 * _milliseconds(lambda: call(max(lens), max(lens)))
