"""More packed sequences than the schedule by cost orders, with and without their longest one stated."""
import pytest
import torch

from attention_reference import assert_within, forward, gradients
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
