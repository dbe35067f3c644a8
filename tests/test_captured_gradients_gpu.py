"""A captured backward pass while other graphs of the same leaves live: what decides is the stream where a leaf's node was made."""
import pytest
import torch

from flashck_b200 import ops
from flashck_b200.ops import fmha

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")]


def _on(stream, call):
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        r = call()
    torch.cuda.current_stream().wait_stream(stream)
    return r


def _attention(q, k, v):
    return ops.fmha_autograd(q, k, v, causal=True)


def _other(q, k, v):
    return [t * 2 for t in (q, k, v)]


def _capture(qkv, w):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(_attention(*qkv), qkv, w)
    return graph, got


# (first use of the leaves, on a side stream?, whether the capture is refused)
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("first,side,refused", [(_attention, True, False), (_other, True, False), (_attention, False, True), (_other, False, True)])
def test_the_stream_of_the_first_graph_decides(monkeypatch, native, first, side, refused, device_ok):
    if not native:
        if first is _other:
            pytest.skip("what another operation made cannot be asked without the binding")
        monkeypatch.setattr(fmha, "_NATIVE", False)
    qkv = [torch.randn(2, 130, h, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for h in (4, 2, 2)]
    w = torch.randn_like(qkv[0])
    stream = torch.cuda.Stream()
    alive = [_on(stream, lambda: first(*qkv)) if side else first(*qkv)]
    alive.append(_on(stream, lambda: _attention(*qkv)) if not side else _attention(*qkv))  # the second use, on the other stream
    if refused:
        with pytest.raises(RuntimeError, match="default stream"):
            _capture(qkv, w)
        return
    graph, got = _capture(qkv, w)
    with torch.no_grad():
        for t in (qkv[0], w):
            t.copy_(t.flip(1))
    graph.replay()
    want = torch.autograd.grad(_attention(*qkv), qkv, w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert alive
