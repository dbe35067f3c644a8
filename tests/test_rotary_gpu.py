"""Rotary embedding by itself: bit for bit against the arithmetic stated pair by pair, its gradient, and what its positions may hold."""
import pytest
import torch

import int4_reference as ref
from flashck_b200 import ops
from flashck_b200.ops import fmha
from flashck_b200.utils.enums import RopeEnum

pytestmark = pytest.mark.gpu


def _normal(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def _pairs(sections, dealt, half):
    if sections is None:
        return [0] * half
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while len(out) < half:
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                out.append(a)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rope", [RopeEnum.HALF_ROTATED, RopeEnum.INTERLEAVED])
@pytest.mark.parametrize("d,width,sections,dealt", [
    (128, 128, None, False), (64, 64, (8, 12, 12), False), (128, 128, (24, 20, 20), True), (128, 32, (0, 16), False), (64, 20, (3, 7), False),
    (8, 2, None, False), (256, 256, (40, 40, 40, 8), True), (80, 48, (8, 8, 8), False), (192, 64, (10, 11, 11), True),
])
@pytest.mark.parametrize("lead,hq,hkv", [((1,), 1, 1), ((2, 37), 6, 2), ((700,), 3, 5), ((3, 1, 4), 16, 1)])
def test_rotation(dtype, rope, d, width, sections, dealt, lead, hq, hkv):
    tokens, axes = torch.Size(lead).numel(), len(sections) if sections else 1
    q, k = _normal(0, *lead, hq, d, dtype=dtype), _normal(1, *lead, hkv, d, dtype=dtype)
    cos, sin = _normal(2, 60, width // 2, dtype=dtype), _normal(3, 60, width // 2, dtype=dtype)
    pos = torch.randint(0, 60, (axes, *lead) if axes > 1 else lead, device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    pair_axis = _pairs(sections, dealt, width // 2)
    before = [x.clone() for x in (q, k)]
    for inverse in (False, True):
        got = ops.apply_rotary(q, k, pos.int(), cos, sin, sections=sections, interleaved_sections=dealt, rope=rope, inverse=inverse)
        for x, y in zip((q, k), got):
            want = ref.rotate(x.flatten(0, -3), cos, sin, pos.view(axes, tokens), pair_axis, rope == RopeEnum.INTERLEAVED, inverse)
            assert y.shape == x.shape and torch.equal(y.flatten(0, -3), want)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    alone, none = ops.apply_rotary(q, None, pos, cos, sin, sections=sections and list(sections), interleaved_sections=dealt, rope=rope, inverse=True)
    assert torch.equal(alone, got[0]) and none is None


def test_misaligned_rows_and_tables():
    for part in range(4):
        q, k, cos, sin = _normal(0, 5, 4, 64), _normal(1, 5, 2, 64), _normal(2, 9, 32), _normal(3, 9, 32)
        t = []
        for i, x in enumerate((q, k, cos, sin)):
            buf = torch.empty(x.numel() + 8, device="cuda", dtype=torch.bfloat16)
            t.append(buf[i == part: x.numel() + (i == part)].view(x.shape).copy_(x))
        pos = torch.arange(5, device="cuda", dtype=torch.int32)
        got = ops.apply_rotary(t[0], t[1], pos, t[2], t[3])
        for x, y in zip(t, got):
            assert torch.equal(y, ref.rotate(x, t[2], t[3], pos[None], [0] * 32, False))


def test_positions_outside_the_tables_turn_by_nan():
    q = torch.ones(5, 2, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.ones(7, 16, device="cuda", dtype=torch.bfloat16)
    pos = torch.tensor([0, 6, 7, -1, -2 ** 31], device="cuda", dtype=torch.int32)
    for rope in (1, 2):
        y, _ = ops.apply_rotary(q, None, pos, t, t, rope=rope)
        assert torch.isfinite(y[:2]).all() and torch.isnan(y[2:, :, :32]).all() and (y[:, :, 32:] == 1).all()
    two = torch.stack([torch.zeros_like(pos), pos])
    y, _ = ops.apply_rotary(q, None, two, t, t, sections=(8, 8))
    assert torch.isfinite(y[..., :8]).all() and torch.isnan(y[2:, :, 8:16]).all()


def test_positions_of_64_bits():
    q = torch.ones(4, 1, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.ones(7, 32, device="cuda", dtype=torch.bfloat16)
    y, _ = ops.apply_rotary(q, None, torch.tensor([3, 2 ** 32 + 3, -2 ** 32 + 3, 2 ** 31], device="cuda"), t, t)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1:]).all()


def test_empty():
    t = torch.ones(7, 16, device="cuda", dtype=torch.bfloat16)
    q = torch.ones(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    y, k = ops.apply_rotary(q, q[:, :1].contiguous(), torch.empty(0, device="cuda", dtype=torch.int32), t, t)
    assert y.shape == q.shape and k.shape == (0, 1, 64)


@pytest.mark.parametrize("rope", [RopeEnum.HALF_ROTATED, RopeEnum.INTERLEAVED])
def test_gradients(rope):
    """Against the transposed matrix of each token's turn, and against differences: the function is linear, so that a difference of two of
    its values is its value at the difference, up to their roundings."""
    q, k = (_normal(i, 2, 33, h, 64, dtype=torch.float16).requires_grad_() for i, h in ((0, 6), (1, 2)))
    pos = torch.randint(0, 50, (3, 2, 33), device="cuda", generator=torch.Generator("cuda").manual_seed(4))
    a = torch.arange(50, device="cuda")[:, None] * 100.0 ** (-torch.arange(32, device="cuda") / 32)
    cos, sin = a.cos().half(), a.sin().half()
    kw = dict(sections=(8, 12, 12), rope=rope)
    y = ops.apply_rotary_autograd(q, k, pos, cos, sin, **kw)
    assert all(torch.equal(u, v) for u, v in zip(y, ops.apply_rotary(q.detach(), k.detach(), pos, cos, sin, **kw)))
    w = [_normal(5 + i, *t.shape, dtype=torch.float16) for i, t in enumerate(y)]
    g = torch.autograd.grad(y, (q, k), w)
    eye = torch.eye(64, device="cuda", dtype=torch.float16)
    for t, dt in zip(w, g):  # column c of a token's matrix is the turned unit vector c
        m = ref.rotate(eye[None].expand(66, 64, 64).contiguous(), cos, sin, pos.view(3, 66), _pairs((8, 12, 12), False, 32), rope == 1)
        want = torch.einsum("tce,the->thc", m.double(), t.flatten(0, 1).double())
        size = torch.einsum("tce,the->thc", m.double().abs(), t.flatten(0, 1).double().abs())
        assert ((dt.flatten(0, 1).double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -22 * size + 2.0 ** -25).all()
    # <w, f(x + h) - f(x)> = <gradient, h>; f's values and the gradient are each off by half a step at most
    h = _normal(9, *q.shape, dtype=torch.float16)
    with torch.no_grad():
        y0, y1 = (ops.apply_rotary((q + s * h).half(), None, pos, cos, sin, **kw)[0].double() for s in (0, 1))
        moved = ((q + h).half() - q.detach()).double()  # what was really added, before its own rounding
        lhs, rhs = (w[0].double() * (y1 - y0)).sum(), (g[0].double() * ((q + h).half().double() - q.double())).sum()
        allowed = 2.0 ** -11 * ((w[0].double().abs() * (y0.abs() + y1.abs())).sum() + (g[0].double() * moved).abs().sum()) + 1e-3
    assert (lhs - rhs).abs() <= allowed


def test_gradients_of_one_input_and_broadcast_ones():
    q, k = _normal(0, 9, 4, 64, dtype=torch.bfloat16), _normal(1, 9, 2, 64, dtype=torch.bfloat16)
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    t = _normal(2, 9, 32, dtype=torch.bfloat16)
    u = _normal(3, 9, 32, dtype=torch.bfloat16)
    one = torch.ones((), device="cuda", dtype=torch.bfloat16)
    for leaf, other in ((0, 1), (1, 0)):
        x = [q.clone(), k.clone()]
        x[leaf].requires_grad_()
        y = ops.apply_rotary_autograd(*x, pos, t, u)
        g, = torch.autograd.grad(y[leaf], x[leaf], one.expand_as(y[leaf]), retain_graph=True)
        assert torch.equal(g, ops.apply_rotary(torch.ones_like(x[leaf]), None, pos, t, u, inverse=True)[0])
        assert not y[other].requires_grad or torch.autograd.grad(y[other].sum(), x[leaf], allow_unused=True)[0] is None \
            or (torch.autograd.grad(y[other].sum(), x[leaf], allow_unused=True)[0] == 0).all()
    q.requires_grad_()
    y, none = ops.apply_rotary_autograd(q, None, pos, t, u)
    assert none is None
    y.sum().backward()
    assert torch.equal(q.grad, ops.apply_rotary(torch.ones_like(y), None, pos, t, u, inverse=True)[0])


def test_attention_behind_the_rotation():
    """Turned queries and keys through the attention and back, as a training step has them; plain autograd over the same arithmetic."""
    q, k, v = (_normal(i, 1, 130, h, 64, dtype=torch.bfloat16).requires_grad_() for i, h in ((0, 4), (1, 2), (2, 2)))
    pos = torch.arange(130, device="cuda", dtype=torch.int32)
    a = torch.arange(130, device="cuda")[:, None] * 10000.0 ** (-torch.arange(32, device="cuda") / 32)
    cos, sin = a.cos().bfloat16(), a.sin().bfloat16()
    w = _normal(7, 1, 130, 4, 64, dtype=torch.bfloat16)
    g = torch.autograd.grad(ops.fmha_autograd(*ops.apply_rotary_autograd(q, k, pos, cos, sin), v, causal=True), (q, k, v), w)
    x = [t.detach().double().requires_grad_() for t in (q, k, v)]

    def turn(t):
        lo, hi = t[..., :32], t[..., 32:]
        c, s = cos.double()[None, :, None], sin.double()[None, :, None]
        return torch.cat([lo * c - hi * s, lo * s + hi * c], -1)

    s = torch.einsum("bihd,bjhd->bhij", turn(x[0]), turn(x[1]).repeat_interleave(2, 2)) / 8
    s = s.masked_fill(torch.ones(130, 130, device="cuda").triu(1).bool(), -torch.inf)
    o = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), x[2].repeat_interleave(2, 2))
    want = torch.autograd.grad(o, x, w.double())
    for a, b in zip(g, want):  # every tensor on the way is rounded to 8 bits: a few half steps (2^-8) of the largest value
        assert ((a.double() - b).abs() <= 8 * 2.0 ** -8 * b.abs().amax()).all()


@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream")
@pytest.mark.parametrize("native", [True, False])
def test_captured(monkeypatch, native):
    if not native:
        monkeypatch.setattr(fmha, "_NATIVE", False)
    q = _normal(0, 20, 4, 64, dtype=torch.bfloat16).requires_grad_()
    pos = torch.arange(20, device="cuda", dtype=torch.int32)
    t = _normal(2, 20, 32, dtype=torch.bfloat16)
    w = _normal(3, 20, 4, 64, dtype=torch.bfloat16)
    call = lambda: torch.autograd.grad(ops.apply_rotary_autograd(q, None, pos, t, t)[0], q, w)[0]  # noqa: E731
    alive = ops.apply_rotary_autograd(q, None, pos, t, t)  # on the default stream: a captured pass is refused while it lives
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(graph):
            call()
    del alive
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    w.copy_(w.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, ops.apply_rotary(w, None, pos, t, t, inverse=True)[0])


def test_the_binding_and_python_agree(monkeypatch):
    assert fmha._native()
    q, k = _normal(0, 9, 4, 64, dtype=torch.bfloat16), _normal(1, 9, 2, 64, dtype=torch.bfloat16)
    pos, t = torch.arange(27, device="cuda", dtype=torch.int32).view(3, 9), _normal(2, 27, 32, dtype=torch.bfloat16)
    calls = lambda: [x for kw in (dict(sections=(8, 12, 12)), dict(sections=(12, 10, 10), interleaved_sections=True, rope=1), dict(sections=[8, 12, 12]))  # noqa: E731
                     for x in ops.apply_rotary(q, k, pos, t, t, **kw)]
    a = calls()
    monkeypatch.setattr(fmha, "_NATIVE", False)
    assert all(torch.equal(x, y) for x, y in zip(a, calls()))
