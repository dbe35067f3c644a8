"""The backward pass against its formula in 64 bits, within bounds that count its roundings."""
import pytest
import torch

from attention_reference import assert_within, forward, gradients, half_step
from flashck_b200 import _lib, ops
from flashck_b200.nn import FlashAttention

pytestmark = pytest.mark.gpu
NONE, CAUSAL = (0, -1, -1), (2, -1, 0)


@pytest.fixture(params=["tcgen05", "general"])
def instance(request):
    """Both instances of the kernels take a test; a problem that the tcgen05 one does not serve runs on the other both times."""
    _lib.set_instance_param(0, "use_sm100_bwd", int(request.param == "tcgen05"))
    yield request.param
    _lib.set_instance_param(0, "use_sm100_bwd", 1)


def _options(mask):
    return dict(mask_type=mask[0], window_size=mask[1:])


def _problem(b, sq, sk, hq, hkv, d, dtype, mask, seed=0, bias=None, slopes=None, cap=0.0, scale=None):
    g = torch.Generator("cuda").manual_seed(seed)
    q, dout = (torch.randn(b, sq, hq, d, device="cuda", generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(b, sk, hkv, d, device="cuda", generator=g).to(dtype) for _ in range(2))
    o, lse = forward(q, k, v, scale or d ** -0.5, mask, bias, slopes, cap)
    return dout, q, k, v, o.to(dtype), lse.float()


def _check(args, mask, bias=None, slopes=None, cap=0.0, dlse=None, scale=None):
    d = args[1].shape[-1]
    want, bound = gradients(*args, scale or d ** -0.5, mask, bias, slopes, cap, dlse)
    got = ops.fmha_bwd(*args, scale=scale, bias=bias, alibi_slopes=slopes, logits_soft_cap=cap, dlse=dlse, return_dbias=bias is not None,
                       **_options(mask))
    for n, x, w, e in zip(("dq", "dk", "dv"), got, want, bound):
        assert_within(n, x, w, e)
    if bias is not None:
        w, e = want[3], bound[3]
        axes = [a for a in (0, 1) if bias.shape[a] == 1]
        if axes:
            w, e = w.sum(axes, keepdim=True), e.sum(axes, keepdim=True)
        assert_within("dbias", got[3], w, e + half_step(bias.dtype) * w.abs() + 2.0 ** -25)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sq,sk,mask", [
    (1, 1, NONE), (1, 300, CAUSAL), (64, 64, CAUSAL), (128, 128, NONE), (129, 129, CAUSAL), (257, 1000, CAUSAL), (300, 5, NONE),
    (200, 100, CAUSAL),                          # rows that see nothing
    (333, 333, (2, 17, 0)), (500, 500, (1, 64, 32)), (260, 700, (3, 5, 300)), (300, 40, (1, 20, 0)),
    (640, 640, (2, 0, 0)), (384, 512, (2, -1, 100)),
])
def test_dense(dtype, d, sq, sk, mask, instance, device_ok):
    _check(_problem(2, sq, sk, 4, 2, d, dtype, mask), mask)


def test_which_instance_serves(instance, device_ok):
    args = _problem(1, 64, 64, 2, 2, 64, torch.bfloat16, NONE)
    ops.fmha_bwd(*args)
    assert _lib.get_instance_param(0, "last_bwd_instance") == int(instance == "tcgen05")
    bias = torch.zeros(1, 1, 64, 64, device="cuda", dtype=torch.bfloat16)
    ops.fmha_bwd(*args, bias=bias)
    assert _lib.get_instance_param(0, "last_bwd_instance") == int(instance == "tcgen05")
    ops.fmha_bwd(args[0], args[1], args[2][:, :0].contiguous(), args[3][:, :0].contiguous(), *args[4:])  # (no key: the general one)
    assert _lib.get_instance_param(0, "last_bwd_instance") == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (12, 4), (7, 7), (6, 2)])
def test_head_groups(d, hq, hkv, instance, device_ok):
    _check(_problem(3, 200, 200, hq, hkv, d, torch.bfloat16, CAUSAL), CAUSAL)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask", [NONE, CAUSAL, (2, 50, 0)])
@pytest.mark.parametrize("slopes_rank", [None, 1, 2])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_alibi_and_soft_cap(d, mask, slopes_rank, cap, instance, device_ok):
    slopes = None if slopes_rank is None else torch.rand(1 if slopes_rank == 1 else 2, 4, device="cuda") * 0.2
    _check(_problem(2, 190, 270, 4, 2, d, torch.bfloat16, mask, slopes=slopes, cap=cap), mask, slopes=slopes, cap=cap)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("planes", [(1, 1), (1, 4), (3, 4)])
@pytest.mark.parametrize("sq,sk,mask", [(70, 131, NONE), (130, 130, CAUSAL), (1, 1, NONE), (300, 264, (2, 60, 5)), (128, 256, NONE)])
@pytest.mark.parametrize("dtype,cap", [(torch.float16, 20.0), (torch.bfloat16, 0.0)])
def test_bias_and_its_gradient(d, planes, sq, sk, mask, dtype, cap, instance, device_ok):
    bias = torch.randn(*planes, sq, sk, device="cuda", dtype=dtype)
    _check(_problem(3, sq, sk, 4, 2, d, dtype, mask, bias=bias, cap=cap), mask, bias=bias, cap=cap)


def test_scale_and_gradient_of_the_lse(instance, device_ok):
    args = _problem(2, 150, 150, 4, 2, 128, torch.bfloat16, CAUSAL, scale=0.3)
    _check(args, CAUSAL, dlse=torch.randn(2, 4, 150, device="cuda"), scale=0.3)


LENGTHS = [([1, 0, 130, 64, 257], [1, 0, 130, 64, 257]), ([5, 128, 3], [300, 128, 0]), ([200], [200]), ([0, 0], [7, 9])]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask", [NONE, CAUSAL, (2, 40, 0)])
@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("pad", [0, 37])
def test_packed(d, mask, lens, pad, instance, device_ok):
    """Sequences of unequal lengths, with rows in front of the first and behind the last one that hold NaN."""
    nq, nk = lens
    hq, hkv, dtype = 4, 2, torch.bfloat16
    starts = [torch.tensor([0] + n).cumsum(0).cuda() + pad for n in lens]
    total = [sum(n) + 2 * pad for n in lens]
    nan = lambda rows, h: torch.full((rows, h, d), float("nan"), device="cuda", dtype=dtype)  # noqa: E731
    q, k, v, dout, o = nan(total[0], hq), nan(total[1], hkv), nan(total[1], hkv), nan(total[0], hq), nan(total[0], hq)
    lse = torch.full((hq, total[0]), float("nan"), device="cuda")
    want = []
    for n, (a, c) in enumerate(zip(nq, nk)):
        args = _problem(1, a, c, hq, hkv, d, dtype, mask, seed=n)
        qs, ks = slice(starts[0][n], starts[0][n + 1]), slice(starts[1][n], starts[1][n + 1])
        for t, x, rows in ((dout, args[0], qs), (q, args[1], qs), (k, args[2], ks), (v, args[3], ks), (o, args[4], qs)):
            t[rows] = x[0]
        lse[:, qs] = args[5][0]
        want.append((qs, ks, *gradients(*args, d ** -0.5, mask)))
    for longest in ((max(nq), max(nk)), (0, 0)):
        dq, dk, dv = ops.fmha_bwd_var_len(dout, q, k, v, o, lse, *starts, *longest, **_options(mask))
        for qs, ks, (wq, wk, wv, _), (eq, ek, ev, _) in want:
            assert_within("dq", dq[qs], wq[0], eq[0])
            assert_within("dk", dk[ks], wk[0], ek[0])
            assert_within("dv", dv[ks], wv[0], ev[0])
        for t, s in ((dq, starts[0]), (dk, starts[1]), (dv, starts[1])):
            assert not t[: s[0]].any() and not t[s[-1]:].any()  # rows of no sequence: zeros


@pytest.mark.parametrize("lens", [[(i * 37) % 200 for i in range(300)],               # more sequences than the schedule orders
                                  [(i * 131) % 700 + 1 for i in range(40)],             # many items per CTA, levels of unequal size
                                  [2000, 1, 1500, 0, 900, 128, 3]])
@pytest.mark.parametrize("hq,hkv,d,mask", [(8, 2, 128, CAUSAL), (6, 6, 64, NONE), (8, 1, 64, (2, 300, 10))])
def test_many_items(lens, hq, hkv, d, mask, device_ok):
    """Several items per CTA: every sequence alone gives the same bits as in the packed call, and some are held to the formula."""
    args = [_problem(1, n, n, hq, hkv, d, torch.bfloat16, mask, seed=i) for i, n in enumerate(lens)]
    dout, q, k, v, o = (torch.cat([a[j][0] for a in args]) for j in range(5))
    lse = torch.cat([a[5][0] for a in args], dim=1).contiguous()
    cu = torch.tensor([0] + lens).cumsum(0).cuda()
    got = ops.fmha_bwd_var_len(dout, q, k, v, o, lse, cu, cu, max(lens), max(lens), **_options(mask))
    at = cu.tolist()
    for i, a in enumerate(args):
        part = [g[at[i]: at[i + 1]] for g in got]
        if i % 10 == 0 or lens[i] > 1000:
            want, bound = gradients(*a, d ** -0.5, mask)
            for n, x, w, e in zip(("dq", "dk", "dv"), part, want, bound):
                assert_within(f"{n} of sequence {i}", x, w[0], e[0])
        assert all(torch.equal(x, y[0]) for x, y in zip(part, ops.fmha_bwd(*a, **_options(mask))))


@pytest.mark.parametrize("planes", [1, 2])
def test_packed_bias_gradient_is_zero_outside_the_blocks(planes, instance, device_ok):
    nq, nk, d, hq = [40, 190], [170, 65], 64, 2
    cu_q, cu_k = (torch.tensor([0] + n).cumsum(0).cuda() for n in (nq, nk))
    bias = torch.randn(1, planes, sum(nq), sum(nk), device="cuda", dtype=torch.bfloat16)
    parts = [_problem(1, a, c, hq, hq, d, torch.bfloat16, NONE, seed=n, bias=bias[:, :, cu_q[n]: cu_q[n + 1], cu_k[n]: cu_k[n + 1]])
             for n, (a, c) in enumerate(zip(nq, nk))]
    dout, q, k, v, o = (torch.cat([p[n][0] for p in parts]) for n in range(5))
    lse = torch.cat([p[5][0] for p in parts], dim=1).contiguous()
    got = ops.fmha_bwd_var_len(dout, q, k, v, o, lse, cu_q, cu_k, max(nq), max(nk), bias=bias, return_dbias=True)[3]
    outside = torch.ones_like(got, dtype=torch.bool)
    for n, p in enumerate(parts):
        block = (slice(None), slice(None), slice(cu_q[n], cu_q[n + 1]), slice(cu_k[n], cu_k[n + 1]))
        want, bound = gradients(*p, d ** -0.5, NONE, bias=bias[block])
        w, e = (t.sum(1, keepdim=True) if planes == 1 else t for t in (want[3], bound[3]))
        assert_within("dbias", got[block], w, e + half_step(bias.dtype) * w.abs())
        outside[block] = False
    assert not got[outside].any()


@pytest.mark.parametrize("d", [64, 128])
def test_nan_of_another_sequence_does_not_spread(d, instance, device_ok):
    """Tiles reach past a sequence's end into the next one, whose rows hold NaN and infinities here."""
    args = _problem(2, 100, 100, 2, 2, d, torch.bfloat16, NONE)
    for t in args[:5]:
        t[1] = float("nan")
        t[1, ::2] = float("inf")
    got = ops.fmha_bwd(*args)
    want, bound = gradients(*(t[:1] for t in args), d ** -0.5, NONE)
    for n, x, w, e in zip(("dq", "dk", "dv"), got, want, bound):
        assert_within(n, x[:1], w, e)


def test_equal_calls_give_equal_bits(instance, device_ok):
    args = _problem(2, 700, 700, 8, 2, 128, torch.bfloat16, CAUSAL)
    first = ops.fmha_bwd(*args, causal=True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.fmha_bwd(*args, causal=True)))


def test_empty_sizes(instance, device_ok):
    def call(b, sq, sk):
        t = lambda n: torch.zeros(b, n, 2, 64, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        return ops.fmha_bwd(t(sq), t(sq), t(sk), t(sk), t(sq), torch.full((b, 2, sq), -float("inf"), device="cuda"))
    for b, sq, sk in ((0, 4, 4), (2, 0, 0), (2, 0, 5), (2, 5, 0)):
        for x in call(b, sq, sk):
            assert not x.any()


def test_differences(device_ok):
    """<gradient, direction> against the difference quotient of the exact loss, for every input at once."""
    d, mask = 64, CAUSAL
    dout, q, k, v, _, _ = _problem(1, 40, 60, 4, 2, d, torch.float16, mask, cap=8.0)
    dirs = [torch.randn_like(t, dtype=torch.float64) for t in (q, k, v)]

    def loss(h):
        o, _ = forward(*(t.double() + h * x for t, x in zip((q, k, v), dirs)), d ** -0.5, mask, cap=8.0)
        return (o * dout.double()).sum()

    o, lse = forward(q, k, v, d ** -0.5, mask, cap=8.0)
    args = (dout, q, k, v, o.half(), lse.float())
    got = ops.fmha_bwd(*args, causal=True, logits_soft_cap=8.0)
    _, bound = gradients(*args, d ** -0.5, mask, cap=8.0)
    h = 1e-5
    slope = (loss(h) - loss(-h)) / (2 * h)
    # O enters D rounded: dq and dk move by dS = P u sum |dO O| at most
    extra = half_step(torch.float16) * (dout.double() * o).abs().sum(-1).amax() * d ** -0.5
    allowed = sum((e * x.abs()).sum() for e, x in zip(bound, dirs))
    allowed = allowed + extra * (dirs[0].abs().sum() * k.double().abs().amax() + q.double().abs().amax() * dirs[1].abs().sum() * q.shape[1])
    assert abs(sum((g.double() * x).sum() for g, x in zip(got, dirs)) - slope) <= allowed


def test_autograd_dense_and_packed(device_ok):
    q, k, v = (torch.randn(2, 77, h, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for h in (4, 2, 2))
    bias = torch.randn(1, 4, 77, 77, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    o, lse = ops.fmha_autograd(q, k, v, causal=True, return_lse=True, bias=bias)
    plain = ops.fmha_fwd(q, k, v, causal=True, return_lse=True, bias=bias)
    assert torch.equal(o, plain[0]) and torch.equal(lse, plain[1])
    w, wl = torch.randn_like(o), torch.randn_like(lse)
    ((o * w).sum() + (lse * wl).sum()).backward()
    want = ops.fmha_bwd(w, q.detach(), k.detach(), v.detach(), o.detach(), lse.detach(), causal=True, bias=bias.detach(), dlse=wl, return_dbias=True)
    for t, g in zip((q, k, v, bias), want):
        assert torch.equal(t.grad, g)
    # the LSE alone; a gradient that is expanded, not contiguous; an input that needs none
    g = torch.autograd.grad(ops.fmha_autograd(q, k, v.detach(), return_lse=True)[1].sum(), (q, k))
    assert all(torch.isfinite(x).all() for x in g)
    g1 = torch.autograd.grad(ops.fmha_autograd(q, k, v).sum(), (q, k, v))
    o, lse = ops.fmha_fwd(q, k, v, return_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(g1, ops.fmha_bwd(torch.ones_like(o), q.detach(), k.detach(), v.detach(), o, lse)))
    cu = torch.tensor([0, 30, 77], device="cuda")
    qp, kp, vp = (t.detach()[0].clone().requires_grad_() for t in (q, k, v))
    ops.fmha_autograd_var_len(qp, kp, vp, cu, cu, 47, 47, causal=True).square().sum().backward()
    assert all(torch.isfinite(t.grad).all() and t.grad.any() for t in (qp, kp, vp))


def test_attention_module_trains(device_ok):
    """The module inside projections: its gradients against the same layer in 64 bits."""
    torch.manual_seed(0)
    attn = FlashAttention(4, 64, 2, causal=True)
    x = torch.randn(2, 50, 96, device="cuda", dtype=torch.bfloat16)
    proj = [torch.nn.Linear(96, h * 64, bias=False, device="cuda", dtype=torch.bfloat16) for h in (4, 2, 2)]
    q, k, v = (p(x).unflatten(-1, (-1, 64)) for p in proj)
    out = attn(q, k, v)
    assert out.requires_grad
    out.square().sum().backward()
    wide = [p.weight.detach().double().requires_grad_() for p in proj]
    qd, kd, vd = ((x.double() @ w.T).unflatten(-1, (-1, 64)) for w in wide)
    o, _ = forward(qd, kd, vd, 64 ** -0.5, CAUSAL)
    o.square().sum().backward()
    for p, w in zip(proj, wide):
        # five roundings of at most half a step on the way (q, o, dO, dq, the product), in norm
        assert (p.weight.grad.double() - w.grad).norm() <= 5 * half_step(torch.bfloat16) * 2 * w.grad.norm()
    with torch.no_grad():
        assert not attn(q, k, v).requires_grad


def test_other_stream_and_captured(instance, device_ok):
    args = _problem(2, 300, 300, 4, 2, 128, torch.bfloat16, CAUSAL)
    want = ops.fmha_bwd(*args, causal=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.fmha_bwd(*args, causal=True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.fmha_bwd(*args, causal=True)
    for t in args[:2]:
        t.copy_(t.flip(1))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, ops.fmha_bwd(*args, causal=True)))


def test_first_call_of_a_thread(device_ok):
    """A thread that has made no CUDA call of its own yet (autograd's worker threads are such): forward and backward."""
    import threading
    args = _problem(1, 130, 130, 2, 2, 128, torch.bfloat16, CAUSAL)
    want = ops.fmha_bwd(*args, causal=True)
    got, failed = [], []

    def work(f):
        try:
            got.append(f())
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    for f in (lambda: ops.fmha_bwd(*args, causal=True), lambda: ops.fmha_fwd(*args[1:4], causal=True)):
        t = threading.Thread(target=work, args=(f,))
        t.start()
        t.join()
    assert not failed, failed
    assert all(torch.equal(a, b) for a, b in zip(got[0], want)) and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("d", [64, 128])
def test_bias_that_hides(d, instance, device_ok):
    """Infinities in a bias: whole rows, whole key tiles, single keys.  What is hidden gets nothing at all."""
    bias = torch.randn(2, 4, 200, 300, device="cuda").to(torch.bfloat16)
    bias[:, :, 5:9] = -torch.inf
    bias[0, :, :, 128:256] = -torch.inf
    bias[1, 2, :, 7] = -torch.inf
    bias[:, :, 40, ::2] = -torch.inf
    got = _check(_problem(2, 200, 300, 4, 2, d, torch.bfloat16, NONE, bias=bias), NONE, bias=bias)
    assert not got[0][:, 5:9].any() and not got[1][0, 128:256].any() and not got[2][0, 128:256].any()
    assert not got[3][torch.isneginf(bias)].any()


def test_padding_of_a_differentiable_output_is_zero(device_ok):
    """The output is multiplied by weights whose gradient is o^T times zeros there: what the memory held must not count."""
    total, cu = 300, torch.tensor([7, 40, 200], device="cuda")
    q, k, v = (torch.randn(total, h, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for h in (4, 2, 2))
    for _ in range(2):
        old = torch.full((total, 4, 64), float("nan"), device="cuda", dtype=torch.bfloat16), torch.full((4, total), float("nan"), device="cuda")
        del old  # (the outputs may lie where these did)
        o, lse = ops.fmha_autograd_var_len(q, k, v, cu, cu, 160, 160, causal=True, return_lse=True)
        for rows in (slice(0, 7), slice(200, None)):
            assert not o[rows].any() and not lse[:, rows].any()
        plain, plain_lse = ops.fmha_fwd_var_len(q, k, v, cu, cu, 160, 160, causal=True, return_lse=True)
        assert torch.equal(o[7:200], plain[7:200]) and torch.equal(lse[:, 7:200], plain_lse[:, 7:200])
    # starts in 32 bits; no padding; a batch without a token
    for starts in ([0, 100, total], [0, 0, 0]):
        c = torch.tensor(starts, device="cuda", dtype=torch.int32)
        o = ops.fmha_autograd_var_len(q, k, v, c, c, total, total)
        assert torch.equal(o, ops.fmha_fwd_var_len(q, k, v, c, c, total, total)) if starts[-1] else not o.any()


def test_gradient_that_starts_off_a_boundary(device_ok):
    q, k, v = (torch.randn(1, 70, 2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for _ in range(3))
    w = torch.randn(q.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view_as(q)
    got, want = (torch.autograd.grad(ops.fmha_autograd(q, k, v), (q, k, v), x) for x in (w, w.clone()))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_step(device_ok):
    """Forward and backward in one graph; refused while a graph of the same leaves from the default stream lives."""
    q, k, v = (torch.randn(2, 130, h, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True) for h in (4, 2, 2))
    w = torch.randn_like(q)
    alive = ops.fmha_autograd(q, k, v, causal=True)
    with pytest.raises(RuntimeError, match="recorded on the default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.fmha_autograd(q, k, v, causal=True).backward(w)
    del alive
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.fmha_autograd(q, k, v, causal=True), (q, k, v), w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(ops.fmha_autograd(q, k, v, causal=True), (q, k, v), w)
    with torch.no_grad():
        for t in (q, w):
            t.copy_(t.flip(1))
    graph.replay()
    want = torch.autograd.grad(ops.fmha_autograd(q, k, v, causal=True), (q, k, v), w)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_streams_at_once(device_ok):
    """Calls of different problems on two streams, in flight together."""
    problems = [_problem(2, 700, 700, 4, 2, d, torch.bfloat16, CAUSAL, seed=d) for d in (64, 128)]
    want = [ops.fmha_bwd(*x, causal=True) for x in problems]
    streams = [torch.cuda.Stream() for _ in problems]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (x, s) in enumerate(zip(problems, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.fmha_bwd(*x, causal=True))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, gs in zip(want, got) for g in gs for a, b in zip(g, w))
    assert _lib.device_status() == 0
