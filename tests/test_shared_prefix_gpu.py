"""Decode over a shared prefix against attention over the concatenation in 64 bits."""
import pytest
import torch

from attention_reference import assert_within, forward, half_step
from flashck_b200 import _lib, ops
from flashck_b200.nn import FlashAttention

pytestmark = pytest.mark.gpu


def _problem(lens, tokens, prefix, hq, hkv, d, dtype, page, seed=0, spare=3):
    """q per sequence, the arguments of the call, and per sequence the concatenated K and V.  Pools and tails hold NaN where no key is."""
    g = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)  # noqa: E731
    kp, vp = normal(prefix, hkv, d), normal(prefix, hkv, d)
    own = [(normal(n, hkv, d), normal(n, hkv, d)) for n in lens]
    q = [normal(t, hq, d) for t in tokens]
    b, cap = len(lens), max(max(lens), 1)
    kw = dict(seqlen_k=torch.tensor(lens, dtype=torch.int32, device="cuda"), prefix_len=prefix)
    nan = lambda *s: torch.full(s, float("nan"), device="cuda", dtype=dtype)  # noqa: E731
    if page:
        n_pre, per = -(-prefix // page), -(-cap // page)
        ids = torch.randperm(n_pre + b * per + spare, generator=g, device="cuda").to(torch.int32)
        k, v = nan(ids.numel(), page, hkv, d), nan(ids.numel(), page, hkv, d)
        table = ids[n_pre: n_pre + b * per].view(b, per).contiguous()
        for pool, pre, i in ((k, kp, 0), (v, vp, 1)):
            flat = pool.view(-1, hkv, d)
            at = lambda pages, n: (pages.long()[:, None] * page + torch.arange(page, device="cuda")).flatten()[:n]  # noqa: E731
            flat[at(ids[:n_pre], prefix)] = pre
            for s, n in enumerate(lens):
                flat[at(table[s], n)] = own[s][i]
        args = (k, v, k, v)
        kw.update(prefix_table=ids[:n_pre].contiguous(), block_table=table)
    else:
        k, v = nan(b, cap, hkv, d), nan(b, cap, hkv, d)
        for s, n in enumerate(lens):
            k[s, :n], v[s, :n] = own[s]
        args = (kp, vp, k, v)
    if len(set(tokens)) > 1:
        kw.update(cu_seqlens_q=torch.tensor([0] + tokens).cumsum(0).cuda(), max_seqlen_q=max(tokens))
        qt = torch.cat(q)
    else:
        qt = torch.stack(q)
    return qt, args, kw, q, [(torch.cat([kp, a]), torch.cat([vp, c])) for a, c in own]


def _check(lens, tokens, prefix, hq, hkv, d, dtype, page, causal=True, scale=None, seed=0):
    qt, args, kw, q, whole = _problem(lens, tokens, prefix, hq, hkv, d, dtype, page, seed)
    o, lse = ops.fmha_fwd_shared_prefix(qt, *args, causal=causal, return_lse=True, scale=scale, **kw)
    packed = "cu_seqlens_q" in kw
    u, row = half_step(dtype), 0
    for s, (k, v) in enumerate(whole):
        n, t = lens[s], tokens[s]
        # own keys: bottom-right causal; the prefix wholly visible even where a sequence has fewer own keys than queries
        bias = torch.zeros(1, 1, t, prefix + n, device="cuda", dtype=torch.float64)
        if causal:
            i, j = torch.arange(t, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            bias[0, 0, :, prefix:].masked_fill_(j > n - t + i, -torch.inf)
        want, want_lse = forward(q[s][None], k[None], v[None], scale or d ** -0.5, (0, -1, -1), bias=bias)
        spread, _ = forward(q[s][None], k[None], v[None].abs(), scale or d ** -0.5, (0, -1, -1), bias=bias)
        # P rounded where it meets V (u of the sum of magnitudes), S and exp as in the backward's bounds, O rounded once
        e = d * 2.0 ** -24 * (q[s].double().abs().amax() * k.double().abs().sum(-1).amax() if k.numel() else 0.0) * (scale or d ** -0.5) + 2.0 ** -18
        got, got_lse = (o[row: row + t], lse[:, row: row + t]) if packed else (o[s], lse[s])
        row += t
        assert_within(f"o of sequence {s}", got, want[0], (u + e) * spread[0] + u * want[0].abs())
        empty = torch.isneginf(want_lse[0])
        assert torch.equal(torch.isneginf(got_lse), empty)
        # the row sum adds the rounded exponentials of thousands of keys: their errors, and a rounding of the LSE itself
        assert ((got_lse - want_lse[0]).abs()[~empty] <= e + 2.0 ** -20 * (1 + want_lse[0].abs()[~empty])).all()
    return o, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("lens,tokens,prefix", [
    ([5, 0, 1, 300], 1, 100), ([40] * 6, 1, 1), ([7, 65, 129], 1, 1000), ([300, 2, 33], 4, 2000), ([1], 1, 5000),
    ([100] * 40, 1, 300), ([9, 90, 5, 0, 17], [1, 4, 2, 3, 1], 777), ([64, 16], 1, 0), ([5, 30], 20, 130),
])
def test_against_the_concatenation(dtype, d, page, lens, tokens, prefix, device_ok):
    tokens = tokens if isinstance(tokens, list) else [tokens] * len(lens)
    _check(lens, tokens, prefix, 8, 2, d, dtype, page)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (16, 1), (12, 4), (7, 7), (20, 4)])
def test_head_groups(d, hq, hkv, device_ok):
    _check([20, 0, 70, 3, 16], [1] * 5, 500, hq, hkv, d, torch.bfloat16, 16)
    _check([20, 30, 70], [3] * 3, 500, hq, hkv, d, torch.bfloat16, 0)


@pytest.mark.parametrize("d", [64, 128])
def test_more_rows_than_one_launch_takes(d, device_ok):
    """700 sequences x 4 heads of a group: the tcgen05 split mode is launched over the rows in runs."""
    _check([i % 5 for i in range(700)], [1] * 700, 260, 4, 1, d, torch.bfloat16, 16)


def test_no_mask_and_a_scale(device_ok):
    _check([10, 50], [4, 4], 300, 8, 2, 128, torch.bfloat16, 16, causal=False, scale=0.2)


def test_same_as_split_kv_over_one_table(device_ok):
    """The prefix's pages in front of every row of the block table, the own pages a slice of its columns."""
    b, d, page, n_pre, per = 5, 128, 16, 20, 4
    ids = torch.randperm(n_pre + b * per, device="cuda").to(torch.int32)
    k, v = (torch.randn(ids.numel(), page, 2, d, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    table = torch.cat([ids[:n_pre].expand(b, -1), ids[n_pre:].view(b, per)], dim=1).contiguous()
    own = torch.tensor([1, 16, 64, 33, 50], dtype=torch.int32, device="cuda")
    q = torch.randn(b, 1, 8, d, device="cuda", dtype=torch.bfloat16)
    got, lse = ops.fmha_fwd_shared_prefix(q, k, v, k, v, prefix_len=n_pre * page, prefix_table=ids[:n_pre].contiguous(), seqlen_k=own,
                                          block_table=table[:, n_pre:], causal=True, return_lse=True)
    want, want_lse = ops.fmha_fwd_splitkv(q, k, v, seqlen_k=own + n_pre * page, block_table=table, causal=True, return_lse=True)
    u = half_step(torch.bfloat16)
    # each side: P rounded (u of the mean |v| a row sees, at most max |v|), O rounded
    assert ((got.double() - want.double()).abs() <= 2 * u * (v.double().abs().amax() + want.double().abs())).all()
    assert ((lse - want_lse).abs() <= 2.0 ** -16).all()


def test_rows_of_no_sequence_are_left(device_ok):
    from flashck_b200 import _lib
    q = torch.randn(9, 4, 64, device="cuda", dtype=torch.bfloat16)
    kp, k = torch.randn(40, 2, 64, device="cuda", dtype=torch.bfloat16), torch.randn(3, 8, 2, 64, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([2, 3, 3, 6], device="cuda")
    o, lse = torch.full_like(q, 7.0), torch.full((4, 9), 7.0, device="cuda")
    n = _lib.lib().FlashckSharedPrefixWorkspace(40, 0, 0, 3, 9, 3, 4, 2, 64, 1, 4)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    sl = torch.tensor([1, 8, 3], dtype=torch.int32, device="cuda")
    p = lambda t: t.data_ptr()  # noqa: E731
    rc = _lib.lib().FmhaFwdSharedPrefix(p(q), p(kp), p(kp), p(k), p(k), p(o), p(lse), p(ws), 0, 0, p(sl), p(cu), 40, 0, 40, 0, 3, 0, 8, 3, 9, 3,
                                        4, 2, 64, 64, 0.0, 1, torch.cuda.current_stream().cuda_stream, 4)
    assert rc == 0
    assert (o[:2] == 7).all() and (o[6:] == 7).all() and (lse[:, :2] == 7).all() and (lse[:, 6:] == 7).all()
    assert not (o[2:6] == 7).all(-1).any() and torch.isfinite(lse[:, 2:6]).all()
    again = ops.fmha_fwd_shared_prefix(q, kp, kp, k, k, seqlen_k=sl, cu_seqlens_q=cu, max_seqlen_q=3, causal=True)
    assert torch.equal(again[2:6], o[2:6])


@pytest.mark.parametrize("prefix", [0, 40])
def test_caches_without_room(prefix, device_ok):
    q, kp = torch.randn(2, 1, 4, 64, device="cuda", dtype=torch.bfloat16), torch.randn(prefix, 2, 64, device="cuda", dtype=torch.bfloat16)
    sl = torch.zeros(2, dtype=torch.int32, device="cuda")
    if not prefix:  # (no tensor of size 0 has an address: a pool of one page that nobody uses)
        kp = torch.randn(1, 2, 64, device="cuda", dtype=torch.bfloat16)
    pool = torch.full((1, 16, 2, 64), float("nan"), device="cuda", dtype=torch.bfloat16)
    o, lse = ops.fmha_fwd_shared_prefix(q, kp, kp, pool, pool, prefix_len=prefix, seqlen_k=sl, return_lse=True,
                                        block_table=torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    if prefix:
        want, want_lse = ops.fmha_fwd_splitkv(q, kp.expand(2, -1, -1, -1).contiguous(), kp.expand(2, -1, -1, -1).contiguous(), return_lse=True)
        assert ((o.double() - want.double()).abs() <= 4 * half_step(torch.bfloat16) * kp.double().abs().amax()).all()
        assert ((lse - want_lse).abs() <= 2.0 ** -16).all()
    else:
        assert not o.any() and torch.isneginf(lse).all()


def test_captured_replayed_and_on_another_stream(device_ok):
    qt, args, kw, _, _ = _problem([30, 5, 100], [1] * 3, 700, 8, 2, 128, torch.bfloat16, 16)
    want = ops.fmha_fwd_shared_prefix(qt, *args, causal=True, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.fmha_fwd_shared_prefix(qt, *args, causal=True, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.fmha_fwd_shared_prefix(qt, *args, causal=True, **kw)
    kw["seqlen_k"].copy_(torch.tensor([3, 77, 1]))
    qt.copy_(qt.flip(0))
    args[2][kw["block_table"].long().flatten()] = 0.25  # (every own page is defined now)
    args[3][kw["block_table"].long().flatten()] = 0.5
    graph.replay()
    assert torch.equal(got, ops.fmha_fwd_shared_prefix(qt, *args, causal=True, **kw))


def test_sample_and_train(device_ok):
    """The operators together: answers are decoded behind one prompt, token by token, then trained on as packed sequences."""
    torch.manual_seed(1)
    b, n_prompt, n_new, d, hkv, hq = 3, 50, 4, 64, 2, 4
    attn = FlashAttention(hq, d, hkv, causal=True)
    mk = lambda *s: torch.randn(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    kp, vp, qp = mk(n_prompt, hkv, d), mk(n_prompt, hkv, d), mk(n_prompt, hq, d)
    kn, vn, qn = mk(b, n_new, hkv, d), mk(b, n_new, hkv, d), mk(b, n_new, hq, d)
    k_cache, v_cache = mk(b, 16, hkv, d), mk(b, 16, hkv, d)
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")
    steps = []
    for t in range(n_new):
        attn.append_kv(None, k_cache, v_cache, kn[:, t: t + 1].contiguous(), vn[:, t: t + 1].contiguous(), lens)
        lens = lens + 1
        steps.append(attn.forward_shared_prefix(qn[:, t: t + 1].contiguous(), kp, vp, k_cache, v_cache, lens))
    decoded = torch.cat(steps, dim=1)
    cu = torch.arange(b + 1, device="cuda") * (n_prompt + n_new)
    q, k, v = (torch.cat([p.expand(b, -1, -1, -1), n], dim=1).flatten(0, 1).requires_grad_() for p, n in ((qp, qn), (kp, kn), (vp, vn)))
    o = attn(q, k, v, cu, cu, n_prompt + n_new, n_prompt + n_new)
    trained = o.detach().view(b, n_prompt + n_new, hq, d)[:, n_prompt:]
    u = half_step(torch.bfloat16)
    assert ((decoded.double() - trained.double()).abs() <= 2 * u * (v.detach().double().abs().amax() + trained.double().abs())).all()
    o.sum().backward()
    assert all(torch.isfinite(t.grad).all() and t.grad.any() for t in (q, k, v))


@pytest.mark.parametrize("page,hq,hkv", [(16, 32, 8), (64, 16, 2)])
def test_split_kv_repeats(page, hq, hkv, device_ok):
    """The decode kernel gives a stage of the ring back only when all of it has been read: equal calls, equal bits."""
    lens, tokens, d = [2000, 40, 1300, 0, 129, 3100], [16, 7, 1, 3, 40, 33], 128
    per = -(-max(lens) // page)
    g = torch.Generator("cuda").manual_seed(1)
    k, v = (torch.randn(6 * per, page, hkv, d, device="cuda", generator=g).bfloat16() for _ in range(2))
    table = torch.randperm(6 * per, device="cuda", generator=g).int().view(6, per)
    cu = torch.tensor([0] + tokens).cumsum(0).cuda()
    q = torch.randn(sum(tokens), hq, d, device="cuda", generator=g).bfloat16()
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    _lib.set_instance_param(2, "use_sm100_splitkv", 0)
    try:
        call = lambda: ops.fmha_fwd_splitkv(q, k, v, seqlen_k=sl, block_table=table, cu_seqlens_q=cu, max_seqlen_q=40, num_splits=3)  # noqa: E731
        first = call()
        differ = torch.zeros((), device="cuda", dtype=torch.int64)
        for _ in range(8000):
            differ += (call() != first).any()
    finally:
        _lib.set_instance_param(2, "use_sm100_splitkv", 1)
    assert int(differ) == 0
