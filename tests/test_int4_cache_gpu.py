"""The 4-bit cache: its write bit for bit, its way back, and decode over it against 64 bits."""
import pytest
import torch

import int4_reference as ref
from flashck_b200 import _lib, ops
from flashck_b200.utils.enums import RopeEnum

pytestmark = pytest.mark.gpu
INVALID = 0x40000000  # FLASHCK_STATUS_APPEND_OVERFLOW


def _g(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _normal(g, *shape, dtype):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(lens):
    return torch.tensor([0] + list(lens), dtype=torch.int64).cumsum(0).cuda()


class Cache:
    """Pools (or contiguous rows) whose unused rows hold any codes and NaN params, and the tokens of each sequence."""

    def __init__(self, lens, hkv, d, group, dtype, page, seed=0, room=None, scale=1.0):
        g = _g(seed)
        self.lens, self.d, self.group, self.page, self.dtype = lens, d, group, page, dtype
        room = room or max(max(lens), 1)
        if page:
            per = -(-room // page)
            ids = torch.randperm(len(lens) * per + 2, generator=g, device="cuda").to(torch.int32)
            self.table, rows = ids[: len(lens) * per].view(len(lens), per).contiguous(), (len(lens) * per + 2, page)
        else:
            self.table, rows = None, (len(lens), room)
        self.parts, self.tokens = [], []
        for _ in range(2):
            codes = torch.randint(0, 256, (*rows, hkv, d // 2), generator=g, device="cuda", dtype=torch.uint8)
            params = torch.full((*rows, hkv, d // group, 2), torch.nan, device="cuda", dtype=dtype)
            self.parts += [codes, params]
        for s, n in enumerate(lens):
            four = []
            for i in range(2):
                c, sc, lo = ref.quantise(_normal(g, n, hkv, d, dtype=dtype) * scale, group)
                four += [ref.pack(c), torch.stack([sc, lo], -1).to(dtype)]
            self.tokens.append(four)
            at = self.rows(s, 0, n)
            for part, x in zip(self.parts, four):
                part.flatten(0, 1)[at] = x
        self.seqlen = _i32(lens)

    def rows(self, s, first, last):
        i = torch.arange(first, last, device="cuda")
        return self.table[s].long()[i // self.page] * self.page + i % self.page if self.page else s * self.parts[0].shape[1] + i


def _attend(c, tokens, hq, mask=(2, -1, 0), scale=None, seed=1, q=None, **kw):
    """Runs the call and holds it against 64 bits."""
    g = _g(seed)
    ragged = len(set(tokens)) > 1
    qs = q or [_normal(g, t, hq, c.d, dtype=c.dtype) for t in tokens]
    if ragged:
        kw.update(cu_seqlens_q=_starts(tokens), max_seqlen_q=max(tokens))
    o, lse = ops.fmha_fwd_splitkv_int4(torch.cat(qs) if ragged else torch.stack(qs), *c.parts, seqlen_k=c.seqlen, block_table=c.table, scale=scale,
                                       mask_type=mask[0], window_size=mask[1:], return_lse=True, **kw)
    row = 0
    for s, q1 in enumerate(qs):
        t = tokens[s]
        got, got_lse = (o[row: row + t], lse[:, row: row + t]) if ragged else (o[s], lse[s])
        row += t
        want, want_lse, bound, lse_bound = ref.attend(q1, *c.tokens[s], scale or c.d ** -0.5, mask)
        ref.assert_within(f"o of sequence {s}", got, want, bound)
        empty = torch.isneginf(want_lse)
        assert torch.equal(torch.isneginf(got_lse), empty), f"sequence {s}"
        assert ((got_lse - want_lse).abs()[~empty] <= lse_bound[~empty]).all(), f"lse of sequence {s}"
    assert _lib.device_status() == 0
    return o, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,group", [(128, 128), (128, 64), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("lens,tokens,hq,hkv,page", [
    ([5, 0, 1, 300], [1] * 4, 8, 8, 16), ([33, 700, 64], [1] * 3, 32, 8, 0), ([257, 31], [1] * 2, 8, 1, 48), ([1000], [1], 16, 2, 64),
    ([90, 17, 200], [3] * 3, 12, 4, 128), ([64, 300, 20], [1, 4, 2], 32, 8, 16), ([140, 5], [20, 5], 6, 3, 256), ([40] * 9, [1] * 9, 5, 5, 16),
])
def test_attend(dtype, d, group, lens, tokens, hq, hkv, page):
    _attend(Cache(lens, hkv, d, group, dtype, page), tokens, hq)


@pytest.mark.parametrize("mask", [(0, -1, -1), (1, -1, 0), (2, 30, 0), (2, 5, 3), (1, 7, 2), (3, 100, 10)])
@pytest.mark.parametrize("tokens,hq", [(1, 8), (6, 8), (9, 4)])
def test_masks(mask, tokens, hq):
    # the last sequence has fewer keys than queries, so that rows see nothing
    _attend(Cache([200, 77, 3], 2, 64, 32, torch.bfloat16, 16), [tokens] * 3, hq, mask)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 200])
def test_splits(splits):
    _attend(Cache([3000, 1, 450], 8, 128, 128, torch.bfloat16, 16), [1] * 3, 32, num_splits=splits)


@pytest.mark.parametrize("batch,hkv", [(300, 1), (700, 8), (150, 3)])
def test_many_sequences(batch, hkv):
    _attend(Cache([1 + 37 * i % 90 for i in range(batch)], hkv, 64, 64, torch.float16, 16), [1] * batch, 4 * hkv)


def test_a_long_cache():
    _attend(Cache([40000], 1, 128, 64, torch.float16, 16), [1], 8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("groups", [1, 4])
def test_scales_of_any_size(dtype, groups):
    """Tokens whose scales differ by 2^20, in both orders, zero scales (constant groups) and huge and tiny queries."""
    top = 2.0 ** 12
    for seed, order in enumerate(("up", "down", "mixed")):
        c = Cache([400, 400], 2, 128, 128 // groups, dtype, 16, seed)
        for s in range(2):
            n = c.lens[s]
            f = 2.0 ** torch.linspace(-20, 0, n, device="cuda") if order != "mixed" else 2.0 ** (-20 * torch.rand(n, generator=_g(seed), device="cuda"))
            f = (f.flip(0) if order == "down" else f)[:, None, None, None] * top
            kc, kp, vc, vp = c.tokens[s]
            vp = (vp.float() * f).to(dtype)
            vp[5:40, :, :, 0] = 0
            kp[50:70, :, :, 0] = 0
            c.tokens[s] = [kc, kp, vc, vp]
            for part, x in zip(c.parts, c.tokens[s]):
                part.flatten(0, 1)[c.rows(s, 0, n)] = x
        q = [_normal(_g(9), 1, 16, 128, dtype=dtype) * a for a in (1.0, 2.0 ** 6)]
        q[0][:, 3:5] *= 2.0 ** -12
        q[0][:, 7] = 0
        _attend(c, [1, 1], 16, q=q)


def test_all_scales_zero_and_growing_scores():
    c = Cache([300], 1, 64, 64, torch.bfloat16, 16)
    c.tokens[0][3][..., 0] = 0
    grow = torch.linspace(0, 300, 300, device="cuda").to(torch.bfloat16)
    c.tokens[0][1][..., 0, 0] = 0
    c.tokens[0][1][..., 0, 1] = grow[:, None]  # key j is constant at j: scores grow without end
    for part, x in zip(c.parts, c.tokens[0]):
        part.flatten(0, 1)[c.rows(0, 0, 300)] = x
    _attend(c, [1], 8, q=[torch.ones(1, 8, 64, device="cuda", dtype=torch.bfloat16)])


def test_hidden_tokens_may_hold_anything():
    """NaN and infinite params of tokens that no query sees, inside the sequence."""
    c = Cache([200, 200], 2, 128, 64, torch.bfloat16, 16)
    for s in range(2):
        for i in (1, 3):
            c.tokens[s][i][:150] = torch.nan
            c.tokens[s][i][60:100] = torch.inf
        for part, x in zip(c.parts, c.tokens[s]):
            part.flatten(0, 1)[c.rows(s, 0, 200)] = x
        for i in (1, 3):
            c.tokens[s][i][:150] = 1.0  # (what the reference multiplies by zero)
    _attend(c, [3, 3], 8, (2, 40, 0))


def test_a_hidden_key_of_one_row_is_seen_by_another():
    c = Cache([50], 1, 64, 64, torch.float16, 16)
    for part in (1, 3):
        c.tokens[0][part][49] = torch.nan
    for part, x in zip(c.parts, c.tokens[0]):
        part.flatten(0, 1)[c.rows(0, 0, 50)] = x
    o, lse = ops.fmha_fwd_splitkv_int4(torch.ones(1, 3, 2, 64, device="cuda", dtype=torch.float16), *c.parts, seqlen_k=c.seqlen,
                                       block_table=c.table, causal=True, return_lse=True)
    assert torch.isfinite(o[0, :2]).all() and torch.isfinite(lse[..., :2]).all() and torch.isnan(o[0, 2]).all()


def test_pages_outside_the_pool_count_as_zeros():
    c = Cache([100, 60], 4, 64, 32, torch.bfloat16, 16)
    good = c.table.clone()
    c.table[0, 2], c.table[1, 0] = -7, c.parts[0].shape[0] + 5
    for s, lo in ((0, 32), (1, 0)):
        for x in c.tokens[s]:
            x[lo: lo + 16] = 0
    _attend(c, [1, 1], 16)
    k, v = ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, max_seqlen_k=100)
    assert (k[0, 32:48] == 0).all() and (v[1, :16] == 0).all() and (k[1, 16:60] != 0).any()
    before = [x.clone() for x in c.parts]
    new = _normal(_g(2), 2, 1, 4, 64, dtype=torch.bfloat16)
    ops.fmha_fwd_append_kv_int4(None, *c.parts, new, new, _i32([40, 3]), rope=RopeEnum.NONE, block_table=c.table)
    assert _lib.device_status() & INVALID
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, c.parts))
    ops.fmha_fwd_append_kv_int4(None, *c.parts, new, new, _i32([40, 3]), rope=RopeEnum.NONE, block_table=good)
    assert _lib.device_status() == 0 and not torch.equal(before[0], c.parts[0])


def test_lengths_behind_the_cache_are_cut():
    for page in (0, 16):
        c = Cache([64, 64], 2, 64, 64, torch.bfloat16, page)
        c.seqlen = _i32([5000, -3])
        c.tokens[1] = [x[:0] for x in c.tokens[1]]
        _attend(c, [1, 1], 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d,group", [(128, 128), (128, 32), (64, 64), (64, 32)])
@pytest.mark.parametrize("hq,hkv,page,rope,rotary_dim,axes", [
    (8, 2, 16, RopeEnum.HALF_ROTATED, None, 0), (5, 5, 0, RopeEnum.INTERLEAVED, None, 1), (6, 3, 24, RopeEnum.HALF_ROTATED, 32, 3),
    (4, 1, 16, RopeEnum.HALF_ROTATED, 20, 2), (8, 8, 1, RopeEnum.INTERLEAVED, 12, 4), (4, 4, 64, RopeEnum.NONE, None, 0),
])
@pytest.mark.parametrize("packed", [False, True])
def test_append(dtype, d, group, hq, hkv, page, rope, rotary_dim, axes, packed):
    g = _g(3)
    cached, new = [0, 37, 100], [3, 1, 8] if packed else [4, 4, 4]
    c = Cache([max(n, 1) for n in cached], hkv, d, group, dtype, page, room=120)
    c.seqlen = _i32(cached)
    total, pad = sum(new), 2 if packed else 0
    q, k, v = _normal(g, total + pad, hq, d, dtype=dtype), _normal(g, total + pad, hkv, d, dtype=dtype), _normal(g, total + pad, hkv, d, dtype=dtype)
    v[0] = 0.25  # constant groups
    k[1, :, : d // 2] = 0
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    width = (rotary_dim or d) // 2
    cos, sin = _normal(g, 130, width, dtype=dtype), _normal(g, 130, width, dtype=dtype)
    at = torch.cat([torch.arange(a, a + n, device="cuda") for a, n in zip(cached, new)])[None]
    pair_axis, kw = [0] * width, {}
    if axes:
        at = torch.randint(0, 130, (axes, total + pad), generator=g, device="cuda", dtype=torch.int32)
        kw["positions"] = at if axes > 1 else at[0].long()
        if axes > 1:
            sections = [width // axes] * (axes - 1)
            sections.append(width - sum(sections))
            kw["sections"] = sections
            pair_axis = [a for a, n in enumerate(sections) for _ in range(n)]
    if rope:
        kw.update(rotary_cos=cos, rotary_sin=sin)
    if packed:
        kw.update(cu_seqlens_q=_starts(new), cu_seqlens_knew=_starts(new))
        args = (q, k, v)
    else:
        args = tuple(x.view(3, 4, *x.shape[1:]) for x in (q, k, v))
        if axes > 1:
            kw["positions"] = at.view(axes, 3, 4)
    before = [x.clone() for x in c.parts]
    q_before = q.clone()
    got_q, got_k, got_v = ops.fmha_fwd_append_kv_int4(args[0], *c.parts, *args[1:], c.seqlen, rope=rope, block_table=c.table, return_kv=True, **kw)
    assert torch.equal(q, q_before) and _lib.device_status() == 0
    turn = (lambda x: ref.rotate(x[:total], cos, sin, at[:, :total], pair_axis, rope == RopeEnum.INTERLEAVED)) if rope else (lambda x: x[:total])
    assert torch.equal(got_q.flatten(0, -3)[:total], turn(q))
    for i, (x, held) in enumerate(((turn(k), got_k), (v[:total], got_v))):
        codes, scale, lo = ref.quantise(x, group)
        params = torch.stack([scale, lo], -1).to(dtype)
        assert torch.equal(held.flatten(0, -3)[:total], ref.values(ref.pack(codes), params).float().to(dtype))
        for s in range(3):
            rows = c.rows(s, cached[s], cached[s] + new[s])
            part = slice(cu[s], cu[s + 1])
            before[2 * i].flatten(0, 1)[rows] = ref.pack(codes[part])
            before[2 * i + 1].flatten(0, 1)[rows] = params[part]
    for a, b in zip(before, c.parts):  # the written rows, and no other (which zero is the least of +0 and -0 is nobody's business)
        assert torch.equal(a, b) if a.dtype == torch.uint8 else torch.equal(torch.nan_to_num(a, 12345.0), torch.nan_to_num(b, 12345.0))
    if packed:
        assert all((x[total:] == 0).all() for x in (got_q, got_k, got_v))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_codes_next_to_a_border(dtype):
    """Values half way between two codes, a step beside it, tiny and huge ranges: the nearer code, ties to even."""
    rows = []
    for scale in (1.0, 2.0 ** -9, 2.0 ** -20, 2.0 ** 9, 3.0, 0.1015625):
        base = torch.zeros(32, dtype=torch.float64)
        base[1] = 15 * scale
        base[2:17] = (torch.arange(15, dtype=torch.float64) + 0.5) * scale
        base[17:31] = (torch.arange(1, 15, dtype=torch.float64)) * scale
        x = base.to(dtype)
        near = torch.nextafter(x.float(), torch.full((32,), torch.inf)).to(dtype)
        rows += [x, near, -x, torch.cat([x[:2], (x[2:].view(torch.int16) + 1).view(dtype)]), x + x[1]]
    x = torch.stack(rows).cuda()
    extreme = torch.finfo(dtype).max / 32
    more = torch.stack([torch.linspace(-extreme, extreme, 32), torch.linspace(0, torch.finfo(dtype).tiny, 32), torch.full((32,), 7.0),
                        torch.cat([torch.zeros(31), torch.tensor([torch.finfo(dtype).smallest_normal / 64])]),
                        torch.linspace(-1, 1, 32) ** 9]).to(dtype).cuda()
    x = torch.cat([x, more])
    n = x.shape[0]
    x = x[:, None, :].repeat(1, 1, 2)
    c = Cache([0], 1, 64, 32, dtype, 0, room=n)
    c.seqlen = _i32([0])
    ops.fmha_fwd_append_kv_int4(None, *c.parts, x[None], x[None].flip(-1).contiguous(), c.seqlen, rope=RopeEnum.NONE)
    for i, y in ((0, x), (2, x.flip(-1))):
        codes, scale, lo = ref.quantise(y, 32)
        assert torch.equal(c.parts[i + 1][0], torch.stack([scale, lo], -1).to(dtype))
        assert torch.equal(c.parts[i][0], ref.pack(codes))


def test_what_is_not_finite_reads_back_as_nan():
    c = Cache([0], 1, 64, 32, torch.bfloat16, 0, room=4)
    x = torch.ones(1, 3, 1, 64, device="cuda", dtype=torch.bfloat16)
    x[0, 0, 0, 3], x[0, 1, 0, 40], x[0, 2, 0, 5] = torch.nan, torch.inf, -torch.inf
    k, v = ops.fmha_fwd_append_kv_int4(None, *c.parts, x, x, _i32([0]), rope=RopeEnum.NONE, return_kv=True)[1:]
    read = ops.fmha_read_kv_int4(*c.parts, _i32([3]), max_seqlen_k=4)
    for y in (k, v, read[0][:, :3], read[1][:, :3]):
        assert torch.isnan(y[0, 0, 0, :32]).all() and torch.isnan(y[0, 1, 0, 32:]).all() and torch.isnan(y[0, 2, 0, :32]).all()
        assert (y[0, 0, 0, 32:] == 1).all() and (y[0, 1, 0, :32] == 1).all()
    assert (read[0][0, 3] == 0).all()


def test_tokens_that_do_not_fit_are_skipped():
    for page in (0, 16):
        c = Cache([30, 32], 2, 64, 64, torch.float16, page, room=32)
        new = _normal(_g(0), 2, 4, 2, 64, dtype=torch.float16)
        before = [x.clone() for x in c.parts]
        ops.fmha_fwd_append_kv_int4(None, *c.parts, new, new, _i32([30, -9]), rope=RopeEnum.NONE, block_table=c.table)
        assert _lib.device_status() & INVALID
        codes, _, _ = ref.quantise(new[0, :2], 64)
        before[0].flatten(0, 1)[c.rows(0, 30, 32)] = before[2].flatten(0, 1)[c.rows(0, 30, 32)] = ref.pack(codes)
        assert torch.equal(before[0], c.parts[0]) and torch.equal(before[2], c.parts[2])


def test_positions_outside_the_tables_turn_by_nan():
    c = Cache([0], 1, 64, 64, torch.bfloat16, 0, room=8)
    x = torch.ones(1, 4, 1, 64, device="cuda", dtype=torch.bfloat16)
    t = torch.ones(5, 32, device="cuda", dtype=torch.bfloat16)
    for rope in (RopeEnum.HALF_ROTATED, RopeEnum.INTERLEAVED):
        q = ops.fmha_fwd_append_kv_int4(x, *c.parts, x, x, _i32([0]), t, t, rope=rope, positions=_i32([4, 5, -1, 2 ** 31 - 1]))
        assert torch.isfinite(q[0, 0]).all() and torch.isnan(q[0, 1:]).all()
        q = ops.fmha_fwd_append_kv_int4(x, *c.parts, x, x, _i32([3]), t, t, rope=rope)
        assert torch.isfinite(q[0, :2]).all() and torch.isnan(q[0, 2:]).all()


def test_fewer_queries_than_new_tokens():
    c = Cache([10, 3], 2, 64, 64, torch.bfloat16, 16, room=32)
    g = _g(4)
    new, q = _normal(g, 2, 6, 2, 64, dtype=torch.bfloat16), _normal(g, 2, 2, 4, 64, dtype=torch.bfloat16)
    cos, sin = _normal(g, 32, 32, dtype=torch.bfloat16), _normal(g, 32, 32, dtype=torch.bfloat16)
    at = torch.randint(0, 32, (2, 6), generator=g, device="cuda", dtype=torch.int32)
    for pos, where in ((None, torch.stack([torch.arange(10, 16), torch.arange(3, 9)]).cuda()), (at, at)):
        got = ops.fmha_fwd_append_kv_int4(q, *c.parts, new, new, c.seqlen, cos, sin, rope=RopeEnum.HALF_ROTATED, positions=pos, block_table=c.table)
        want = ref.rotate(q.flatten(0, 1), cos, sin, where[:, 4:].flatten()[None], [0] * 32, False)
        assert torch.equal(got.flatten(0, 1), want)


@pytest.mark.parametrize("d,group,hkv,page", [(128, 128, 8, 16), (64, 32, 3, 0), (128, 32, 1, 7)])
def test_read(d, group, hkv, page):
    c = Cache([50, 0, 1, 131], hkv, d, group, torch.bfloat16, page)
    want = [torch.cat([ref.values(t[i], t[i + 1]).float().to(torch.bfloat16) for t in c.tokens]) for i in (0, 2)]
    got = ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, cu_seqlens_k=_starts(c.lens), total_k=182)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, cu_seqlens_k=_starts([52, 0, 1, 129]), total_k=190)
    for a, b in zip(got, want):
        assert torch.equal(a[:50], b[:50]) and (a[50:52] == 0).all() and torch.equal(a[52:182], b[50:180]) and (a[182:] == 0).all()
    got = ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, max_seqlen_k=140)
    for a, b in zip(got, want):
        row = 0
        for s, n in enumerate(c.lens):
            assert torch.equal(a[s, :n], b[row: row + n]) and (a[s, n:] == 0).all()
            row += n


def test_cache_batch_idx():
    c = Cache([40, 90, 20], 2, 64, 64, torch.bfloat16, 0)
    order = torch.tensor([2, 0], device="cuda")
    q = _normal(_g(1), 2, 1, 4, 64, dtype=torch.bfloat16)
    lens = _i32([20, 40])
    o = ops.fmha_fwd_splitkv_int4(q, *c.parts, seqlen_k=lens, cache_batch_idx=order, causal=True)
    picked = [x[order].contiguous() for x in c.parts]
    assert torch.equal(o, ops.fmha_fwd_splitkv_int4(q, *picked, seqlen_k=lens, causal=True))
    k = ops.fmha_read_kv_int4(*c.parts, lens, cache_batch_idx=order, max_seqlen_k=40)[0]
    assert torch.equal(k, ops.fmha_read_kv_int4(*picked, lens, max_seqlen_k=40)[0])
    ops.fmha_fwd_append_kv_int4(None, *c.parts, q[:, :, :2].contiguous(), q[:, :, :2].contiguous(), lens, rope=RopeEnum.NONE, cache_batch_idx=order)
    ops.fmha_fwd_append_kv_int4(None, *picked, q[:, :, :2].contiguous(), q[:, :, :2].contiguous(), lens, rope=RopeEnum.NONE)
    assert all(torch.equal(a[order].view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c.parts, picked))


@pytest.mark.parametrize("dtype,d,group,page", [(torch.bfloat16, 128, 64, 16), (torch.float16, 64, 32, 0)])
def test_a_conversation(dtype, d, group, page):
    """A prompt is written, two tokens are decoded, and the next chunk attends to the cache read back: every step against 64 bits."""
    g, hq, hkv, prompt, room = _g(5), 8, 2, [70, 33], 140
    kp, vp = (ops.int4_cache(2 * -(-room // page) if page else 2, page or room, hkv, d, group=group, dtype=dtype) for _ in range(2))
    parts = [kp[0], kp[1], vp[0], vp[1]]
    table = torch.randperm(kp[0].shape[0], generator=g, device="cuda").to(torch.int32).view(2, -1).contiguous() if page else None
    cos, sin = (t.to(dtype) for t in _angles(200, d // 2))
    lens, held = [0, 0], [[], []]
    for step, new in enumerate((prompt, [1, 1], [1, 1], [40, 25])):
        total = sum(new)
        q, k, v = (_normal(g, total, h, d, dtype=dtype) for h in (hq, hkv, hkv))
        cu = _starts(new)
        q, kh, vh = ops.fmha_fwd_append_kv_int4(q, *parts, k, v, _i32(lens), cos, sin, rope=RopeEnum.HALF_ROTATED, block_table=table, cu_seqlens_q=cu,
                                                cu_seqlens_knew=cu, return_kv=True)
        lens = [a + n for a, n in zip(lens, new)]
        seqlen = _i32(lens)
        k_all, v_all = ops.fmha_read_kv_int4(*parts, seqlen, block_table=table, cu_seqlens_k=_starts(lens), total_k=sum(lens))
        for s in range(2):
            part = slice(int(cu[s]), int(cu[s + 1]))
            held[s].append((kh[part], vh[part]))
        assert torch.equal(k_all, torch.cat([x for s in range(2) for x, _ in held[s]]))
        assert torch.equal(v_all, torch.cat([x for s in range(2) for _, x in held[s]]))
        if max(new) > 1:
            o = ops.fmha_fwd_var_len(q, k_all, v_all, cu, _starts(lens), max(new), max(lens), causal=True)
            tolerance = 2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -9  # K, V, P and O each rounded: 4 half steps of values up to 4
        else:
            o = ops.fmha_fwd_splitkv_int4(q, *parts, seqlen_k=seqlen, block_table=table, cu_seqlens_q=cu, max_seqlen_q=1, causal=True)
            tolerance = None
        for s in range(2):
            rows = (table[s].long()[torch.arange(lens[s], device="cuda") // page] * page + torch.arange(lens[s], device="cuda") % page) if page \
                else s * room + torch.arange(lens[s], device="cuda")
            part = slice(int(cu[s]), int(cu[s + 1]))
            want, _, bound, _ = ref.attend(q[part], *(x.flatten(0, 1)[rows] for x in parts), d ** -0.5, (2, -1, 0))
            if tolerance:
                assert ((o[part] - want).abs() <= 4 * tolerance).all()
            else:
                ref.assert_within(f"step {step}", o[part], want, bound)
    assert _lib.device_status() == 0


def _angles(rows, half):
    a = torch.arange(rows, device="cuda")[:, None] * 10000.0 ** (-torch.arange(half, device="cuda") / half)
    return a.cos(), a.sin()


def _serve(c, q, new, seqlen, cos, sin):
    q = ops.fmha_fwd_append_kv_int4(q, *c.parts, new, new, seqlen, cos, sin, rope=RopeEnum.HALF_ROTATED, block_table=c.table)
    o = ops.fmha_fwd_splitkv_int4(q, *c.parts, seqlen_k=seqlen + 1, block_table=c.table, causal=True)
    return (o,) + ops.fmha_read_kv_int4(*c.parts, seqlen + 1, block_table=c.table, max_seqlen_k=310)


def test_captured_and_on_two_streams():
    g = _g(6)
    cos, sin = (t.to(torch.bfloat16) for t in _angles(400, 64))
    calls = []
    for seed in range(2):
        c = Cache([300, 17, 160], 4, 128, 64, torch.bfloat16, 16, seed, room=320)
        calls.append((c, _normal(g, 3, 1, 16, 128, dtype=torch.bfloat16), _normal(g, 3, 1, 4, 128, dtype=torch.bfloat16), c.seqlen, cos, sin))
    want = [[x.clone() for x in _serve(*a)] for a in calls]
    graphs = []
    for a in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, _serve(*a)))
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(3):  # both graphs at once
        for (graph, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (_, got), w in zip(graphs, want):
        assert all(torch.equal(x, y) for x, y in zip(got, w))
    got = []
    for a, s in zip(calls, streams):  # both eager, at once
        with torch.cuda.stream(s):
            got.append([_serve(*a) for _ in range(5)][-1])
    torch.cuda.synchronize()
    for x, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, w))
    assert _lib.device_status() == 0


def test_rows_behind_the_last_sequence_are_left():
    c = Cache([40, 30], 2, 64, 64, torch.bfloat16, 16)
    q = _normal(_g(0), 7, 4, 64, dtype=torch.bfloat16)
    lse = torch.full((4, 3, 7), torch.nan, device="cuda")
    acc = torch.full((4, 3, 7, 64), torch.nan, device="cuda")
    cu = _starts([2, 1])
    rc = _lib.lib().FmhaFwdSplitKVInt4(q.data_ptr(), *(x.data_ptr() for x in c.parts), lse.data_ptr(), acc.data_ptr(), cu.data_ptr(),
                                       c.seqlen.data_ptr(), c.table.data_ptr(), 0, 2, 7, 2, 4, 2, 64, 64, 3, c.table.shape[1], 16, c.parts[0].shape[0],
                                       0.0, -1, 0, 2, torch.cuda.current_stream().cuda_stream, 4)
    assert rc == 0
    assert torch.isnan(lse[..., 3:]).all() and torch.isnan(acc[:, :, 3:]).all() and not torch.isnan(lse[..., :3]).any()


def test_the_binding_and_python_agree(monkeypatch):
    from flashck_b200.ops import fmha
    assert fmha._native()
    c = Cache([90, 17], 2, 64, 32, torch.float16, 16, room=128)
    q, new = _normal(_g(1), 2, 2, 4, 64, dtype=torch.float16), _normal(_g(2), 2, 2, 2, 64, dtype=torch.float16)
    cos, sin = (t.to(torch.float16) for t in _angles(200, 32))
    pos = torch.randint(0, 200, (3, 2, 2), generator=_g(3), device="cuda", dtype=torch.int32)

    def all_calls():
        out = list(ops.fmha_fwd_append_kv_int4(q, *c.parts, new, new, c.seqlen, cos, sin, rope=2, positions=pos, sections=(8, 12, 12),
                                               interleaved_sections=True, block_table=c.table, return_kv=True))
        out.append(ops.fmha_fwd_append_kv_int4(q, *c.parts, new, new, c.seqlen, cos, sin, rope=1, rotary_dim=64, block_table=c.table))
        assert ops.fmha_fwd_append_kv_int4(None, *c.parts, new, new, c.seqlen, rope=0, block_table=c.table) is None
        out += ops.fmha_fwd_splitkv_int4(q, *c.parts, seqlen_k=c.seqlen, block_table=c.table, causal=True, return_lse=True)
        out.append(ops.fmha_fwd_splitkv_int4(q.flatten(0, 1), *c.parts, seqlen_k=c.seqlen, block_table=c.table, cu_seqlens_q=_starts([3, 1]),
                                             max_seqlen_q=3, window_size=(20, 0)))
        out += ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, max_seqlen_k=50)
        out += ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, cu_seqlens_k=_starts([90, 17]), total_k=107)
        return out

    a = all_calls()
    monkeypatch.setattr(fmha, "_NATIVE", False)
    assert all(torch.equal(x, y) for x, y in zip(a, all_calls()))


def test_equal_calls_give_equal_bits():
    """Many short segments and both ways in which the teams of warps share the rows; a read of a stage too early shows as a difference."""
    for tokens, hq, group in (([1] * 40, 32, 128), ([1] * 40, 64, 64), ([1, 4] * 20, 32, 64), ([4] * 40, 32, 32)):
        c = Cache([1 + 131 * i % 700 for i in range(40)], 8, 128, group, torch.bfloat16, 16)
        c.seqlen = torch.maximum(c.seqlen, _i32(tokens))
        q = _normal(_g(3), sum(tokens), hq, 128, dtype=torch.bfloat16)
        call = lambda: ops.fmha_fwd_splitkv_int4(q, *c.parts, seqlen_k=c.seqlen, block_table=c.table, cu_seqlens_q=_starts(tokens),  # noqa: E731
                                                 max_seqlen_q=max(tokens), causal=True, return_lse=True)
        first = call()
        for _ in range(60):
            again = call()
            assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(first, again))
    assert _lib.device_status() == 0


def test_pools_of_more_than_4_gigabytes():
    """The pages in use lie at the end of pools whose offsets pass 32 bits."""
    pages, page, hkv, d = 600000, 128, 1, 128  # 4.9e9 bytes of codes, each
    parts = []
    for _ in range(2):
        parts += [torch.empty(pages, page, hkv, d // 2, dtype=torch.uint8, device="cuda"), torch.empty(pages, page, hkv, 1, 2, dtype=torch.bfloat16, device="cuda")]
    table = _i32([[pages - 1, pages - 7, pages - 3]])
    g = _g(0)
    k, v, q = (_normal(g, 1, 300, h, d, dtype=torch.bfloat16) for h in (1, 1, 8))
    held = ops.fmha_fwd_append_kv_int4(q, *parts, k, v, _i32([0]), rope=RopeEnum.NONE, block_table=table, return_kv=True)[1:]
    assert all(torch.equal(a, b) for a, b in zip(held, ops.fmha_read_kv_int4(*parts, _i32([300]), block_table=table, max_seqlen_k=300)))
    o = ops.fmha_fwd_splitkv_int4(q[:, :1].contiguous(), *parts, seqlen_k=_i32([300]), block_table=table)
    rows = (table[0].long()[torch.arange(300, device="cuda") // page] * page + torch.arange(300, device="cuda") % page)
    want, _, bound, _ = ref.attend(q[0, :1], *(x.flatten(0, 1)[rows] for x in parts), d ** -0.5, (0, -1, -1))
    ref.assert_within("o", o[0], want, bound)


def test_the_module():
    from flashck_b200.nn import FlashAttention
    layer = FlashAttention(8, 64, 2, causal=True)
    c = Cache([40, 9], 2, 64, 32, torch.float16, 16, room=64)
    q, new = _normal(_g(1), 2, 1, 8, 64, dtype=torch.float16), _normal(_g(2), 2, 1, 2, 64, dtype=torch.float16)
    cos, sin = (t.to(torch.float16) for t in _angles(100, 32))
    turned = layer.append_kv_int4(q, *c.parts, new, new, c.seqlen, (cos, sin), block_table=c.table)
    assert torch.equal(turned, ops.fmha_fwd_append_kv_int4(q, *c.parts, new, new, c.seqlen, cos, sin, block_table=c.table))
    o = layer.forward_int4(turned, *c.parts, c.seqlen + 1, block_table=c.table)
    assert torch.equal(o, ops.fmha_fwd_splitkv_int4(turned, *c.parts, seqlen_k=c.seqlen + 1, block_table=c.table, causal=True))
    with pytest.raises(ValueError, match="must end in"):
        layer.forward_int4(q[..., :4, :].contiguous(), *c.parts, c.seqlen, block_table=c.table)


def test_calls_that_do_not_fit_are_refused():
    c = Cache([40, 9], 2, 64, 32, torch.float16, 16, room=64)
    q, new = _normal(_g(1), 2, 1, 8, 64, dtype=torch.float16), _normal(_g(2), 2, 1, 2, 64, dtype=torch.float16)
    attend = lambda q=q, parts=c.parts, **kw: ops.fmha_fwd_splitkv_int4(q, *parts, **{**dict(seqlen_k=c.seqlen, block_table=c.table), **kw})  # noqa: E731
    append = lambda k=new, v=new, q=q, **kw: ops.fmha_fwd_append_kv_int4(q, *c.parts, k, v, c.seqlen, **{**dict(rope=0, block_table=c.table), **kw})  # noqa: E731
    kc, kp, vc, vp = c.parts
    cos = torch.ones(70, 32, device="cuda", dtype=torch.float16)
    cases = [
        (lambda: attend(q.bfloat16()), TypeError), (lambda: attend(q[:1]), ValueError), (lambda: attend(q[..., :32].contiguous()), ValueError),
        (lambda: attend(q[:, :, :3].contiguous()), ValueError), (lambda: attend(seqlen_k=c.seqlen[:1]), ValueError),
        (lambda: attend(block_table=c.table[:1]), ValueError), (lambda: attend(block_table=None, parts=[x[:1] for x in c.parts]), ValueError),
        (lambda: attend(parts=[kc, kp, vc[:1], vp]), ValueError), (lambda: attend(parts=[kc, kp[:, :8].contiguous(), vc, vp]), ValueError),
        (lambda: attend(parts=[kc, kp.bfloat16(), vc, vp]), TypeError), (lambda: attend(parts=[kc.int(), kp, vc, vp]), TypeError),
        (lambda: attend(parts=[kc[..., :16].contiguous(), kp, vc[..., :16].contiguous(), vp]), ValueError),
        (lambda: attend(parts=[kc, kp.transpose(0, 1), vc, vp]), ValueError), (lambda: attend(cu_seqlens_q=_starts([1, 1])), ValueError),
        (lambda: attend(q.flatten(0, 1), cu_seqlens_q=_starts([2])), ValueError), (lambda: attend(seqlen_k=None), TypeError),
        (lambda: attend(parts=[x.view(-1, 8, *x.shape[2:]) for x in c.parts]), ValueError), (lambda: attend(num_splits=5000), RuntimeError),
        (lambda: attend(torch.cat([q.flatten(), q.flatten()])[4: 4 + q.numel()].view(q.shape)), ValueError),
        (lambda: append(k=new[..., :32].contiguous()), ValueError), (lambda: append(v=new[:, :, :1].contiguous()), ValueError),
        (lambda: append(q=q[:1]), ValueError), (lambda: append(cu_seqlens_knew=_starts([1, 1])), ValueError), (lambda: append(rope=1), ValueError),
        (lambda: append(rope=1, rotary_cos=cos, rotary_sin=cos[:, :8].contiguous()), ValueError),
        (lambda: append(rope=1, rotary_cos=cos, rotary_sin=cos, rotary_dim=32), ValueError),
        (lambda: append(rope=1, rotary_cos=cos.bfloat16(), rotary_sin=cos.bfloat16()), TypeError),
        (lambda: append(rope=1, rotary_cos=cos, rotary_sin=cos, positions=_i32([1, 2, 3])), ValueError),
        (lambda: append(rope=1, rotary_cos=cos, rotary_sin=cos, positions=_i32([[1, 2], [3, 4]])), ValueError),
        (lambda: append(rope=1, rotary_cos=cos, rotary_sin=cos, positions=_i32([[1, 2], [3, 4]]), sections=(16, 17)), ValueError),
        (lambda: append(rope=1, rotary_cos=cos, rotary_sin=cos, positions=torch.ones(2, device="cuda")), TypeError),
        (lambda: append(positions=_i32([1, 2])), ValueError), (lambda: append(rope=5, rotary_cos=cos, rotary_sin=cos), RuntimeError),
        (lambda: ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table), ValueError),
        (lambda: ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, max_seqlen_k=-1), ValueError),
        (lambda: ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, total_k=5), ValueError),
        (lambda: ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, cu_seqlens_k=_starts([5]), total_k=5), ValueError),
        (lambda: ops.apply_rotary(q, None, _i32([0, 1, 2]), cos, cos), ValueError), (lambda: ops.apply_rotary(q, new.bfloat16(), _i32([0, 1]), cos, cos), TypeError),
        (lambda: ops.apply_rotary(q, None, _i32([0, 1]), cos, cos, rope=0), ValueError),
        (lambda: ops.apply_rotary(q[..., :32].contiguous(), None, _i32([0, 1]), cos, cos), ValueError),
        (lambda: ops.apply_rotary(q[..., :60].contiguous(), None, _i32([0, 1]), cos[:, :30].contiguous(), cos[:, :30].contiguous()), RuntimeError),
        (lambda: ops.apply_rotary(q.transpose(1, 2), None, _i32([0, 1]), cos, cos), ValueError),
    ]
    for i, (call, error) in enumerate(cases):
        with pytest.raises(error):
            call()
            pytest.fail(f"case {i} was taken")
    # nothing to do is no error
    assert attend(q[:, :0]).shape == (2, 0, 8, 64)
    k, v = ops.fmha_read_kv_int4(*c.parts, c.seqlen, block_table=c.table, max_seqlen_k=0)
    assert k.shape == (2, 0, 2, 64)
    assert append(k=new[:, :0].contiguous(), v=new[:, :0].contiguous(), q=None) is None


@pytest.mark.parametrize("mask", [(0, -1, -1), (1, -1, 0), (2, -1, 0), (2, 30, 0), (2, 5, 3), (3, 100, 10)])
@pytest.mark.parametrize("tokens,hq,hkv", [(2, 4, 2), (4, 3, 3), (3, 1, 1), (5, 1, 1), (8, 2, 2)])
def test_masks_of_few_rows(mask, tokens, hq, hkv):
    """Several tokens and up to 4, and up to 8 rows per kv head."""
    _attend(Cache([200, 77, 3], hkv, 128, 64, torch.bfloat16, 16), [tokens] * 3, hq, mask)


def test_as_many_sequences_as_are_taken():
    """The schedule of 8192 sequences leaves room for few stages.  A split per sequence makes a sequence's bits its own."""
    lens = [1 + 53 * i % 70 for i in range(8192)]
    c = Cache([4096 * 16], 2, 128, 32, torch.bfloat16, 0)  # (values only: the pools are laid out below)
    parts = [x.view(4096, 16, *x.shape[2:]) for x in c.parts]
    table = torch.randint(0, 4096, (8192, 5), generator=_g(0), device="cuda", dtype=torch.int32)
    for hq in (2, 16):
        q = _normal(_g(1), 8192, 1, hq, 128, dtype=torch.bfloat16)
        call = lambda s: ops.fmha_fwd_splitkv_int4(q[s], *parts, seqlen_k=_i32(lens[s]), block_table=table[s], num_splits=1)  # noqa: E731
        whole = call(slice(0, 8192))
        assert torch.isfinite(whole).all()
        for i in range(0, 8192, 1024):
            assert torch.equal(whole[i: i + 1024], call(slice(i, i + 1024)))
    with pytest.raises(RuntimeError, match="8192"):
        ops.fmha_fwd_splitkv_int4(torch.cat([q, q[:1]]), *parts, seqlen_k=_i32(lens + [1]), block_table=torch.cat([table, table[:1]]))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("splits", [0, 1, 2, 3, 40, 128])
@pytest.mark.parametrize("d,group", [(64, 32), (128, 128)])
def test_batches_of_few_and_many_rows(d, group, splits):
    """Sequences of up to 8 rows per kv head beside ones of more, whose tiles cost more: pieces that begin and end at any unit of a tile."""
    lens = [3000, 1, 0, 33, 700, 31, 32, 2000, 64, 5, 257, 1500]
    tokens = [1, 4, 3, 3, 2, 4, 1, 4, 0, 3, 2, 3]
    _attend(Cache(lens, 2, d, group, torch.float16, 16), tokens, 8, num_splits=splits)
    _attend(Cache([40 + 29 * i for i in range(70)], 8, d, group, torch.bfloat16, 0), [1 + i * i % 4 for i in range(70)], 32, num_splits=splits)


@pytest.mark.parametrize("splits", [0, 2, 30, 128])
@pytest.mark.parametrize("tokens,hq", [([1] * 14, 16), ([1, 4, 3, 3, 2, 4, 1, 4, 1, 3, 2, 3, 1, 4], 64)])
def test_long_and_short_sequences_together(tokens, hq, splits):
    """Enough work that a sequence's beginning counts in the split of the work: ones of one tile, of none and of hundreds next to one another."""
    lens = [9000, 1, 0, 32, 11000, 33, 12001, 2, 20000, 31, 64, 15000, 700, 6]
    _attend(Cache(lens, 16, 64, 64, torch.bfloat16, 16), tokens, hq, num_splits=splits)


def test_a_schedule_past_32_bits_is_refused():
    parts = [torch.zeros(1, 1 << 16, 1, n, dtype=t, device="cuda") for n, t in ((32, torch.uint8), (2, torch.float16)) * 2]
    parts = [x if x.dtype == torch.uint8 else x.view(1, 1 << 16, 1, 1, 2) for x in parts]
    table = torch.zeros(1024, 1 << 12, dtype=torch.int32, device="cuda")
    q = torch.zeros(1024, 1, 1, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="schedule"):
        ops.fmha_fwd_splitkv_int4(q, *parts, seqlen_k=_i32([1] * 1024), block_table=table)
    assert _lib.device_status() == 0
