"""Serving from a key/value cache held in 4 bits, and the rotation of queries and keys, as measurable cases.

A case is a dict of plain values.  ``op`` names the path:

* ``attend`` -- ``fmha_fwd_splitkv_int4``: one new token per sequence, or a few, against a paged or contiguous 4-bit cache
* ``append`` -- ``fmha_fwd_append_kv_int4``: queries and new keys rotated, new keys and values quantised as they are written; the
  values that the cache then holds for them are returned
* ``read``   -- ``fmha_read_kv_int4``: the cache back as 16-bit keys and values, packed, as a prefill over it takes them
* ``rotary`` -- ``apply_rotary``: queries and keys rotated by the positions of their tokens along one or several axes
* ``train``  -- ``apply_rotary_autograd`` and its backward

A group of ``group`` neighbouring channels of a token's head is held as ``lo + scale * code``: lo its least value, scale
``(hi - lo) / 15`` in the element type, code 0..15 the nearest, ties to even; byte j of a row holds channel 2j in its low and 2j + 1 in
its high four bits.  ``run`` computes the operators in elementary torch operations, or with ``own`` through ``flashck_b200.ops``.
Lengths are fixed by ``lens_seed``, so that the work of a case does not depend on the seed of its values.
"""
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_MOST_FLOPS, _MOST_BYTES = 7e10, 2.4e9  # of a drawn case: what the largest listed ones take


def _attend(name, dtype, batch, hq, hkv, d, group, lo, hi, **more):
    case = dict(name=name, op="attend", dtype=dtype, batch=batch, hq=hq, hkv=hkv, d=d, group=group, lo=lo, hi=hi, page=16, window=-1,
                tokens_lo=1, tokens_hi=1, lens_seed=1)
    case.update(more)
    return case


def _append(name, dtype, batch, hq, hkv, d, group, lo, hi, new_lo, new_hi, **more):
    case = dict(name=name, op="append", dtype=dtype, batch=batch, hq=hq, hkv=hkv, d=d, group=group, lo=lo, hi=hi, new_lo=new_lo,
                new_hi=new_hi, page=16, rope="half", axes=0, lens_seed=1)
    case.update(more)
    return case


def _read(name, dtype, batch, hkv, d, group, lo, hi, **more):
    case = dict(name=name, op="read", dtype=dtype, batch=batch, hq=hkv, hkv=hkv, d=d, group=group, lo=lo, hi=hi, page=16, lens_seed=1)
    case.update(more)
    return case


def _rotary(name, dtype, batch, hq, hkv, d, tokens, **more):
    case = dict(name=name, op="rotary", dtype=dtype, batch=batch, hq=hq, hkv=hkv, d=d, tokens=tokens, rope="half", axes=3, rotary_dim=d)
    case.update(more)
    return case


def listed():
    return [
        # one conversation: latency
        _attend("attend_single", "bf16", 1, 32, 8, 128, 128, 2000, 4000, lens_seed=5),
        # a full serving batch, one token each
        _attend("attend_batch", "bf16", 64, 32, 8, 128, 128, 1024, 32768, lens_seed=4321),
        # very long contexts, scales of half heads
        _attend("attend_long", "bf16", 4, 64, 8, 128, 64, 524288, 524288, page=64),
        # speculative decoding: one to four drafted tokens per sequence, contiguous caches of head dim 64, scales of 32 channels
        _attend("attend_drafted", "fp16", 48, 32, 8, 64, 32, 300, 8000, page=0, tokens_lo=1, tokens_hi=4, lens_seed=77),
        # the write of a decode step
        _append("append_step", "bf16", 32, 32, 8, 128, 128, 2048, 16384, 1, 1, lens_seed=99),
        # whole prompts written as they are prefilled
        _append("append_prompts", "bf16", 16, 32, 8, 128, 64, 0, 0, 512, 4096, lens_seed=1234),
        # prompts with images: positions along time, height and width; a chunk behind what is cached
        _append("append_images", "fp16", 6, 16, 2, 64, 32, 1024, 4096, 128, 768, axes=3, page=64, lens_seed=21),
        # what a chunked prefill of six conversations reads back
        _read("read_chunked", "bf16", 6, 8, 128, 128, 1024, 16384, lens_seed=21),
        # a few short contiguous caches, head dim 64
        _read("read_short", "fp16", 5, 4, 64, 32, 1, 300, page=0, lens_seed=7),
        # the smallest call: two short prompts, plain positions, neighbouring pairs
        _rotary("rotary_tiny", "fp16", 2, 8, 8, 64, 128, axes=1, rope="pairs"),
        # prefill of an image prompt
        _rotary("rotary_images", "bf16", 1, 32, 8, 128, 16384),
        # a layer of a training step, forward and backward, an odd length
        _rotary("rotary_train", "bf16", 2, 32, 8, 128, 4095, op="train"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_once(rng):
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 16), (8, 8), (16, 2), (12, 4), (8, 1)])
    dtype, d, seed = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([128, 128, 64]), rng.randrange(1 << 20)
    group, page = rng.choice([g for g in (32, 64, 128) if g <= d]), rng.choice([0, 16, 16, 48, 64, 128])
    rope = rng.choice(["half", "half", "pairs"])
    kind = rng.choice(["attend", "attend", "attend", "append", "append", "read", "rotary", "train"])
    if kind == "attend":
        lo, tokens = _log_int(rng, 1, 65536), rng.choice([1, 1, 1, 2, 5, 8, 16])
        case = _attend("", dtype, _log_int(rng, 1, 256), hq, hkv, d, group, lo, lo * rng.randint(1, 8), page=page, lens_seed=seed,
                       tokens_lo=rng.choice([1, tokens]), tokens_hi=tokens, window=rng.choice([-1, -1, -1, _log_int(rng, 16, 4096)]))
    elif kind == "append":
        new = rng.choice([1, _log_int(rng, 1, 2048)])
        case = _append("", dtype, _log_int(rng, 1, 128), hq, hkv, d, group, 0, _log_int(rng, 1, 8192), rng.choice([1, new]), new,
                       page=page, rope=rope, axes=rng.choice([0, 0, 1, 2, 3]), lens_seed=seed)
    elif kind == "read":
        lo = _log_int(rng, 1, 8192)
        case = _read("", dtype, _log_int(rng, 1, 128), hkv, d, group, rng.choice([0, lo]), lo * rng.randint(1, 8), page=page, lens_seed=seed)
    else:
        case = _rotary("", dtype, rng.choice([1, 2, 5]), hq, hkv, d, _log_int(rng, 1, 16384), op=kind, rope=rope, axes=rng.choice([1, 2, 3]),
                       rotary_dim=rng.choice([d, d, d // 2]))
    del case["name"]
    return case


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        rows = 4 if case["op"] != "attend" else case["tokens_hi"] * case["hq"] // case["hkv"]
        if w["flops"] * max(1, rows // 8) <= _MOST_FLOPS and 0 < w["bytes"] <= _MOST_BYTES and case["batch"] * case.get("hi", 1) <= 1 << 22:
            return case


# ---- sizes of a case -----------------------------------------------------------------------------------------------
def _drawn_lens(n, lo, hi, seed):
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(n)]


def _lens(case):
    """(new tokens, cached tokens) of every sequence; the cached ones of ``attend`` include the new, those of ``append`` do not."""
    b, seed = case["batch"], case.get("lens_seed", 0)
    if case["op"] in ("rotary", "train"):
        return [case["tokens"]] * b, [0] * b
    cached = _drawn_lens(b, case["lo"], case["hi"], seed)
    if case["op"] == "attend":
        new = _drawn_lens(b, case["tokens_lo"], case["tokens_hi"], seed + 1)
        return new, [max(k, n) for k, n in zip(cached, new)]
    if case["op"] == "append":
        return _drawn_lens(b, case["new_lo"], case["new_hi"], seed + 1), cached
    return [0] * b, cached


def _pairs(case, new, cached):
    """Visible (query, key) pairs of a sequence: query i sees the keys up to cached - new + i, or the last ``window`` + 1 of them."""
    last = range(cached - new, cached)
    return sum(i + 1 if case["window"] < 0 else min(i, case["window"]) + 1 for i in last)


def _seen(case, new, cached):
    """Keys of a sequence that any query sees: what has to be read of its cache."""
    return cached if case["window"] < 0 else min(cached, new + case["window"])


def work(case):
    new, cached = _lens(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    tq = sum(new)
    if case["op"] in ("rotary", "train"):  # Q, K (and their gradients) read and written; positions; the tables' rows
        times = 2 if case["op"] == "train" else 1
        side = max(2, int(tq ** 0.5))
        return {"bytes": times * (4 * tq * (hq + hkv) * d + 8 * tq * case["axes"]) + 2 * case["rotary_dim"] * side,
                "flops": times * 3 * tq * (hq + hkv) * case["rotary_dim"]}
    token = 2 * hkv * (d // 2 + 4 * d // case["group"])  # bytes of a cached token, K and V: codes, scale and least value
    size = case["page"]
    if case["op"] == "attend":
        seen = [_seen(case, n, c) for n, c in zip(new, cached)]
        pages = sum(-(-s // size) for s in seen) if size else 0
        return {"bytes": sum(seen) * token + tq * hq * (4 * d + 4) + 4 * pages + 4 * case["batch"],
                "flops": 4 * d * hq * sum(_pairs(case, n, c) for n, c in zip(new, cached))}
    if case["op"] == "append":  # q, k, v read; q, the cache's rows and the values they stand for written; a row of the tables per token
        return {"bytes": tq * (4 * hq * d + 8 * hkv * d + token + 2 * d), "flops": 3 * tq * (hq + hkv) * d}
    return {"bytes": sum(cached) * (token + 4 * hkv * d), "flops": 2 * sum(cached) * 2 * hkv * d}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _starts(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0)


def _tables(rows, half, dt):
    """cos / sin of position * 10000^(-i / half), in the element type."""
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64, device="cuda") / half)
    return angle.cos().to(dt), angle.sin().to(dt)


def _sections(axes, half):
    """Pairs of a head's rotation per axis: for three axes a quarter turns with time, the rest in equal shares with height and width."""
    return {1: None, 2: (half // 2, half - half // 2), 3: (half // 4, (half - half // 4) // 2, half - half // 4 - (half - half // 4) // 2)}[axes]


def _image_positions(axes, first, n):
    """Positions [axes, n] of tokens that walk an image row by row behind ``first`` tokens of text (one axis: one after the other)."""
    i = torch.arange(n, dtype=torch.int32)
    side = max(1, int(n ** 0.5))
    return torch.stack([first + i] if axes == 1 else [torch.full_like(i, first), first + i // side, first + i % side][3 - axes:])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt, b, hq, hkv, d = _DTYPES[case["dtype"]], case["batch"], case["hq"], case["hkv"], case["d"]
    new, cached = _lens(case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt)

    s = dict(case=case, new=new, cached=cached)
    if case["op"] in ("rotary", "train"):
        n, half = case["tokens"], case["rotary_dim"] // 2
        s["q"], s["k"] = normal(b, n, hq, d), normal(b, n, hkv, d)
        s["positions"] = torch.stack([_image_positions(case["axes"], 7 * i, n) for i in range(b)], 1).cuda()  # [axes, b, n]
        s["sections"] = _sections(case["axes"], half)
        s["cos"], s["sin"] = _tables(n + 7 * b, half, dt)
        if case["op"] == "train":
            s["q"].requires_grad_()
            s["k"].requires_grad_()
            s["dq"], s["dk"] = normal(b, n, hq, d), normal(b, n, hkv, d)
        return s
    page, room = case["page"], max(c + (n if case["op"] == "append" else 0) for n, c in zip(new, cached))
    s["seqlen_k"] = torch.tensor(cached, dtype=torch.int32, device="cuda")
    if page:
        pages = max(1, -(-room // page))
        s["table"] = torch.randperm(b * pages, generator=g, device="cuda").to(torch.int32).view(b, pages)
        rows = (b * pages, page)
    else:
        s["table"], rows = None, (b, max(1, room))
    for n in "kv":
        s[n + "_codes"] = torch.empty(*rows, hkv, d // 2, dtype=torch.uint8, device="cuda")
        s[n + "_params"] = torch.empty(*rows, hkv, d // case["group"], 2, dtype=dt, device="cuda")
        step = max(1, (1 << 26) // (rows[1] * hkv * d)) if case["op"] != "append" else rows[0]
        for i in range(0, rows[0], step):
            codes, params = s[n + "_codes"][i: i + step], s[n + "_params"][i: i + step]
            if case["op"] == "append":  # (rows that the call writes or leaves alone)
                codes.zero_()
                params.zero_()
            else:
                c, p = _quantise(normal(*codes.shape[:-1], d), case["group"], torch.float32)
                codes.copy_(c)
                params.copy_(p)
    if case["op"] == "attend":
        ragged = case["tokens_lo"] < case["tokens_hi"]
        s["q"] = normal(sum(new), hq, d) if ragged else normal(b, new[0], hq, d)
        s["cu"] = _starts(new).cuda() if ragged else None
    elif case["op"] == "append":
        s["q"], s["knew"], s["vnew"] = normal(sum(new), hq, d), normal(sum(new), hkv, d), normal(sum(new), hkv, d)
        s["cu"] = _starts(new).cuda()
        s["cos"], s["sin"] = _tables(room + 1, d // 2, dt)
        axes = case["axes"]
        s["sections"] = _sections(axes, d // 2) if axes else None
        s["positions"] = torch.cat([_image_positions(axes, c, n) for n, c in zip(new, cached)], 1).cuda() if axes else None
    else:
        s["cu"] = _starts(cached).cuda()
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _quantise(x, group, wide=torch.float64):
    """(codes, params) of [..., d].  A value between two codes goes to the nearer one, which 64 bits decide."""
    x = x.unflatten(-1, (-1, group))
    lo, hi = x.float().amin(-1, keepdim=True), x.float().amax(-1, keepdim=True)
    scale = ((hi - lo).to(wide) / 15).float().to(x.dtype)
    code = ((x.float() - lo).to(wide) / scale.to(wide)).round_().nan_to_num_(0.0).clamp_(0, 15)
    code = code.to(torch.uint8).flatten(-2)
    return code[..., ::2] | (code[..., 1::2] << 4), torch.cat([scale, lo.to(x.dtype)], -1)


def _values(codes, params, wide=torch.float32):
    """What codes [..., d / 2] with params [..., groups, 2] stand for, [..., d]."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).to(wide)
    return (code.unflatten(-1, (params.shape[-2], -1)) * params[..., :1].to(wide) + params[..., 1:].to(wide)).flatten(-2)


def _rows_of(s, n, which):
    """The first ``which`` tokens of sequence n: (K codes, K params, V codes, V params)."""
    r = []
    for name in ("k_codes", "k_params", "v_codes", "v_params"):
        x = s[name]
        if s["table"] is None:
            r.append(x[n, :which])
        else:
            r.append(x[s["table"][n, : -(-which // x.shape[1])]].flatten(0, 1)[:which])
    return r


def _angles(s, positions, wide=torch.float32):
    """cos and sin [..., half] of positions [axes, ...], each pair by the position along its axis."""
    half = s["cos"].shape[-1]
    sections = s["sections"] or (half,)
    at = torch.cat([positions[a][..., None].expand(*positions.shape[1:], n) for a, n in enumerate(sections)], -1).long()
    pair = torch.arange(half, device=at.device)
    return s["cos"][at, pair].to(wide), s["sin"][at, pair].to(wide)


def _rotated(x, cos, sin, rope):
    """[..., heads, d] turned by cos / sin [..., half], in their type; channels behind the rotated ones stay."""
    half = cos.shape[-1]
    turned, rest = x[..., : 2 * half].to(cos.dtype), x[..., 2 * half:].to(cos.dtype)
    a, b = (turned[..., :half], turned[..., half:]) if rope == "half" else (turned[..., ::2], turned[..., 1::2])
    c, s = cos.unsqueeze(-2), sin.unsqueeze(-2)
    y = (a * c - b * s, a * s + b * c)
    return torch.cat([torch.cat(y, -1) if rope == "half" else torch.stack(y, -1).flatten(-2), rest], -1)


def _plain_attend(s):
    case, hq, hkv, d = s["case"], s["case"]["hq"], s["case"]["hkv"], s["case"]["d"]
    o, lse, row = [], [], 0
    for n, (lq, lk) in enumerate(zip(s["new"], s["cached"])):
        q = (s["q"][n] if s["cu"] is None else s["q"][row: row + lq]).float() * d ** -0.5
        row += lq
        kc, kp, vc, vp = _rows_of(s, n, lk)
        x = q.view(lq, hkv, hq // hkv, d).permute(1, 0, 2, 3).flatten(1, 2) @ _values(kc, kp).permute(1, 2, 0)  # [hkv, lq * g, lk]
        x = x.view(hkv, lq, hq // hkv, lk)
        i, j = torch.arange(lk - lq, lk, device="cuda")[:, None, None], torch.arange(lk, device="cuda")
        hidden = j > i
        if case["window"] >= 0:
            hidden |= j < i - case["window"]
        x = x.masked_fill(hidden, float("-inf"))
        m = x.amax(-1, keepdim=True)
        p = (x - m).exp_()
        total = p.sum(-1, keepdim=True)
        part = (p.flatten(1, 2) @ _values(vc, vp).transpose(0, 1)).view(hkv, lq, hq // hkv, d) / total
        o.append(part.permute(1, 0, 2, 3).flatten(1, 2).to(s["q"].dtype))
        lse.append((m + total.log())[..., 0].permute(0, 2, 1).flatten(0, 1))
    return (torch.stack(o), torch.stack(lse)) if s["cu"] is None else (torch.cat(o), torch.cat(lse, 1))


def _token_places(s):
    """Of every new token: its sequence and its position in the cache."""
    total = sum(s["new"])
    seq = torch.repeat_interleave(torch.arange(len(s["new"]), device="cuda"), s["cu"].diff(), output_size=total)
    return seq, s["seqlen_k"].long()[seq] + torch.arange(total, device="cuda") - s["cu"][seq]


def _plain_append(s):
    case = s["case"]
    seq, at = _token_places(s)
    cos, sin = _angles(s, at[None] if s["positions"] is None else s["positions"])
    dt = s["q"].dtype
    q, k = _rotated(s["q"], cos, sin, case["rope"]).to(dt), _rotated(s["knew"], cos, sin, case["rope"]).to(dt)
    page = case["page"]
    where = (s["table"].long()[seq, at // page], at % page) if page else (seq, at)
    held = []
    for n, x in (("k", k), ("v", s["vnew"])):
        codes, params = _quantise(x, case["group"])
        s[n + "_codes"][where], s[n + "_params"][where] = codes, params
        held.append(_values(codes, params).to(dt))
    return (q, *held)


def _plain_read(s):
    k, v = [], []
    for n, lk in enumerate(s["cached"]):
        kc, kp, vc, vp = _rows_of(s, n, lk)
        k.append(_values(kc, kp).to(kp.dtype))
        v.append(_values(vc, vp).to(vp.dtype))
    return torch.cat(k), torch.cat(v)


def _plain_rotary(s):
    cos, sin = _angles(s, s["positions"])
    dt, rope = s["q"].dtype, s["case"]["rope"]
    y = [_rotated(s[n].detach(), cos, sin, rope).to(dt) for n in "qk"]
    if s["case"]["op"] == "train":  # the gradient is turned back
        y += [_rotated(s[n], cos, -sin, rope).to(dt) for n in ("dq", "dk")]
    return tuple(y)


def run(s):
    case = s["case"]
    if own:
        from flashck_b200 import ops
        from flashck_b200.utils.enums import RopeEnum
        if case["op"] == "attend":
            return ops.fmha_fwd_splitkv_int4(s["q"], s["k_codes"], s["k_params"], s["v_codes"], s["v_params"], seqlen_k=s["seqlen_k"],
                                             block_table=s["table"], cu_seqlens_q=s["cu"], max_seqlen_q=case["tokens_hi"], causal=True,
                                             window_size=(case["window"], 0), return_lse=True)
        if case["op"] == "read":
            return ops.fmha_read_kv_int4(s["k_codes"], s["k_params"], s["v_codes"], s["v_params"], s["seqlen_k"], block_table=s["table"],
                                         cu_seqlens_k=s["cu"], total_k=sum(s["cached"]))
        rope = RopeEnum.HALF_ROTATED if case["rope"] == "half" else RopeEnum.INTERLEAVED
        if case["op"] == "append":
            return ops.fmha_fwd_append_kv_int4(s["q"], s["k_codes"], s["k_params"], s["v_codes"], s["v_params"], s["knew"], s["vnew"],
                                               s["seqlen_k"], s["cos"], s["sin"], rope=rope, positions=s["positions"],
                                               sections=s["sections"], block_table=s["table"], cu_seqlens_q=s["cu"],
                                               cu_seqlens_knew=s["cu"], return_kv=True)
        if case["op"] == "rotary":
            return ops.apply_rotary(s["q"], s["k"], s["positions"], s["cos"], s["sin"], sections=s["sections"], rope=rope)
        y = ops.apply_rotary_autograd(s["q"], s["k"], s["positions"], s["cos"], s["sin"], sections=s["sections"], rope=rope)
        return tuple(t.detach() for t in y) + torch.autograd.grad(y, (s["q"], s["k"]), (s["dq"], s["dk"]))
    with torch.no_grad():
        return {"attend": _plain_attend, "append": _plain_append, "read": _plain_read}.get(case["op"], _plain_rotary)(s)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _exact_values(codes, params):
    codes = codes.to(torch.int64)
    u = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    u[..., ::2], u[..., 1::2] = codes % 16, codes // 16
    group = u.shape[-1] // params.shape[-2]
    scale, least = (params[..., i].double().repeat_interleave(group, -1) for i in (0, 1))
    return least + scale * u


def _exact_held(x, group):
    """What the cache holds for x [t, heads, d], channel group by channel group."""
    out = x.double().clone()
    for i in range(0, x.shape[-1], group):
        part = x[..., i: i + group].double()
        least, most = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        step = ((most - least) / 15).to(x.dtype).double()
        code = torch.where(step > 0, torch.round((part - least) / step.clamp_min(5e-324)), torch.zeros_like(part)).clamp(max=15)
        out[..., i: i + group] = least + step * code
    return out


def _exact_turned(s, x, positions, sign=1.0):
    """Pair by pair: (a, b) -> (a cos - b sin, a sin + b cos).  positions [axes, ...] of x [..., heads, d]."""
    half = s["cos"].shape[-1]
    axis = [a for a, n in enumerate(s["sections"] or (half,)) for _ in range(n)]
    out = x.double().clone()
    for i in range(half):
        at = positions[axis[i]].long()
        c, sn = s["cos"][at, i].double()[..., None], sign * s["sin"][at, i].double()[..., None]
        p, r = (i, i + half) if s["case"]["rope"] == "half" else (2 * i, 2 * i + 1)
        a, b = x[..., p].double(), x[..., r].double()
        out[..., p], out[..., r] = a * c - b * sn, a * sn + b * c
    return out


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    with torch.no_grad():
        if case["op"] in ("rotary", "train"):
            r = [_exact_turned(s, s[n].detach(), s["positions"]) for n in "qk"]
            return tuple(r + [_exact_turned(s, s[n], s["positions"], -1.0) for n in ("dq", "dk") if n in s])
        if case["op"] == "read":
            rows = [_rows_of(s, n, lk) for n, lk in enumerate(s["cached"])]
            return tuple(torch.cat([_exact_values(r[i], r[i + 1]) for r in rows]) for i in (0, 2))
        if case["op"] == "append":
            at = s["positions"] if s["positions"] is not None else torch.cat(
                [torch.arange(c, c + n, device="cuda") for n, c in zip(s["new"], s["cached"])])[None]
            q, k = _exact_turned(s, s["q"], at), _exact_turned(s, s["knew"], at)
            return q, _exact_held(k.to(s["knew"].dtype), case["group"]), _exact_held(s["vnew"], case["group"])
        o, lse, row = [], [], 0
        for n, (lq, lk) in enumerate(zip(s["new"], s["cached"])):
            q = (s["q"][n] if s["cu"] is None else s["q"][row: row + lq]).double()
            row += lq
            kc, kp, vc, vp = _rows_of(s, n, lk)
            heads_o, heads_l = [], []
            for h in range(hkv):  # a kv head at a time: 64-bit keys and values are large
                x = torch.einsum("tgd,jd->gtj", q.unflatten(1, (hkv, hq // hkv))[:, h], _exact_values(kc[:, h], kp[:, h])) / d ** 0.5
                last = torch.arange(lk - lq, lk, device="cuda")[:, None]
                j = torch.arange(lk, device="cuda")[None]
                x = torch.where((j > last) | ((case["window"] >= 0) & (j < last - case["window"])), -torch.inf, x)
                heads_l.append(torch.logsumexp(x, -1))
                heads_o.append(torch.einsum("gtj,jd->tgd", torch.softmax(x, -1), _exact_values(vc[:, h], vp[:, h])))
            o.append(torch.cat(heads_o, 1))
            lse.append(torch.cat(heads_l, 0))
        return (torch.stack(o), torch.stack(lse)) if s["cu"] is None else (torch.cat(o), torch.cat(lse, 1))
