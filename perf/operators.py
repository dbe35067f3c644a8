"""The operators next to the attention forward, as measurable cases: its backward pass, and decode over a shared prefix.

A case is a dict of plain values.  ``op`` names the path:

* ``bwd``    -- ``fmha_bwd`` / ``fmha_bwd_var_len``: dQ, dK, dV (and the gradient of a bias tensor) from dO and the forward's O and LSE
* ``step``   -- ``fmha_autograd`` and its backward: what a training step spends in attention
* ``prefix`` -- ``fmha_fwd_shared_prefix``: new tokens of many sequences against one prefix and each sequence's own cache

``run`` computes them in elementary torch operations, or with ``own`` through ``flashck_b200.ops``.  Lengths are fixed by
``lens_seed``, so that the work of a case does not depend on the seed of its values.
"""
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_MOST_FLOPS, _MOST_BYTES = 2.2e12, 1.4e9  # of a drawn case: what the largest listed ones take


def _bwd(name, dtype, batch, hq, hkv, d, **more):
    case = dict(name=name, op="bwd", dtype=dtype, batch=batch, hq=hq, hkv=hkv, d=d, mask="causal", window=0, add="none", cap=0.0)
    case.update(more)
    return case


def _prefix(name, dtype, batch, hq, hkv, d, **more):
    case = dict(name=name, op="prefix", dtype=dtype, batch=batch, hq=hq, hkv=hkv, d=d, tokens_lo=1, tokens_hi=1)
    case.update(more)
    return case


def listed():
    return [
        # two short prompts, where the call itself is what takes the time
        _bwd("bwd_tiny", "fp16", 2, 8, 8, 64, sq=128, sk=128),
        # pre-training: two full sequences of a grouped-query model
        _bwd("bwd_causal", "bf16", 2, 32, 8, 128, sq=4096, sk=4096),
        # fine-tuning on packed documents of unequal lengths
        _bwd("bwd_varlen", "bf16", 16, 32, 8, 128, lo=512, hi=4096, lens_seed=1234),
        # an encoder: head dim 64, no mask, a length that no tile divides
        _bwd("bwd_encoder_hdim64", "bf16", 16, 16, 16, 64, sq=1025, sk=1025, mask="none"),
        # a sliding window and a logits soft cap
        _bwd("bwd_window_softcap", "bf16", 2, 32, 8, 128, sq=5000, sk=5000, mask="window", window=1023, cap=30.0),
        # a learned relative-position bias, one plane per head, shared by the batch
        _bwd("bwd_bias_per_head", "bf16", 2, 16, 16, 128, sq=1024, sk=1024, mask="none", add="bias1"),
        # a layer's attention in a training step, forward and backward
        dict(_bwd("train_step", "fp16", 4, 16, 16, 128, sq=2048, sk=2048), op="step"),
        # a few answers behind one prompt, just begun; the prompt ends inside a page
        _prefix("prefix_few", "bf16", 8, 32, 8, 128, prefix=1000, lo=0, hi=60, page=16, lens_seed=3),
        # a serving batch behind a long system prompt
        _prefix("prefix_batch", "bf16", 64, 32, 8, 128, prefix=8192, lo=64, hi=2048, page=16, lens_seed=17),
        # many questions about one very long document
        _prefix("prefix_document", "bf16", 32, 64, 8, 128, prefix=131072, lo=1, hi=4096, page=64, lens_seed=29),
        # speculative decoding: one to four drafted tokens per sequence, contiguous caches of head dim 64
        _prefix("prefix_drafted", "fp16", 48, 32, 8, 64, prefix=4000, lo=8, hi=500, page=0, lens_seed=41, tokens_lo=1, tokens_hi=4),
        # the whole batch's rows fill one tile per kv head many times over: 256 samples of one prompt
        _prefix("prefix_samples", "bf16", 256, 32, 8, 128, prefix=2000, lo=1, hi=300, page=16, lens_seed=53),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_once(rng):
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 16), (8, 8), (16, 2), (12, 4)])
    dtype, d, seed = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([128, 128, 64]), rng.randrange(1 << 20)
    kind = rng.choice(["dense", "dense", "varlen", "step", "prefix", "prefix"])
    if kind == "prefix":
        lo = _log_int(rng, 1, 1000)
        tokens = rng.choice([1, 1, 1, 2, 5, 8])
        case = _prefix("", dtype, _log_int(rng, 2, 256), hq, hkv, d, prefix=_log_int(rng, 50, 131072), lo=lo, hi=lo * rng.randint(1, 8),
                       page=rng.choice([0, 16, 16, 64]), lens_seed=seed, tokens_lo=rng.choice([1, tokens]), tokens_hi=tokens)
    else:
        case = _bwd("", dtype, _log_int(rng, 1, 32), hq, hkv, d, mask=rng.choice(["none", "causal", "causal", "window"]))
        if case["mask"] == "window":
            case["window"] = _log_int(rng, 16, 4096)
        if kind == "varlen":
            lo = _log_int(rng, 1, 1024)
            case.update(lo=lo, hi=lo * rng.randint(2, 8), lens_seed=seed)
        else:
            sq = _log_int(rng, 32, 8192)
            case.update(sq=sq, sk=sq + rng.choice([0, 0, 0, rng.randint(1, sq)]), cap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                        add=rng.choice(["none", "none", "none", "alibi", "bias0", "bias1", "bias2"]))
            if kind == "step":
                case.update(op="step", add="none")
    del case["name"]
    return case


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        dear = case.get("cap", 0.0) > 0 or case.get("add", "none") != "none"  # (score additions: more time per FLOP)
        rows = case["batch"] * case["tokens_hi"] * case["hq"] if case["op"] == "prefix" else 0
        if w["flops"] <= _MOST_FLOPS / (8 if dear else 1) and w["bytes"] <= _MOST_BYTES and rows * case.get("prefix", 0) <= 1 << 29:
            return case


# ---- sizes of a case -----------------------------------------------------------------------------------------------
def _drawn_lens(n, lo, hi, seed):
    rng = random.Random(seed)
    return [rng.randint(lo, hi) for _ in range(n)]


def _lens(case):
    """(query lengths, key lengths) of every sequence; of a shared prefix: the keys of its own cache."""
    b = case["batch"]
    if case["op"] == "prefix":
        nq = _drawn_lens(b, case["tokens_lo"], case["tokens_hi"], case["lens_seed"] + 1)
        return nq, [max(k, q) for k, q in zip(_drawn_lens(b, case["lo"], case["hi"], case["lens_seed"]), nq)]
    if "lo" in case:
        n = _drawn_lens(b, case["lo"], case["hi"], case["lens_seed"])
        return n, n
    return [case["sq"]] * b, [case["sk"]] * b


def _pairs(case, nq, nk):
    """Visible (query, key) pairs of one sequence: bottom-right aligned causal or window masks, or everything."""
    if case.get("mask", "causal") == "none":
        return nq * nk
    full = nq * (nk - nq) + nq * (nq + 1) // 2
    if case.get("mask", "causal") == "causal":
        return full
    hidden = max(0, nk - case["window"] - 1)  # keys the last row no longer sees; one fewer for each row before it
    rows = min(nq, hidden)
    return full - (rows * hidden - rows * (rows - 1) // 2)


def work(case):
    nq, nk = _lens(case)
    b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    tq, tk = sum(nq), sum(nk)
    pairs = sum(_pairs(case, q, k) for q, k in zip(nq, nk))
    if case["op"] == "prefix":  # Q, the prefix's K/V and every own K/V read, page ids read, O and LSE written
        size = case["page"]
        pages = (-(-case["prefix"] // size) + sum(-(-k // size) for k in nk)) if size else 0
        return {"bytes": tq * hq * (4 * d + 4) + (case["prefix"] + tk) * hkv * 4 * d + 4 * pages + 4 * b,
                "flops": 4 * d * hq * (pairs + tq * case["prefix"])}
    if case["op"] == "step":  # forward and backward: Q, K, V, dO read, O, dQ, dK, dV written; seven products
        return {"bytes": tq * hq * 8 * d + tk * hkv * 8 * d, "flops": 14 * d * hq * pairs}
    nbytes = tq * hq * (8 * d + 4) + tk * hkv * 8 * d  # Q, O, dO, LSE read, dQ written; K, V read, dK, dV written
    if case["add"].startswith("bias"):
        nbytes += 4 * case["sq"] * case["sk"] * {"0": 1, "1": hq, "2": b * hq}[case["add"][-1]]
    return {"bytes": nbytes, "flops": 10 * d * hq * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _starts(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0)


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt, b, hq, hkv, d = _DTYPES[case["dtype"]], case["batch"], case["hq"], case["hkv"], case["d"]
    nq, nk = _lens(case)

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dt)

    s = dict(case=case, nq=nq, nk=nk)
    if case["op"] == "prefix":
        ragged, page = case["tokens_lo"] < case["tokens_hi"], case["page"]
        s["q"] = normal(sum(nq), hq, d) if ragged else normal(b, nq[0], hq, d)
        s["cu_q"] = _starts(nq).cuda() if ragged else None
        s["seqlen_k"] = torch.tensor(nk, dtype=torch.int32, device="cuda")
        if page:
            own_pages, n_prefix = max(-(-k // page) for k in nk), -(-case["prefix"] // page)
            pool = b * own_pages + n_prefix
            ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
            s["k"], s["v"] = normal(pool, page, hkv, d), normal(pool, page, hkv, d)
            s["kp"], s["vp"] = s["k"], s["v"]
            s["prefix_table"], s["table"] = ids[:n_prefix].contiguous(), ids[n_prefix:].view(b, own_pages).contiguous()
        else:
            s["k"], s["v"] = normal(b, max(nk), hkv, d), normal(b, max(nk), hkv, d)
            s["kp"], s["vp"] = normal(case["prefix"], hkv, d), normal(case["prefix"], hkv, d)
            s["prefix_table"] = s["table"] = None
        return s
    if "lo" in case:
        s["q"], s["k"], s["v"], s["dout"] = normal(sum(nq), hq, d), normal(sum(nk), hkv, d), normal(sum(nk), hkv, d), normal(sum(nq), hq, d)
        s["cu"] = _starts(nq).cuda()
    else:
        sq, sk = case["sq"], case["sk"]
        s["q"], s["k"], s["v"], s["dout"] = normal(b, sq, hq, d), normal(b, sk, hkv, d), normal(b, sk, hkv, d), normal(b, sq, hq, d)
    s["slopes"] = 2.0 ** (-8.0 / hq * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32))[None] if case["add"] == "alibi" else None
    planes = {"bias0": (1, 1), "bias1": (1, hq), "bias2": (b, hq)}.get(case["add"])
    s["bias"] = normal(*planes, case["sq"], case["sk"]) if planes else None
    if case["op"] == "step":
        for n in "qkv":
            s[n].requires_grad_()
    else:
        with torch.no_grad():
            s["o"], s["lse"] = _plain_forward(s)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------
def _pieces(s):
    """Slices of the batch whose score matrices fit the memory, as (query rows, key rows, sequences) of [b, s, h, d] views."""
    case = s["case"]
    if "lo" in case:
        q0 = k0 = 0
        for nq, nk in zip(s["nq"], s["nk"]):
            yield slice(q0, q0 + nq), slice(k0, k0 + nk), None
            q0, k0 = q0 + nq, k0 + nk
    else:
        n = max(1, (1 << 30) // (case["sq"] * case["sk"] * case["hq"]))
        for i in range(0, case["batch"], n):
            yield slice(i, i + n), slice(i, i + n), slice(i, i + n)


def _heads_first(x, rows, hq):
    """[b, hq, s, d] in fp32 of the given rows; key heads are repeated for their group."""
    x = x[rows].float()
    x = (x[None] if x.dim() == 3 else x).transpose(1, 2)
    return x.repeat_interleave(hq // x.shape[1], dim=1)


def _visible(case, sq, sk, device):
    i, j = torch.arange(sq, device=device)[:, None] + (sk - sq), torch.arange(sk, device=device)[None]
    if case["mask"] == "none":
        return torch.ones(sq, sk, dtype=torch.bool, device=device)
    return (j <= i) & (j >= i - case["window"]) if case["mask"] == "window" else j <= i


def _plain_scores(s, q, k, seqs):
    """Scores with the additions of the case, -inf where masked, and the derivative of the soft cap."""
    case = s["case"]
    x = (q * case["d"] ** -0.5) @ k.transpose(2, 3)
    slope = None
    if case["cap"] > 0:
        t = torch.tanh(x / case["cap"])
        x, slope = t * case["cap"], 1 - t * t
    sq, sk = x.shape[2:]
    if s["slopes"] is not None:
        away = (torch.arange(sq, device=x.device)[:, None] + (sk - sq) - torch.arange(sk, device=x.device)[None]).abs()
        x = x - s["slopes"][:, :, None, None] * away
    if s["bias"] is not None:
        x = x + (s["bias"][seqs] if s["bias"].shape[0] > 1 else s["bias"]).float()
    return x.masked_fill(~_visible(case, sq, sk, x.device), float("-inf")), slope


def _put(out, rows, x):
    """Writes [b, h, s, d] to the rows of a [.., s, h, d] tensor, rounding once."""
    x = x.transpose(1, 2)
    out[rows] = (x[0] if out.dim() == 3 else x).to(out.dtype)


def _plain_forward(s):
    case, hq = s["case"], s["case"]["hq"]
    o = torch.empty_like(s["q"])
    lse = torch.empty((hq, s["q"].shape[0]) if "lo" in case else (case["batch"], hq, case["sq"]), device="cuda")
    for qr, kr, seqs in _pieces(s):
        x, _ = _plain_scores(s, _heads_first(s["q"], qr, hq), _heads_first(s["k"], kr, hq), seqs)
        m = x.amax(-1, keepdim=True).clamp_min(-1e30)
        p = (x - m).exp_()
        total = p.sum(-1, keepdim=True)
        part = (m + total.log())[..., 0]
        if "lo" in case:
            lse[:, qr] = part[0]
        else:
            lse[qr] = part
        _put(o, qr, (p @ _heads_first(s["v"], kr, hq)) / total.clamp_min(1e-30))
    return o, lse


def _plain_backward(s, o, lse):
    case, hq, hkv, scale = s["case"], s["case"]["hq"], s["case"]["hkv"], s["case"]["d"] ** -0.5
    dq, dk, dv = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
    dbias = torch.zeros(s["bias"].shape, device="cuda") if s["bias"] is not None else None
    for qr, kr, seqs in _pieces(s):
        q, k, v = _heads_first(s["q"], qr, hq), _heads_first(s["k"], kr, hq), _heads_first(s["v"], kr, hq)
        do, rows_o = _heads_first(s["dout"], qr, hq), _heads_first(o, qr, hq)
        x, slope = _plain_scores(s, q, k, seqs)
        p = (x - (lse[None, :, qr] if "lo" in case else lse[qr])[..., None]).exp_()
        dt = p * (do @ v.transpose(2, 3) - (do * rows_o).sum(-1, keepdim=True))
        if dbias is not None:
            if dbias.shape[0] > 1:
                dbias[seqs] = dt
            else:
                dbias += dt.sum(0, keepdim=True).sum(1, keepdim=True) if dbias.shape[1] == 1 else dt.sum(0, keepdim=True)
        ds = dt if slope is None else dt * slope

        def grouped(y):  # the sum over the heads of a group
            return y.unflatten(1, (hkv, hq // hkv)).sum(2)

        _put(dv, kr, grouped(p.transpose(2, 3) @ do))
        _put(dk, kr, grouped(ds.transpose(2, 3) @ q) * scale)
        _put(dq, qr, (ds @ k) * scale)
    return (dq, dk, dv) if dbias is None else (dq, dk, dv, dbias.to(s["q"].dtype))


def _plain_prefix(s):
    case, b, hq, hkv, d = s["case"], s["case"]["batch"], s["case"]["hq"], s["case"]["hkv"], s["case"]["d"]
    g, most_k, most_q = hq // hkv, max(s["nk"]), max(s["nq"])
    kp, vp, k, v = s["kp"], s["vp"], s["k"], s["v"]
    if case["page"]:  # gather the pages
        kp, vp = kp[s["prefix_table"]].flatten(0, 1)[: case["prefix"]], vp[s["prefix_table"]].flatten(0, 1)[: case["prefix"]]
        k, v = k[s["table"]].flatten(1, 2)[:, :most_k], v[s["table"]].flatten(1, 2)[:, :most_k]
    n_k = s["seqlen_k"].long()
    if s["cu_q"] is None:
        q, n_q = s["q"].float(), torch.full_like(n_k, most_q)
    else:  # sequences padded to the longest
        n_q = s["cu_q"].diff()
        here = torch.arange(most_q, device="cuda")[None] < n_q[:, None]
        q = torch.zeros(b, most_q, hq, d, device="cuda")
        q[here] = s["q"].float()
    q = (q * d ** -0.5).view(b, most_q, hkv, g, d)
    # scores [hkv, b, t, g, keys]
    x_own = q.permute(2, 0, 1, 3, 4).flatten(2, 3) @ k.float().permute(2, 0, 3, 1)
    x_own = x_own.view(hkv, b, most_q, g, most_k)
    i, j = torch.arange(most_q, device="cuda")[None, :, None], torch.arange(most_k, device="cuda")
    seen = j <= (n_k - n_q)[:, None, None] + i
    x_own = x_own.masked_fill(~seen[None, :, :, None], float("-inf"))
    x_pre = q.permute(2, 0, 1, 3, 4).flatten(1, 3) @ kp.float().permute(1, 2, 0)
    x_pre = x_pre.view(hkv, b, most_q, g, case["prefix"])
    m = torch.maximum(x_own.amax(-1, keepdim=True), x_pre.amax(-1, keepdim=True))
    p_own, p_pre = (x_own - m).exp_(), (x_pre - m).exp_()
    total = p_own.sum(-1, keepdim=True) + p_pre.sum(-1, keepdim=True)
    # rows behind a sequence's keys are masked, and what lies there does not count
    v = v.float().masked_fill((j[None] >= n_k[:, None])[:, :, None, None], 0.0)
    o = (p_own.flatten(2, 3) @ v.permute(2, 0, 1, 3)).view(hkv, b, most_q, g, d)
    o = (o + (p_pre.flatten(1, 3) @ vp.float().transpose(0, 1)).view(hkv, b, most_q, g, d)) / total
    o = o.permute(1, 2, 0, 3, 4).flatten(2, 3).to(s["q"].dtype)  # [b, t, hq, d]
    lse = (m + total.log())[..., 0].permute(1, 0, 3, 2).flatten(1, 2)  # [b, hq, t]
    return (o, lse) if s["cu_q"] is None else (o[here], lse.transpose(1, 2)[here].T.contiguous())


def _options(s):
    case = s["case"]
    return dict(causal=case["mask"] != "none", window_size=(case["window"], 0) if case["mask"] == "window" else (-1, -1),
                logits_soft_cap=case["cap"])


def run(s):
    case = s["case"]
    if own:
        from flashck_b200 import ops
        if case["op"] == "prefix":
            return ops.fmha_fwd_shared_prefix(s["q"], s["kp"], s["vp"], s["k"], s["v"], prefix_len=case["prefix"], prefix_table=s["prefix_table"],
                                              seqlen_k=s["seqlen_k"], block_table=s["table"], cu_seqlens_q=s["cu_q"],
                                              max_seqlen_q=case["tokens_hi"], causal=True, return_lse=True)
        if case["op"] == "step":
            o = ops.fmha_autograd(s["q"], s["k"], s["v"], **_options(s))
            return (o.detach(),) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["dout"])
        if "lo" in case:
            return ops.fmha_bwd_var_len(s["dout"], s["q"], s["k"], s["v"], s["o"], s["lse"], s["cu"], s["cu"], max(s["nq"]), max(s["nk"]),
                                        **_options(s))
        return ops.fmha_bwd(s["dout"], s["q"], s["k"], s["v"], s["o"], s["lse"], alibi_slopes=s["slopes"], bias=s["bias"],
                            return_dbias=s["bias"] is not None, **_options(s))
    with torch.no_grad():
        if case["op"] == "prefix":
            return _plain_prefix(s)
        if case["op"] == "step":
            o, lse = _plain_forward(s)
            return (o,) + _plain_backward(s, o, lse)
        return _plain_backward(s, s["o"], s["lse"])


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_prefix(s) if case["op"] == "prefix" else _exact_gradients(s)


def _exact_gradients(s):
    """Head by head and sequence by sequence.  ``step`` starts from Q, K, V alone; ``bwd`` from the O and LSE that it is given."""
    case = s["case"]
    b, hq, hkv, d, packed = case["batch"], case["hq"], case["hkv"], case["d"], "lo" in case
    wide = {n: s[n].detach().double() for n in ("q", "k", "v", "dout")}
    out = {n: torch.zeros_like(wide[n]) for n in ("q", "k", "v")}
    o_out = torch.zeros_like(wide["q"])
    dbias = torch.zeros(s["bias"].shape, dtype=torch.float64, device="cuda") if s["bias"] is not None else None
    q0 = k0 = 0
    for n in range(b):
        lq, lk = s["nq"][n], s["nk"][n]
        qs, ks = (slice(q0, q0 + lq), slice(k0, k0 + lk)) if packed else (n, n)
        q0, k0 = q0 + lq, k0 + lk
        distance = torch.arange(lk - lq, lk, device="cuda")[:, None] - torch.arange(lk, device="cuda")[None]
        hidden = torch.zeros_like(distance, dtype=torch.bool) if case["mask"] == "none" else distance < 0
        if case["mask"] == "window":
            hidden |= distance > case["window"]
        for h in range(hq):
            kh = h * hkv // hq
            q, do = wide["q"][qs][:, h], wide["dout"][qs][:, h]
            k, v = wide["k"][ks][:, kh], wide["v"][ks][:, kh]
            x = torch.einsum("id,jd->ij", q, k) / d ** 0.5
            capped = torch.tanh(x / case["cap"]) if case["cap"] > 0 else None
            if capped is not None:
                x = capped * case["cap"]
            if s["slopes"] is not None:
                x = x - s["slopes"][0, h].double() * distance.abs()
            plane = (n if s["bias"].shape[0] > 1 else 0, h if s["bias"].shape[1] > 1 else 0) if s["bias"] is not None else None
            if plane is not None:
                x = x + s["bias"][plane].double()
            x = torch.where(hidden, -torch.inf, x)
            if case["op"] == "step":
                p = torch.softmax(x, dim=1)
                o = p @ v
                o_out[qs][:, h] = o
            else:
                lse = s["lse"][h, qs] if packed else s["lse"][n, h]
                p, o = torch.exp(x - lse.double()[:, None]), s["o"][qs][:, h].double()
            grad = p * (torch.einsum("id,jd->ij", do, v) - torch.einsum("id,id->i", do, o)[:, None])
            if plane is not None:
                dbias[plane] += grad
            if capped is not None:
                grad = grad - grad * capped ** 2
            out["v"][ks][:, kh] += p.T @ do
            out["k"][ks][:, kh] += grad.T @ q / d ** 0.5
            out["q"][qs][:, h] = grad @ k / d ** 0.5
    r = (out["q"], out["k"], out["v"])
    return (o_out,) + r if case["op"] == "step" else r if dbias is None else r + (dbias,)


def _exact_prefix(s):
    """Sequence by sequence, over the concatenation of the prefix and the sequence's own keys."""
    case = s["case"]
    hq, hkv, d, page, length = case["hq"], case["hkv"], case["d"], case["page"], case["prefix"]

    def tokens(cache, ids, n):
        return torch.cat([cache[i] for i in ids[: -(-n // page)].tolist()] or [cache[0]])[:n].double()

    kp, vp = (tokens(s[c], s["prefix_table"], length) if page else s[c].double() for c in ("kp", "vp"))
    o, lse, row = [], [], 0
    for n, (lq, lk) in enumerate(zip(s["nq"], s["nk"])):
        q = (s["q"][n] if s["cu_q"] is None else s["q"][row: row + lq]).double()
        row += lq
        k, v = (tokens(s[c], s["table"][n], lk) if page else s[c][n, :lk].double() for c in ("k", "v"))
        k, v = torch.cat([kp, k]), torch.cat([vp, v])
        x = torch.einsum("thgd,jhd->hgtj", q.unflatten(1, (hkv, hq // hkv)), k).flatten(0, 1) / d ** 0.5
        last = torch.arange(length + lk - lq, length + lk, device="cuda")
        x = torch.where(torch.arange(length + lk, device="cuda")[None] > last[:, None], -torch.inf, x)
        lse.append(torch.logsumexp(x, dim=-1))
        o.append(torch.einsum("hgtj,jhd->thgd", torch.softmax(x, dim=-1).unflatten(0, (hkv, hq // hkv)), v).flatten(1, 2))
    return (torch.stack(o), torch.stack(lse)) if s["cu_q"] is None else (torch.cat(o), torch.cat(lse, dim=1))
