"""What is measured of the paged-cache operators: `page_plan` (block tables, positions and slots from request lengths),
`kv_append` (a ragged batch of new tokens' K and V into the pages) and `attn_extend` (attention of ragged chunks of new
tokens over the paged cache; one new token per request is plain decode).

Pages hold 128 tokens: K [page][kv head][128 tokens][dim], V [page][kv head][dim][128 tokens] (dim-major), in e4m3 codes or
bf16.  With `own` false `run` computes the operators from elementary torch operations in fp32; with `own` true it calls
the package's entry points.
"""
import math
import random

import torch

own = False
PAGE = 128


# ---- cases -----------------------------------------------------------------------------------------------------
def _plan(name, batch, single, new_lo, new_hi, ctx_lo, ctx_hi, lens):
    return dict(name=name, op="plan", batch=batch, single=single, new_lo=new_lo, new_hi=new_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi,
                lens=lens)


def _append(name, dtype, kv_heads, dim, batch, single, new_lo, new_hi, ctx_lo, ctx_hi, lens):
    return dict(name=name, op="append", dtype=dtype, kv_heads=kv_heads, dim=dim, batch=batch, single=single, new_lo=new_lo,
                new_hi=new_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi, lens=lens)


def _attend(name, dtype, q_heads, kv_heads, dim, gate, batch, single, new_lo, new_hi, ctx_lo, ctx_hi, lens):
    return dict(name=name, op="attend", dtype=dtype, q_heads=q_heads, kv_heads=kv_heads, dim=dim, gate=gate, batch=batch,
                single=single, new_lo=new_lo, new_hi=new_hi, ctx_lo=ctx_lo, ctx_hi=ctx_hi, lens=lens)


def listed():
    """`single` of the `batch` requests have one new token, the others new_lo..new_hi; every request has ctx_lo..ctx_hi
    tokens in the cache already."""
    return [
        # a lone request's next token
        _plan("plan_one", 1, 1, 1, 1, 777, 777, 1),
        # a serving step: most requests decode, a few prompts arrive in chunks
        _plan("plan_step", 96, 80, 65, 700, 0, 8192, 2),
        # a large ragged batch of prompt chunks
        _plan("plan_prompts", 1500, 500, 1, 130, 0, 8192, 3),
        # plain decode of a batch of 64: one token each, bytes scattered into 64 pages
        _append("append_decode", "e4m3", 2, 256, 64, 64, 1, 1, 1, 2047, 4),
        # prompts of the usual length, page-unaligned starts
        _append("append_prompts", "e4m3", 2, 256, 6, 0, 700, 1700, 0, 300, 5),
        # bf16 cache, narrower heads, a mixed step
        _append("append_mixed_bf16", "bf16", 4, 128, 40, 24, 30, 500, 1, 1500, 6),
        # the smallest call: the next token of one short conversation
        _attend("attend_one", "e4m3", 16, 2, 256, True, 1, 1, 1, 1, 777, 777, 7),
        # plain decode at the batch and context of the framework's benchmark
        _attend("attend_decode", "e4m3", 16, 2, 256, True, 64, 64, 1, 1, 8191, 8191, 8),
        # few requests with long histories, bf16 cache: the key axis has to be split over the GPU
        _attend("attend_long_bf16", "bf16", 16, 2, 256, True, 2, 2, 1, 1, 60001, 65535, 9),
        # a serving step: decoding requests next to prompt chunks of odd sizes
        _attend("attend_mixed", "e4m3", 16, 2, 256, True, 18, 12, 33, 513, 0, 8000, 10),
        # chunked prompts, narrower heads, a group of 3 query heads per kv head, bf16
        _attend("attend_chunk_bf16", "bf16", 12, 4, 128, False, 3, 0, 1001, 1501, 0, 2500, 11),
        # the largest: four prompt chunks of 2048 tokens behind 6144 cached ones
        _attend("attend_chunk", "e4m3", 16, 2, 256, True, 4, 0, 2048, 2048, 6144, 6144, 12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attend", "attend", "attend", "attend"])
    lens = rng.randrange(1 << 30)
    while True:
        if op == "plan":
            batch = _log_int(rng, 1, 1500)
            hi = _log_int(rng, 1, max(1, min(2048, 60000 // batch)))
            c = dict(op=op, batch=batch, single=rng.randint(0, batch), new_lo=rng.randint(1, hi), new_hi=hi,
                     ctx_lo=0, ctx_hi=_log_int(rng, 1, 8192), lens=lens)
            return c
        dtype = rng.choice(["e4m3", "bf16"])
        heads = rng.choice([(16, 2, 256), (16, 2, 256), (8, 1, 256), (12, 4, 128), (32, 8, 128)])
        if op == "append":
            batch = _log_int(rng, 1, 256)
            hi = _log_int(rng, 1, max(1, min(2048, 8000 // batch)))
            return dict(op=op, dtype=dtype, kv_heads=heads[1], dim=heads[2], batch=batch, single=rng.randint(0, batch),
                        new_lo=rng.randint(1, hi), new_hi=hi, ctx_lo=0, ctx_hi=_log_int(rng, 1, 2047), lens=lens)
        batch = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, 2048)
        ctx_hi = _log_int(rng, 16, 65535)
        c = dict(op=op, dtype=dtype, q_heads=heads[0], kv_heads=heads[1], dim=heads[2], gate=rng.random() < 0.7, batch=batch,
                 single=rng.choice([0, batch, rng.randint(0, batch)]), new_lo=rng.randint(1, hi), new_hi=hi,
                 ctx_lo=rng.randint(0, ctx_hi), ctx_hi=ctx_hi, lens=lens)
        new, ctx = _lens(c)
        longest = max(n + x for n, x in zip(new, ctx))
        # what the plain form holds: padded scores and padded fp32 keys and values
        if (c["q_heads"] * batch * max(new) * longest <= 1.1e9 and batch * longest * c["kv_heads"] * c["dim"] <= 3e8
                and work(c)["flops"] <= 0.97e12):
            return c


def _lens(case):
    """(new tokens, cached tokens) of every request: host integers, fixed by the case."""
    r = random.Random(case["lens"])
    new = [1 if b < case["single"] else _log_int(r, case["new_lo"], case["new_hi"]) for b in range(case["batch"])]
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["batch"])]
    order = list(range(case["batch"]))
    r.shuffle(order)
    return [new[i] for i in order], [ctx[i] for i in order]


def _pages(n):
    return (n + PAGE - 1) // PAGE


# ---- inputs ----------------------------------------------------------------------------------------------------
def _values(shape, dtype, g, dev):
    """N(0, 1) values as e4m3 codes (uint8) or bf16, drawn in slices of the first axis."""
    out = torch.empty(shape, dtype=torch.uint8 if dtype == "e4m3" else torch.bfloat16, device=dev)
    rows = max(1, (1 << 27) // max(1, out[0].numel()))
    for i in range(0, shape[0], rows):
        x = torch.randn(out[i:i + rows].shape, generator=g, device=dev)
        out[i:i + rows] = x.to(torch.float8_e4m3fn).view(torch.uint8) if dtype == "e4m3" else x.to(torch.bfloat16)
    return out


def _tables(new, ctx, spare, g, dev):
    """Page ids of every request in a random order of the pool: [batch, widest] int32, -1 behind a request's pages."""
    need = torch.tensor([_pages(n + x) for n, x in zip(new, ctx)], device=dev)
    width, total = int(max(_pages(n + x) for n, x in zip(new, ctx))), sum(_pages(n + x) for n, x in zip(new, ctx))
    ids = torch.randperm(total + spare, generator=g, device=dev).to(torch.int32)
    first = need.cumsum(0) - need
    col = torch.arange(width, device=dev)[None, :]
    return torch.where(col < need[:, None], ids[(first[:, None] + col).clamp(max=total - 1)], -1).to(torch.int32), total + spare


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    new, ctx = _lens(case)
    T, B = sum(new), case["batch"]
    i32 = dict(dtype=torch.int32, device=dev)
    s = dict(op=case["op"], new=torch.tensor(new, **i32), ctx=torch.tensor(ctx, **i32), T=T)
    if case["op"] == "plan":
        # a pool in use: the cached tokens' pages are in the table, the new ones come off the free list; the token
        # buffers of a captured step are a little longer than the tokens at hand
        width = max(_pages(n + x) for n, x in zip(new, ctx)) + 2
        old = sum(_pages(x) for x in ctx)
        fresh = sum(_pages(n + x) - _pages(x) for n, x in zip(new, ctx))
        s["num_pages"] = old + fresh + 40
        ids = torch.randperm(s["num_pages"], generator=g, device=dev).to(torch.int32)
        have = torch.tensor([_pages(x) for x in ctx], device=dev)
        first = have.cumsum(0) - have
        col = torch.arange(width, device=dev)[None, :]
        s["table"] = torch.where(col < have[:, None], ids[(first[:, None] + col).clamp(max=max(old - 1, 0))], -1).to(torch.int32)
        s["free"] = ids[old:].contiguous()
        s["n_free"] = torch.tensor([s["num_pages"] - old - 7], **i32)
        s["rows"] = (T + 63) // 64 * 64
        return s
    s["table"], P = _tables(new, ctx, 3, g, dev)
    D, hkv, dt = case["dim"], case["kv_heads"], case["dtype"]
    s["kcache"] = _values((P, hkv, PAGE, D), dt, g, dev)
    s["vcache"] = _values((P, hkv, D, PAGE), dt, g, dev)
    s["cu"] = torch.cat([torch.zeros(1, **i32), s["new"].cumsum(0).to(torch.int32)])
    s["seqlens"] = s["ctx"] + s["new"]
    s["most_new"], s["most_pages"] = max(new), max(_pages(n + x) for n, x in zip(new, ctx))
    if case["op"] == "append":
        s["k"], s["v"] = _values((T, hkv, D), dt, g, dev), _values((T, hkv, D), dt, g, dev)
        req, idx = _rows(s)
        pos = (s["ctx"][req] + idx).long()
        s["slots"] = s["table"][req, pos // PAGE].long() * PAGE + pos % PAGE
        return s
    s["q"] = _values((T, case["q_heads"], D), dt, g, dev)
    s["gate"] = _values((T, case["q_heads"], D), "bf16", g, dev) if case["gate"] else None
    s["scale"] = 1.0 / math.sqrt(D)
    return s


def _rows(s):
    """Request and place within it of every token row."""
    t = torch.arange(s["T"], dtype=torch.int32, device=s["cu"].device)
    req = torch.searchsorted(s["cu"], t, right=True) - 1
    return req, t - s["cu"][req]


# ---- one pass --------------------------------------------------------------------------------------------------
def run(state):
    s = state
    if own:
        from bundles_b200 import ops
        if s["op"] == "plan":
            p = ops.page_plan(s["ctx"], s["new"], s["table"], s["num_pages"], s["rows"], free_pages=s["free"], n_free=s["n_free"])
            return [p.cu_seqlens, p.seqlens, p.positions, p.slots, s["table"], p.n_left]
        if s["op"] == "append":
            ops.kv_append(s["k"], s["v"], s["kcache"], s["vcache"], s["slots"])
            return _cache_values(s)
        return ops.attn_extend(s["q"], s["gate"], s["kcache"], s["vcache"], s["table"], s["cu"], s["seqlens"], scale=s["scale"])
    return {"plan": _plain_plan, "append": _plain_append, "attend": _plain_attend}[s["op"]](s)


def _cache_values(s):
    """The caches as the values that their codes stand for."""
    e4m3 = s["kcache"].dtype == torch.uint8
    return [c.view(torch.float8_e4m3fn) if e4m3 else c for c in (s["kcache"], s["vcache"])]


def _plain_plan(s):
    dev, B, R = s["ctx"].device, s["ctx"].shape[0], s["rows"]
    total = s["new"].cumsum(0)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), total]).to(torch.int32)
    seqlens = s["ctx"] + s["new"]
    have, need = (s["ctx"] + PAGE - 1) // PAGE, (seqlens + PAGE - 1) // PAGE
    taken = (need - have).cumsum(0)
    first = taken - (need - have)
    col = torch.arange(s["table"].shape[1], device=dev)[None, :]
    k = (first[:, None] + col - have[:, None]).clamp(min=0)
    fresh = s["free"][(s["n_free"] - 1 - k).clamp(min=0).long()]
    s["table"].copy_(torch.where((col >= have[:, None]) & (col < need[:, None]), fresh, s["table"]))
    t = torch.arange(R, device=dev, dtype=torch.int32)
    req = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=B - 1)
    pos = (s["ctx"][req] + t - cu[req]).long()
    live = t < cu[-1]
    slot = s["table"][req, (pos // PAGE).clamp(max=s["table"].shape[1] - 1)].long() * PAGE + pos % PAGE
    return [cu, seqlens, torch.where(live, pos, 0), torch.where(live, slot, -1), s["table"], s["n_free"] - taken[-1].to(torch.int32)]


def _plain_append(s):
    page, o = s["slots"] // PAGE, s["slots"] % PAGE
    s["kcache"][page, :, o] = s["k"]
    s["vcache"][page, :, :, o] = s["v"]
    return _cache_values(s)


def _floats(x):
    return x.view(torch.float8_e4m3fn).float() if x.dtype == torch.uint8 else x.float()


def _plain_attend(s):
    """All requests at once, padded to the most new tokens and the longest history, in fp32."""
    B, N, M = s["table"].shape[0], s["most_new"], s["most_pages"]
    T, hq, D = s["q"].shape
    hkv = s["kcache"].shape[1]
    pages = s["table"][:, :M].clamp(min=0).long()
    k = _floats(s["kcache"][pages]).permute(0, 2, 1, 3, 4).reshape(B, hkv, M * PAGE, D)
    key = torch.arange(M * PAGE, device=pages.device)
    i = torch.arange(N, device=pages.device)
    rows = (s["cu"][:-1, None] + i).clamp(max=T - 1).long()
    q = _floats(s["q"][rows]).reshape(B, N, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, D)
    p = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(B, hkv, hq // hkv, N, M * PAGE)
    del k
    p.masked_fill_((key > (s["ctx"][:, None] + i)[:, :, None])[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    v = _floats(s["vcache"][pages]).permute(0, 2, 1, 4, 3).reshape(B, hkv, M * PAGE, D)
    v = torch.where((key < s["seqlens"][:, None])[:, None, :, None], v, 0.0)
    o = (p.view(B, hkv, -1, M * PAGE) @ v).view(B, hkv, hq // hkv, N, D) / total
    req, at = _rows(s)
    o = o.permute(0, 3, 1, 2, 4)[req, at].reshape(T, hq, D)
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.to(torch.bfloat16).reshape(T, hq * D)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    new, ctx = _lens(case)
    T, B = sum(new), case["batch"]
    if case["op"] == "plan":  # lengths in; cu, seqlens, positions, slots and the new table entries out
        fresh = sum(_pages(n + x) - _pages(x) for n, x in zip(new, ctx))
        return {"bytes": 8 * B + 8 * B + 16 * T + 8 * fresh + 8, "flops": 0}
    esize = 1 if case["dtype"] == "e4m3" else 2
    row = case["kv_heads"] * case["dim"] * esize
    if case["op"] == "append":  # K and V in and out
        return {"bytes": 4 * T * row + 8 * T, "flops": 0}
    keys = sum(n + x for n, x in zip(new, ctx))
    seen = sum(n * x + n * (n + 1) // 2 for n, x in zip(new, ctx))
    qd = case["q_heads"] * case["dim"]
    return {"bytes": 2 * keys * row + T * qd * (esize + 2 + (2 if case["gate"] else 0)) + 4 * sum(_pages(n + x) for n, x in zip(new, ctx)),
            "flops": 4 * qd * seen}


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _decoded(x):
    """e4m3 codes by their bits, or bf16 values, as fp64."""
    if x.dtype != torch.uint8:
        return x.double()
    code = torch.arange(256, device=x.device)
    e, m = (code >> 3) & 15, (code & 7).double()
    mag = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e.double() - 10))
    mag = torch.where((code & 127) == 127, math.nan, mag)
    return torch.where(code >= 128, -mag, mag)[x.long()]


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    new, ctx = _lens(case)
    if case["op"] == "append":  # a token's K is one row of its page, its V one column
        kc, vc = _decoded(s["kcache"]), _decoded(s["vcache"]).transpose(2, 3).contiguous()
        for cache, x in ((kc, s["k"]), (vc, s["v"])):
            flat = cache.transpose(1, 2).reshape(-1, *x.shape[1:])  # [slot, kv head, dim]
            flat[s["slots"]] = _decoded(x)
            cache.copy_(flat.view(cache.shape[0], PAGE, *x.shape[1:]).transpose(1, 2))
        return [kc, vc.transpose(2, 3).contiguous()]
    T, hq, D = s["q"].shape
    hkv = case["kv_heads"]
    grp = hq // hkv
    out = torch.empty(T, hq, D, dtype=torch.float64, device=s["q"].device)
    t0 = 0
    for b, (n, c) in enumerate(zip(new, ctx)):
        ids = s["table"][b, :_pages(n + c)].long()
        for h in range(hkv):
            keys = _decoded(s["kcache"][ids, h]).reshape(-1, D)[:n + c]
            vals = _decoded(s["vcache"][ids, h]).transpose(1, 2).reshape(-1, D)[:n + c]
            for i in range(0, n, 256):
                m = min(256, n - i)
                q = _decoded(s["q"][t0 + i:t0 + i + m, h * grp:(h + 1) * grp])
                score = torch.einsum("mgd,kd->mgk", q, keys) * s["scale"]
                hidden = torch.arange(n + c, device=q.device)[None, :] > torch.arange(c + i, c + i + m, device=q.device)[:, None]
                weight = torch.softmax(score.masked_fill(hidden[:, None, :], -math.inf), dim=-1)
                out[t0 + i:t0 + i + m, h * grp:(h + 1) * grp] = torch.einsum("mgk,kd->mgd", weight, vals)
        t0 += n
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out.reshape(T, hq * D)
