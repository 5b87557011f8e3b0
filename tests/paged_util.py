"""Inputs and comparison shared by the tests of the paged-cache operators."""
import numpy as np
import torch

from oracle import paged as op

PAGE = 128


def e4(g, *shape):
    return torch.randn(*shape, generator=g).to(torch.float8_e4m3fn).view(torch.uint8)


def bf(g, *shape):
    return torch.randn(*shape, generator=g).to(torch.bfloat16)


def as_np(t):
    t = t.detach().cpu()
    return t.float().numpy() if t.dtype == torch.bfloat16 else t.numpy()


def make(batch, dtype="e4m3", heads=(16, 2, 256), gate=True, seed=0, pad_rows=0, width=None):
    """`batch`: (new, cached) tokens per request.  Everything that no request owns holds NaN: pages of nobody, the places
    behind a request's last token, the rows behind the last request; table entries behind the last page are out of range."""
    hq, hkv, D = heads
    g = torch.Generator().manual_seed(1000 + seed)
    rnd = e4 if dtype == "e4m3" else bf
    nan = 0x7f if dtype == "e4m3" else float("nan")
    B, T = len(batch), sum(n for n, _ in batch) + pad_rows
    need = [-(-(n + c) // PAGE) for n, c in batch]
    W = max(need + [1]) + 1 if width is None else width
    P = sum(need) + 3
    ids = torch.randperm(P, generator=g).to(torch.int32)
    table = torch.full((B, W), 1 << 30, dtype=torch.int32)
    kc, vc = rnd(g, P, hkv, PAGE, D), rnd(g, P, hkv, D, PAGE)
    at = 0
    for b, (n, c) in enumerate(batch):
        table[b, :min(W, need[b])] = ids[at:at + min(W, need[b])]
        at += need[b]
        if (n + c) % PAGE:
            kc[ids[at - 1].item(), :, (n + c) % PAGE:] = nan
            vc[ids[at - 1].item(), :, :, (n + c) % PAGE:] = nan
    for i in ids[at:].tolist():
        kc[i] = nan
        vc[i] = nan
    cu = torch.tensor([0] + list(np.cumsum([n for n, _ in batch])), dtype=torch.int32)
    q = rnd(g, T, hq, D)
    q[int(cu[-1]):] = nan
    return dict(q=q, gate=bf(g, T, hq, D) if gate else None, kcache=kc, vcache=vc, page_table=table, cu_seqlens=cu,
                seqlens=torch.tensor([n + c for n, c in batch], dtype=torch.int32)), D ** -0.5


def want(d, scale):
    return op.attn_extend(as_np(d["q"]), None if d["gate"] is None else as_np(d["gate"]), as_np(d["kcache"]), as_np(d["vcache"]),
                          as_np(d["page_table"]), as_np(d["cu_seqlens"]), as_np(d["seqlens"]), scale)


def on(d, dev):
    return {k: None if v is None else v.to(dev) for k, v in d.items()}


def check(got, d, scale, ref=None):
    """bf16 output: half a step of the result, 2^-8 relative (eps / 2).  Probabilities are kept to half a step of 2^-8 in
    the P . V product (bf16, or an e5m2 value plus an e4m3 remainder of the same total precision), which moves the result by
    at most 2^-8 times the spread, twice that where the row sum takes the rounded values too.  1/16 more for the fp32
    scores and exponentials (some 2^-18 relative).  The remainder's floor, 2^-10 against a largest probability of at least
    2^8 in the same units, adds at most 2^-18 per key, below the rest for the lengths here."""
    ref, spread = want(d, scale) if ref is None else ref
    T = d["q"].shape[0]
    n = int(d["cu_seqlens"][-1])
    got = got.detach().float().cpu().numpy().astype(np.float64).reshape(ref.shape)
    assert np.isfinite(got[:n]).all()
    err = np.abs(got[:n] - ref[:n])
    lim = 2.0 ** -8 * np.abs(ref[:n]) + 2.125 * 2.0 ** -8 * spread[:n] + 1e-30
    assert (err <= lim).all(), f"worst {np.max(err / lim)} of the limit, {T} rows"
    return err, ref
