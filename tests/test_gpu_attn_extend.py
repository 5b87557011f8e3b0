"""Attention of ragged chunks over the paged cache against the float64 oracle."""
import numpy as np
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)

BATCHES = {
    "first_token": [(1, 0)],
    "page_edges": [(1, 126), (1, 127), (1, 128), (4, 300), (2, 127)],
    "empty_requests": [(0, 50), (17, 0), (0, 0), (130, 5), (1, 777), (0, 1)],
    "one_chunk": [(257, 383)],
    "split_keys": [(1, 5000), (3, 2049)],
}


def _run(d, scale, **kw):
    from bundles_b200 import ops
    status = ops.new_status(DEV)
    out = ops.attn_extend(**pu.on(d, DEV), scale=scale, status=status, **kw)
    torch.cuda.synchronize()
    return out, ops.read_status(status)


@pytest.mark.parametrize("batch", list(BATCHES))
@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
@pytest.mark.parametrize("heads", [(16, 2, 256), (12, 4, 128)])
def test_matches_oracle(batch, dtype, heads):
    d, scale = pu.make(BATCHES[batch], dtype, heads, seed=len(batch))
    out, st = _run(d, scale)
    assert st == 0
    pu.check(out, d, scale)


@pytest.mark.parametrize("heads,dtype", [((8, 1, 256), "e4m3"), ((4, 4, 128), "e4m3"), ((40, 2, 128), "bf16"),
                                         ((20, 1, 256), "bf16"), ((128, 1, 128), "e4m3"), ((5, 5, 256), "e4m3")])
def test_head_layouts(heads, dtype):
    d, scale = pu.make([(1, 200), (9, 121), (40, 0)], dtype, heads, gate=False, seed=heads[0])
    out, st = _run(d, scale)
    assert st == 0
    pu.check(out, d, scale)


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
def test_many_requests(dtype):
    """More requests than a warp and than the GPU has SMs, among them empty ones."""
    r = np.random.RandomState(3)
    batch = [(int(r.choice([0, 1, 1, 1, 2, 5])), int(r.randint(0, 300))) for _ in range(333)]
    d, scale = pu.make(batch, dtype, (8, 2, 128), seed=5)
    out, st = _run(d, scale)
    assert st == 0
    pu.check(out, d, scale)


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
def test_rows_that_see_nothing_and_rows_of_nobody(dtype):
    """seqlens below the new tokens: the first rows see no key and are zero.  Rows behind the last request stay."""
    d, scale = pu.make([(6, 0), (3, 130), (140, 20)], dtype, seed=8, pad_rows=9)
    d["seqlens"] = torch.tensor([2, 0, 150], dtype=torch.int32)
    from bundles_b200 import ops
    out = torch.full((d["q"].shape[0], 4096), 7.0, dtype=torch.bfloat16, device=DEV)
    assert ops.attn_extend(**pu.on(d, DEV), scale=scale, out=out) is out
    torch.cuda.synchronize()
    n = int(d["cu_seqlens"][-1])
    assert (out[n:] == 7.0).all()
    assert (out[:4] == 0).all() and (out[6:9] == 0).all()
    pu.check(out, d, scale)


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
def test_pages_outside_the_pool_are_masked(dtype):
    d, scale = pu.make([(1, 1000), (33, 500)], dtype, seed=11)
    d["page_table"][0, 3] = -1
    d["page_table"][0, 7] = d["kcache"].shape[0]
    d["page_table"][1, 0] = -2147483648
    out, st = _run(d, scale)
    assert st == 112
    pu.check(out, d, scale)
    d["page_table"][:] = -5    # nothing left to see
    out, st = _run(d, scale)
    assert st == 112 and (out == 0).all()


def test_table_narrower_than_the_request():
    d, scale = pu.make([(5, 300)], seed=12, width=2)
    out, st = _run(d, scale)
    assert st == 112
    pu.check(out, d, scale)


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
def test_token_strides(dtype):
    """q and gate as slices of wider rows (a fused projection's output)."""
    d, scale = pu.make([(3, 140), (50, 90)], dtype, seed=13)
    from bundles_b200 import ops
    c = pu.on(d, DEV)
    T = c["q"].shape[0]
    for name, pad in (("q", 2), ("gate", 1)):
        wide = torch.zeros(T, 16 + pad, 256, dtype=c[name].dtype, device=DEV)
        wide[:, :16] = c[name]
        c[name] = wide[:, :16]
    out = ops.attn_extend(**c, scale=scale)
    plain, _ = _run(d, scale)
    assert torch.equal(out, plain)
    pu.check(out, d, scale)


def test_extreme_scores():
    """Scores far apart (one key takes all), all equal (zero queries) and a maximum that keeps rising along the keys."""
    d, scale = pu.make([(2, 700), (20, 260)], "bf16", seed=14)
    q = d["q"].float()
    q[0] *= 60.0
    q[1] = 0.0
    d["q"] = q.to(torch.bfloat16)
    out, _ = _run(d, scale)
    pu.check(out, d, scale)
    d, scale = pu.make([(1, 1500)], "e4m3", seed=15)
    base = torch.randn(256, generator=torch.Generator().manual_seed(2))
    d["q"][:] = base.to(torch.float8_e4m3fn).view(torch.uint8)
    k = torch.zeros(1501, 256)
    k[:] = base * (torch.arange(1501.0) / 700.0)[:, None]        # rising scores: the running maximum moves on every page
    codes = k.to(torch.float8_e4m3fn).view(torch.uint8)
    for j in range(12):
        n = min(128, 1501 - j * 128)
        d["kcache"][int(d["page_table"][0, j]), :, :n] = codes[j * 128:j * 128 + n]
    out, _ = _run(d, scale)
    pu.check(out, d, scale)


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
def test_a_dominant_first_key(dtype):
    """One key far above a long even tail: the tail still has to count (each of its weights is 2^-11 of the first)."""
    d, scale = pu.make([(1, 4000)], dtype, seed=16)
    val = (lambda t: t.to(torch.float8_e4m3fn).view(torch.uint8)) if dtype == "e4m3" else (lambda t: t.to(torch.bfloat16))
    d["q"][:] = val(torch.ones(1, 16, 256))
    first = int(d["page_table"][0, 0])
    for j in range(32):
        page, n = int(d["page_table"][0, j]), min(128, 4001 - j * 128)
        d["kcache"][page, :, :n] = val(torch.zeros(2, n, 256))
        d["vcache"][page, :, :, :n] = val(torch.ones(2, 256, n))
    d["kcache"][first, :, 0] = val(torch.full((2, 256), 0.46875))   # 7.5 nats: e^7.5 = 2^10.8
    d["vcache"][first, :, :, 0] = val(torch.zeros(2, 256))
    out, _ = _run(d, scale)
    pu.check(out, d, scale)
    assert float(out.float().abs().max()) > 0.3


def test_same_bits_twice_and_with_a_given_workspace():
    from bundles_b200 import ops
    d, scale = pu.make([(1, 3000), (200, 900), (7, 0)], seed=17)
    c = pu.on(d, DEV)
    a = ops.attn_extend(**c, scale=scale)
    ws = ops.attn_extend_workspace(c["q"].shape[0], 16, 2, 256, DEV)
    ws.fill_(255)
    b = ops.attn_extend(**c, scale=scale, ws=ws)
    e = ops.attn_extend(**c, scale=scale, ws=ws)
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, e)


def test_agrees_with_the_verify_core_on_four_drafts():
    from bundles_b200 import ops, synth
    cfg = pu.on(synth.attn_verify(seed=77, B=3, ctx=700, ragged=True), DEV)
    ref = ops.attn_verify(cfg["q"], cfg["gate"], cfg["k_new"], cfg["v_new"], cfg["kcache"], cfg["vcache"], cfg["page_table"],
                          cfg["seqlens"])
    cu = torch.arange(0, 13, 4, dtype=torch.int32, device=DEV)
    out = ops.attn_extend(cfg["q"], cfg["gate"], cfg["kcache"], cfg["vcache"], cfg["page_table"], cu, cfg["seqlens"])
    torch.cuda.synchronize()
    host = dict(q=cfg["q"], gate=cfg["gate"], kcache=cfg["kcache"], vcache=cfg["vcache"], page_table=cfg["page_table"],
                cu_seqlens=cu, seqlens=cfg["seqlens"])
    _, want = pu.check(out, host, 1 / 16)
    # the verify core rounds the normalised row to bf16 before the gate: half a step more
    assert np.all(np.abs(ref.float().cpu().numpy().reshape(want.shape) - want) <= 2.0 ** -6 * np.maximum(np.abs(want), 0.25))


def test_other_stream_and_graph_replay_with_new_lengths():
    """Captured once, replayed with other lengths, tables and contents in the same buffers."""
    from bundles_b200 import ops
    first, scale = pu.make([(1, 400), (30, 100), (1, 5)], seed=18, width=8)
    second, _ = pu.make([(20, 0), (1, 600), (11, 130)], seed=19, width=8)
    assert first["q"].shape == second["q"].shape
    P = max(first["kcache"].shape[0], second["kcache"].shape[0])
    c = pu.on(first, DEV)
    for n in ("kcache", "vcache"):
        c[n] = torch.zeros(P, *first[n].shape[1:], dtype=torch.uint8, device=DEV)
        c[n][:first[n].shape[0]] = first[n].to(DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        eager = ops.attn_extend(**c, scale=scale)
    st.synchronize()
    pu.check(eager, first, scale)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.attn_extend(**c, scale=scale)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    for n in ("q", "gate", "page_table", "cu_seqlens", "seqlens"):
        c[n].copy_(second[n])
    for n in ("kcache", "vcache"):
        c[n][:second[n].shape[0]] = second[n].to(DEV)
    graph.replay()
    torch.cuda.synchronize()
    pu.check(out, second, scale)


def test_pool_past_four_gigabytes():
    """Page offsets beyond 2^32 bytes."""
    from bundles_b200 import ops
    d, scale = pu.make([(3, 290), (1, 128)], seed=20)
    P = 66000
    kc = torch.empty(P, 2, 128, 256, dtype=torch.uint8, device=DEV)
    vc = torch.empty(P, 2, 256, 128, dtype=torch.uint8, device=DEV)
    c = pu.on(d, DEV)
    n = c["kcache"].shape[0]
    kc[P - n:] = c["kcache"]
    vc[P - n:] = c["vcache"]
    c["kcache"], c["vcache"] = kc, vc
    c["page_table"] = torch.where(c["page_table"] < n, c["page_table"] + (P - n), c["page_table"]).to(torch.int32)
    out = ops.attn_extend(**c, scale=scale)
    torch.cuda.synchronize()
    pu.check(out, d, scale)


def test_lengths_that_are_nonsense_stay_in_bounds():
    """Row bounds outside [0, T), a request that runs backwards, lengths below zero and far beyond the table: the sound rows are
    right, the clamped ones are written inside the output, nothing else is."""
    from bundles_b200 import ops
    d, scale = pu.make([(6, 200), (4, 30), (10, 90)], seed=23)
    c = pu.on(d, DEV)
    whole = ops.attn_extend(**c, scale=scale)
    i32 = dict(dtype=torch.int32, device=DEV)
    out = torch.full_like(whole, 7.0)
    c["cu_seqlens"] = torch.tensor([-50, 6, 3, 20], **i32)         # rows 0..5, none, 3..19: the last two requests lie
    c["seqlens"] = torch.tensor([206, -2147483648, 100], **i32)
    c["cu_seqlens"][3] = 3                                          # ... the last has none either
    ops.attn_extend(**c, scale=scale, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out[:6], whole[:6]) and (out[6:] == 7.0).all()
    c["cu_seqlens"] = torch.tensor([0, 6, 10, 2147483647], **i32)   # the last request's rows end with the buffer
    c["seqlens"] = torch.tensor([206, 34, 100], **i32)
    ops.attn_extend(**c, scale=scale, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out, whole)
    c["seqlens"] = torch.tensor([2147483647, -5, 2147483647], **i32)  # everything in the table is seen; nothing is
    ops.attn_extend(**c, scale=scale, out=out)
    torch.cuda.synchronize()
    assert torch.isnan(out[:6]).all() and (out[6:10] == 0).all()


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
@pytest.mark.parametrize("heads", [(16, 2, 256), (12, 4, 128)])
def test_back_to_back_calls_of_changing_shape(dtype, heads):
    """Calls of many shapes in a row on one stream, every output as from a call alone: items of one page between long ones,
    warps without rows, cut and whole tiles."""
    from bundles_b200 import ops
    sets = []
    for k, b in enumerate(([(1, 60)] * 40, [(1, 5000)], [(300, 10)], [(1, 0), (90, 1000), (1, 127)], [(2, 64)] * 7)):
        d, scale = pu.make(b, dtype, heads, seed=60 + k)
        sets.append(pu.on(d, DEV))
    status = ops.new_status(DEV)
    alone = []
    for c in sets:
        alone.append(ops.attn_extend(**c, scale=scale))
        torch.cuda.synchronize()
    for _ in range(20):
        outs = [ops.attn_extend(**c, scale=scale, status=status) for c in sets]
    torch.cuda.synchronize()
    assert ops.read_status(status) == 0
    assert all(torch.equal(a, b) for a, b in zip(outs, alone))


def test_two_streams_at_once():
    from bundles_b200 import ops
    cases = [pu.make([(1, 3000), (70, 200)], seed=70 + k)[0] for k in range(2)]
    dev = [pu.on(d, DEV) for d in cases]
    want = [ops.attn_extend(**c) for c in dev]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(ops.attn_extend(**dev[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(o, want[k]) for o in got[k])


def test_refusals_of_tensors_that_do_not_fit():
    from bundles_b200 import ops
    d, _ = pu.make([(3, 140)], seed=80)
    c = pu.on(d, DEV)

    def bad(match, **kw):
        with pytest.raises(ops.B200Error, match=match):
            ops.attn_extend(**{**c, **kw})
    bad("must be", q=c["q"].to(torch.bfloat16))
    bad("must be", q=c["q"][:, :, :128].contiguous())
    bad("contiguous", q=c["q"].transpose(0, 1).contiguous().transpose(0, 1))
    bad("row per token", gate=c["gate"][:2])
    bad("fit together", cu_seqlens=c["cu_seqlens"][:1].contiguous())
    bad("CUDA", seqlens=c["seqlens"].cpu())
    bad("CUDA", page_table=c["page_table"].cpu())
    bad("K \\[pages", vcache=c["vcache"].transpose(2, 3).contiguous())
    bad("out must be", out=torch.empty(3, 4000, dtype=torch.bfloat16, device=DEV))
    bad("code -1", scale=0.0)
    bad("code -3", ws=torch.empty(64, dtype=torch.uint8, device=DEV))
    bad("code -2", q=torch.zeros(3 * 4096 + 1, dtype=torch.uint8, device=DEV)[1:].view(3, 16, 256))
    assert ops.attn_extend(c["q"][:0], c["gate"][:0], *[c[n] for n in ("kcache", "vcache", "page_table", "cu_seqlens", "seqlens")]).shape == (0, 4096)


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("heads,dtype", [((16, 2, 256), "e4m3"), ((16, 2, 256), "bf16"), ((12, 4, 128), "e4m3"), ((4, 4, 128), "bf16")])
def test_values_that_are_not_finite_reach_the_rows_that_see_them_only(heads, dtype, gate):
    """NaN and infinities in K and V of new tokens in the middle of a chunk: the rows before them are as the formula says, those
    from them on are not finite where the formula says so.  Whole tiles and cut ones, keys on two pages."""
    d, scale = pu.make([(40, 100), (150, 1900), (3, 126)], dtype, heads, gate=gate, seed=90)
    one = (lambda v: 0x7f) if dtype == "e4m3" else (lambda v: v)      # e4m3 has NaN only
    inf, nan = float("inf"), float("nan")
    for b, pos, dim, v in ((0, 127, 5, nan), (0, 128, 17, inf), (0, 135, 17, -inf), (1, 1910, 100, inf), (1, 1919, 3, nan),
                           (1, 2049, 64, -inf), (2, 128, 127, nan)):
        page = int(d["page_table"][b, pos // 128])
        d["vcache"][page, :, dim, pos % 128] = one(v)
    d["kcache"][int(d["page_table"][1, 2040 // 128]), :, 2040 % 128, 9] = one(nan)
    out, st = _run(d, scale)
    assert st == 0
    with np.errstate(all="ignore"):
        ref, spread = pu.want(d, scale)
    got = out.float().cpu().numpy().astype(np.float64).reshape(ref.shape)
    assert np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(np.isinf(got), np.isinf(ref))
    assert np.array_equal(np.sign(got[np.isinf(got)]), np.sign(ref[np.isinf(ref)]))
    fine = np.isfinite(ref)
    assert fine.mean() > 0.5 and not fine.all()
    err = np.abs(got[fine] - ref[fine])
    assert (err <= 2.0 ** -8 * np.abs(ref[fine]) + 2.125 * 2.0 ** -8 * spread[fine]).all()


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
def test_abandoned_waits_wind_down(dtype):
    """With a wait budget of one nanosecond the first wait that is not over at once gives up: the call ends with a status code,
    every role returns, and the next ordinary call gives the same bits as before."""
    from bundles_b200 import ops
    d, scale = pu.make([(300, 2000), (1, 5000), (70, 64)], dtype, seed=95)
    c = pu.on(d, DEV)
    want = ops.attn_extend(**c, scale=scale)
    torch.cuda.synchronize()
    bad = ops.new_status(DEV)
    ops.set_wait_budget_ns(1)
    try:
        ops.attn_extend(**c, scale=scale, status=bad)
        torch.cuda.synchronize()
    finally:
        ops.set_wait_budget_ns(0)
    assert ops.read_status(bad) in range(101, 107)
    st = ops.new_status(DEV)
    again = ops.attn_extend(**c, scale=scale, status=st)
    torch.cuda.synchronize()
    assert ops.read_status(st) == 0 and torch.equal(again, want)
