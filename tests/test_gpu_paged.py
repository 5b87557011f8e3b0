"""Block tables and slots from request lengths, the append, and the three paged operators as a server runs them."""
import numpy as np
import pytest
import torch

import paged_util as pu
from oracle import paged as op

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _plan(ctx, new, W, T, P, free=None, n_free=None, seed=0, spoil=None):
    from bundles_b200 import ops
    r = np.random.RandomState(seed)
    B = len(ctx)
    table = np.full((B, W), -9, np.int32)
    ids = r.permutation(P).astype(np.int32)
    at = 0
    for b in range(B):
        have = min(W, max(0, -(-ctx[b] // 128)))
        table[b, :have] = ids[at:at + have]
        at += have
    if free is None:
        free = ids[at:].copy()
    if spoil is not None:
        spoil(table, free)
    n_free = len(free) if n_free is None else n_free
    ref = op.page_plan(ctx, new, table, P, T, free, n_free)
    d = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)  # noqa: E731
    tab, status = torch.from_numpy(table).to(DEV), ops.new_status(DEV)
    n = d([n_free])
    p = ops.page_plan(d(ctx), d(new), tab, P, T, torch.from_numpy(free).to(DEV), n, status=status)
    torch.cuda.synchronize()
    got = [t.cpu().numpy() for t in (p.cu_seqlens, p.seqlens, p.positions, p.slots, tab)] + [int(p.n_left)]
    for name, a, b in zip(("cu", "seqlens", "positions", "slots", "table", "n_left"), got, ref):
        assert np.array_equal(a, b), name
    assert int(n) == n_free
    st = ops.read_status(status)
    assert (st in ref[6]) if ref[6] else st == 0
    return ref


@pytest.mark.parametrize("B,T,seed", [(1, 1, 1), (7, 500, 2), (300, 1111, 3), (1025, 4000, 4)])
def test_page_plan_matches_oracle(B, T, seed):
    r = np.random.RandomState(seed)
    ctx = r.randint(0, 700, B)
    new = r.multinomial(T - T // 9, r.dirichlet(np.ones(B) * 0.3)).astype(int)
    ctx[r.rand(B) < 0.2] = 0
    ctx[r.rand(B) < 0.2] = 128 * r.randint(1, 5)
    W = max(-(-(c + n) // 128) for c, n in zip(ctx, new)) + 1
    P = int(sum(-(-(c + n) // 128) for c, n in zip(ctx, new))) + 5
    ref = _plan(ctx.tolist(), new.tolist(), W, T, P, seed=seed)
    assert not ref[6]


def test_page_plan_largest_batch():
    r = np.random.RandomState(9)
    ctx, new = r.randint(0, 400, 8192), r.randint(0, 4, 8192)
    assert not _plan(ctx.tolist(), new.tolist(), 4, int(new.sum()) + 3, 40000, seed=9)[6]


def test_page_plan_shortages_and_bad_values():
    codes = _plan([100, 0, 250], [300, 200, 10], 4, 600, 20, n_free=2)[6]     # two pages for five
    assert codes == {111}
    assert _plan([100, 500], [300, 20], 4, 400, 20)[6] == {111}               # the table ends inside the second request
    assert _plan([100, -5, 0], [3, 7, -2], 4, 64, 20)[6] == {113}             # negative lengths count as 0
    assert _plan([10, 20, 30], [30, 30, 30], 2, 70, 9)[6] == {113}            # the rows end inside the last request
    assert _plan([10, 20, 30], [0, 0, 0], 2, 5, 9)[6] == set()                # nothing new

    def spoil(table, free):
        table[0, 0] = 99
        free[-1] = -3
        free[-2] = 1 << 20
    assert _plan([100, 0, 0], [5, 129, 1], 4, 140, 20, spoil=spoil)[6] == {112}


def test_page_plan_without_a_free_list():
    from bundles_b200 import ops
    table = torch.arange(12, dtype=torch.int32, device=DEV).flip(0).reshape(3, 4).contiguous()
    ctx, new = [130, 0, 383], [200, 1, 2]
    ref = op.page_plan(ctx, new, table.cpu().numpy(), 12, 210)
    keep = table.clone()
    p = ops.page_plan(torch.tensor(ctx, dtype=torch.int32, device=DEV), torch.tensor(new, dtype=torch.int32, device=DEV), table, 12,
                      210)
    torch.cuda.synchronize()
    for a, b in zip(p[:4], ref[:4]):
        assert np.array_equal(a.cpu().numpy(), b)
    assert torch.equal(table, keep)


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
@pytest.mark.parametrize("heads", [(2, 256), (4, 128), (1, 256)])
def test_kv_append_matches_oracle(dtype, heads):
    """Single tokens, runs inside a page, runs over page edges at every alignment, skipped rows; nothing else moves."""
    from bundles_b200 import ops
    hkv, D = heads
    g = torch.Generator().manual_seed(31)
    rnd = pu.e4 if dtype == "e4m3" else pu.bf
    P = 40
    pages = torch.randperm(P, generator=g).tolist()
    slots = []
    for start, n in ((0, 1), (127, 1), (5, 1), (3, 200), (16, 16), (17, 15), (32, 300), (120, 9), (64, 64), (1, 127), (0, 128)):
        ids = [pages.pop() for _ in range(-(-(start + n) // 128))]
        slots += [ids[(start + i) // 128] * 128 + (start + i) % 128 for i in range(n)]
        slots += [-1] * (start % 3)
    slots += [P * 128, 1 << 40]                                     # outside the pool
    T = len(slots)
    k, v, kc, vc = rnd(g, T, hkv, D), rnd(g, T, hkv, D), rnd(g, P, hkv, 128, D), rnd(g, P, hkv, D, 128)
    raw = lambda t: t.view(torch.int16).numpy() if t.dtype == torch.bfloat16 else t.numpy()  # noqa: E731
    rk, rv = op.kv_append(raw(k), raw(v), raw(kc), raw(vc), slots)
    sl, status = torch.tensor(slots, dtype=torch.int64, device=DEV), ops.new_status(DEV)
    for pad in (0, 1):                                              # tokens side by side, then rows of a wider tensor
        wide = torch.zeros(T, hkv + pad, D, dtype=k.dtype)
        wide[:, :hkv] = k
        a, b = kc.to(DEV), vc.to(DEV)
        ops.kv_append(wide.to(DEV)[:, :hkv], v.to(DEV), a, b, sl, status=status)
        torch.cuda.synchronize()
        assert ops.read_status(status) == 112
        assert np.array_equal(raw(a.cpu()), rk) and np.array_equal(raw(b.cpu()), rv)


def test_kv_append_of_nothing():
    from bundles_b200 import ops
    kc, vc = torch.zeros(2, 1, 128, 128, dtype=torch.uint8, device=DEV), torch.zeros(2, 1, 128, 128, dtype=torch.uint8, device=DEV)
    e = torch.empty(0, 1, 128, dtype=torch.uint8, device=DEV)
    ops.kv_append(e, e, kc, vc, torch.empty(0, dtype=torch.int64, device=DEV))
    ops.kv_append(torch.ones(3, 1, 128, dtype=torch.uint8, device=DEV), torch.ones(3, 1, 128, dtype=torch.uint8, device=DEV), kc, vc,
                  torch.full((3,), -1, dtype=torch.int64, device=DEV))
    torch.cuda.synchronize()
    assert not kc.any() and not vc.any()


@pytest.mark.parametrize("dtype", ["e4m3", "bf16"])
def test_a_server_of_the_three(dtype):
    """Prompts in chunks, then decode, through the three operators captured in one graph per row count; every step's
    output is compared with the oracle on the whole history."""
    from bundles_b200 import ops
    hq, hkv, D, P, W, B = 16, 2, 256, 24, 6, 3
    g = torch.Generator().manual_seed(41)
    rnd = pu.e4 if dtype == "e4m3" else pu.bf
    dt = torch.uint8 if dtype == "e4m3" else torch.bfloat16
    nan = 0x7f if dtype == "e4m3" else float("nan")
    kc = torch.full((P, hkv, 128, D), nan, dtype=dt, device=DEV)
    vc = torch.full((P, hkv, D, 128), nan, dtype=dt, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.full((B, W), -1, **i32)
    free = torch.randperm(P, generator=g).to(torch.int32).to(DEV)
    n_free, ctx, new = torch.full((1,), P, **i32), torch.zeros(B, **i32), torch.zeros(B, **i32)
    status = ops.new_status(DEV)
    rows = 224
    k, v, q = (torch.zeros(rows, h, D, dtype=dt, device=DEV) for h in (hkv, hkv, hq))
    gate = torch.zeros(rows, hq, D, dtype=torch.bfloat16, device=DEV)
    out = torch.zeros(rows, hq * D, dtype=torch.bfloat16, device=DEV)

    def step():
        p = ops.page_plan(ctx, new, table, P, rows, free, n_free, status=status)
        ops.kv_append(k, v, kc, vc, p.slots, status=status)
        ops.attn_extend(q, gate, kc, vc, table, p.cu_seqlens, p.seqlens, out=out, status=status)
        n_free.copy_(p.n_left)
        ctx.copy_(p.seqlens)
        return p

    graph = torch.cuda.CUDAGraph()
    step()                                  # no new tokens: changes nothing
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan = step()
    hist_k = [np.zeros((0, hkv, D), np.float32) for _ in range(B)]
    hist_v = [np.zeros((0, hkv, D), np.float32) for _ in range(B)]
    raw = lambda t: op.e4m3_decode(t.numpy()) if dtype == "e4m3" else t.float().numpy()  # noqa: E731
    for lens in ([100, 0, 30], [100, 90, 1], [1, 130, 1], [1, 1, 1], [60, 1, 128], [0, 1, 0], [1, 1, 1]):
        T = sum(lens)
        hk, hv, hqq, hg = rnd(g, T, hkv, D), rnd(g, T, hkv, D), rnd(g, T, hq, D), pu.bf(g, T, hq, D)
        for dst, src in ((k, hk), (v, hv), (q, hqq), (gate, hg)):
            dst[:T] = src.to(DEV)
        new.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert ops.read_status(status) == 0
        at = 0
        for b, n in enumerate(lens):
            hist_k[b] = np.concatenate([hist_k[b], raw(hk[at:at + n])])
            hist_v[b] = np.concatenate([hist_v[b], raw(hv[at:at + n])])
            at += n
        # the oracle on pages laid out plainly from the whole history
        need = [-(-len(h) // 128) for h in hist_k]
        pk = np.zeros((sum(need), hkv, 128, D), np.float32)
        pv = np.zeros((sum(need), hkv, D, 128), np.float32)
        tab, base = np.full((B, W), -1, np.int32), 0
        for b in range(B):
            for j in range(len(hist_k[b])):
                pk[base + j // 128, :, j % 128] = hist_k[b][j]
                pv[base + j // 128, :, :, j % 128] = hist_v[b][j]
            tab[b, :need[b]] = np.arange(base, base + need[b])
            base += need[b]
        cu = np.concatenate([[0], np.cumsum(lens)])
        assert plan.cu_seqlens.tolist() == cu.tolist() and plan.seqlens.tolist() == [len(h) for h in hist_k]
        ref = op.attn_extend(raw(hqq), hg.float().numpy(), pk, pv, tab, cu, [len(h) for h in hist_k], D ** -0.5)
        pu.check(out[:T], dict(q=q[:T], cu_seqlens=torch.tensor(cu)), None, ref)
    assert int(n_free) == P - sum(need)


def test_torch_registry():
    import bundles_b200.torch_ops  # noqa: F401
    b = torch.ops.b200nodes
    d, scale = pu.make([(5, 200), (1, 30)], seed=51)
    c = pu.on(d, DEV)
    want = torch.empty(0)
    cu, sl, pos, slots, left = b.page_plan(torch.tensor([200, 30], dtype=torch.int32, device=DEV),
                                           torch.tensor([5, 1], dtype=torch.int32, device=DEV), c["page_table"], c["kcache"].shape[0],
                                           6, None, None)
    assert cu.tolist() == [0, 5, 6] and pos.tolist() == [200, 201, 202, 203, 204, 30]
    b.kv_append(pu.e4(torch.Generator().manual_seed(1), 6, 2, 256).to(DEV), pu.e4(torch.Generator().manual_seed(2), 6, 2, 256).to(DEV),
                c["kcache"], c["vcache"], slots)
    want = b.attn_extend(c["q"], c["gate"], c["kcache"], c["vcache"], c["page_table"], cu, sl, scale)
    torch.cuda.synchronize()
    host = {k: (t.cpu() if t is not None else None) for k, t in c.items()}
    pu.check(want, host, scale)
