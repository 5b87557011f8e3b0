"""CPU checks of the paged-cache operators: refusals, and the oracle against a second statement of the definitions."""
import ctypes as C

import numpy as np
import pytest
import torch

from bundles_b200 import _lib, build, ops
from oracle import paged as op


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


one = C.c_void_p(4096)      # never dereferenced: the checks fail first
odd = C.c_void_p(4100)


def test_page_plan_refusals(lib):
    def call(ctx=one, B=2, W=4, P=8, free=one, cap=4, n_free=one, T=16, slots=one, left=one):
        return lib.b200_page_plan(ctx, one, B, one, W, P, free, cap, n_free, T, one, one, one, slots, left, None, None)
    assert call(ctx=None) == -1 and call(slots=None) == -1
    assert call(n_free=None) == -1 and call(left=None) == -1
    assert call(B=0) == -1 and call(B=8193) == -1 and call(T=0) == -1 and call(W=0) == -1 and call(P=0) == -1 and call(cap=0) == -1
    assert call(W=(1 << 23) + 1) == -1 and call(T=(1 << 29) + 1) == -1
    assert b"b200_page_plan" in lib.b200_last_error()


def test_kv_append_refusals(lib):
    def call(k=one, ks=512, vs=512, T=4, H=2, D=256, bf16=0, kc=one, P=8, slots=one):
        return lib.b200_kv_append(k, one, ks, vs, T, H, D, bf16, kc, one, P, slots, None, None)
    assert call(k=None) == -1 and call(slots=None) == -1
    assert call(T=-1) == -1 and call(H=0) == -1 and call(H=129) == -1 and call(D=192) == -1 and call(P=0) == -1
    assert call(ks=511) == -1 and call(vs=0) == -1
    assert call(k=odd) == -2 and call(kc=odd) == -2 and call(ks=520) == -2 and call(vs=516, bf16=1) == -2
    assert call(T=0) == 0


def test_attn_extend_refusals(lib):
    def call(q=one, qs=4096, gate=one, gs=4096, kc=one, P=8, W=4, B=2, T=16, hq=16, hkv=2, D=256, bf16=0, scale=0.0625, out=one,
             ws=one, n=1 << 30):
        return lib.b200_attn_extend(q, qs, gate, gs, kc, one, P, one, W, one, one, B, T, hq, hkv, D, bf16, scale, out, ws, n, None,
                                    None)
    for bad in (dict(q=None), dict(kc=None), dict(out=None), dict(ws=None), dict(B=0), dict(B=8193), dict(T=0), dict(T=(1 << 24) + 1),
                dict(P=0), dict(W=0), dict(W=(1 << 23) + 1), dict(hq=15), dict(hq=0), dict(hkv=0), dict(hq=258, hkv=2, qs=1 << 17, gs=1 << 17),
                dict(D=64), dict(P=1 << 23), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                dict(qs=4095), dict(gs=4000)):
        assert call(**bad) == -1, bad
    for bad in (dict(q=odd), dict(kc=odd), dict(out=odd), dict(ws=odd), dict(gate=odd), dict(qs=4100), dict(gs=4100)):
        assert call(**bad) == -2, bad
    need = lib.b200_attn_extend_workspace_bytes(16, 16, 2, 256)
    assert need > 0 and call(n=need - 1) == -3
    assert lib.b200_attn_extend_workspace_bytes(0, 16, 2, 256) == 0


def test_host_side_refusals():
    """The Python layer refuses before it reaches the library (CPU tensors are never accepted)."""
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ops.B200Error, match="CUDA"):
        ops.attn_extend(z(4, 16, 256), None, z(2, 2, 128, 256), z(2, 2, 256, 128), i(1, 2), i(2), i(1))
    with pytest.raises(ops.B200Error, match="e4m3 codes"):
        ops.attn_extend(z(4, 16, 256), None, z(2, 2, 128, 256, dt=torch.float16), z(2, 2, 256, 128), i(1, 2), i(2), i(1))
    with pytest.raises(ops.B200Error, match="CUDA"):
        ops.kv_append(z(4, 2, 256), z(4, 2, 256), z(2, 2, 128, 256), z(2, 2, 256, 128), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ops.B200Error, match="CUDA"):
        ops.page_plan(i(1), i(1), i(1, 2), 4, 8)


def test_oracle_plan_by_hand():
    table = np.array([[5, -9, -9], [7, 3, -9]], np.int32)
    cu, sl, pos, slots, tab, left, codes = op.page_plan([100, 256], [30, 2], table, 10, 34, np.array([1, 2, 8], np.int32), 2)
    assert cu.tolist() == [0, 30, 32] and sl.tolist() == [130, 258] and left == 0 and codes == set()
    assert tab.tolist() == [[5, 2, -9], [7, 3, 1]]
    assert pos[:32].tolist() == list(range(100, 130)) + [256, 257]
    assert slots[:32].tolist() == [5 * 128 + j for j in range(100, 128)] + [2 * 128, 2 * 128 + 1] + [128, 129]
    assert slots[32:].tolist() == [-1, -1] and pos[32:].tolist() == [0, 0]


def test_oracle_attention_against_dense():
    """One request over shuffled pages equals causal attention on the gathered rows."""
    r = np.random.RandomState(0)
    n, new, D = 200, 70, 16
    K, V, q = r.randn(n, 1, D), r.randn(n, 1, D), r.randn(new, 2, D)
    kc, vc = np.full((4, 1, 128, D), np.nan), np.full((4, 1, D, 128), np.nan)
    table = np.array([[3, 1]], np.int32)
    slots = [int(table[0, j // 128]) * 128 + j % 128 for j in range(n)]
    kc, vc = op.kv_append(K, V, kc, vc, slots)
    out, spread = op.attn_extend(q, None, kc, vc, table, [0, new], [n], 0.25)
    s = torch.einsum("tgd,kd->gtk", torch.from_numpy(q), torch.from_numpy(K[:, 0])) * 0.25
    hide = torch.arange(n)[None] > torch.arange(n - new, n)[:, None]
    p = torch.softmax(s.masked_fill(hide, float("-inf")), -1)
    ref = torch.einsum("gtk,kd->tgd", p, torch.from_numpy(V[:, 0])).numpy()
    assert np.abs(out - ref).max() < 1e-12 and (spread >= np.abs(out) - 1e-12).all()
