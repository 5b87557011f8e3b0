"""Oracle for the paged-cache operators: block tables and slots from request lengths, the append, ragged chunk attention.

Test infrastructure only (see oracle/__init__.py).  PARITY UNPINNED: the reference's nodes have no counterpart (its engine
builds tables on the host and its prefill and decode attention are library calls, attn_fused.py:158-162); these restate the
definitions in the public header, whole numbers exactly and the attention in float64.
"""
from __future__ import annotations

import numpy as np

from .numerics import e4m3_decode

PAGE = 128
ST_NO_PAGE, ST_BAD_PAGE, ST_BAD_LEN = 111, 112, 113


def page_plan(ctx, new, table, num_pages, T, free=None, n_free=0):
    """Returns (cu, seqlens, positions, slots, table', n_left, codes): `codes` is the set of status codes that apply."""
    B, W = table.shape
    table, codes = table.copy(), set()
    cu, seqlens = [0], []
    positions, slots = np.zeros(T, np.int64), np.full(T, -1, np.int64)
    n_free = 0 if free is None else max(0, min(int(n_free), len(free)))
    used = 0
    for b in range(B):
        c, n = int(ctx[b]), int(new[b])
        if c < 0 or n < 0:
            codes.add(ST_BAD_LEN)
        if c > W * PAGE:
            codes.add(ST_NO_PAGE)
        c, n = min(max(c, 0), W * PAGE), max(n, 0)
        if cu[-1] + n > T:
            codes.add(ST_BAD_LEN)
            n = T - cu[-1]
        have, need = -(-c // PAGE), -(-(c + n) // PAGE)
        if free is not None:
            for j in range(have, min(need, W)):
                pid = int(free[n_free - 1 - used]) if used < n_free else -1
                if used >= n_free:
                    codes.add(ST_NO_PAGE)
                elif not 0 <= pid < num_pages:
                    codes.add(ST_BAD_PAGE)
                    pid = -1
                table[b, j] = pid
                used += 1
        for i in range(n):
            pos = c + i
            positions[cu[-1] + i] = pos
            if pos // PAGE >= W:
                codes.add(ST_NO_PAGE)
                continue
            pid = int(table[b, pos // PAGE])
            if 0 <= pid < num_pages:
                slots[cu[-1] + i] = pid * PAGE + pos % PAGE
            elif pos // PAGE < have or free is None:
                codes.add(ST_BAD_PAGE)
        cu.append(cu[-1] + n)
        seqlens.append(c + n)
    return np.array(cu, np.int32), np.array(seqlens, np.int32), positions, slots, table, max(0, n_free - used), codes


def kv_append(k, v, kcache, vcache, slots):
    """k, v [T, Hkv, D], kcache [P, Hkv, 128, D], vcache [P, Hkv, D, 128]: any element type; copies returned."""
    kc, vc = kcache.copy(), vcache.copy()
    for t, s in enumerate(slots):
        if 0 <= s < kc.shape[0] * PAGE:
            kc[s // PAGE, :, s % PAGE, :] = k[t]
            vc[s // PAGE, :, :, s % PAGE] = v[t]
    return kc, vc


def attn_extend(q, gate, kcache, vcache, table, cu, seqlens, scale):
    """float64.  q, caches: uint8 e4m3 codes or float arrays; gate float or None.  Returns (out [T, Hq, D], spread), where
    spread = |gate factor| * sum_j p_j |v_j| / sum_j p_j: what a relative error of the weights is multiplied by.  Rows of
    no request are NaN."""
    val = lambda a: e4m3_decode(a).astype(np.float64) if a.dtype == np.uint8 else a.astype(np.float64)  # noqa: E731
    T, hq, D = q.shape
    P, hkv = kcache.shape[:2]
    g = hq // hkv
    out, spread = np.full((T, hq, D), np.nan), np.full((T, hq, D), np.nan)
    qf = val(q)
    for b in range(len(seqlens)):
        lo, hi, n = int(cu[b]), int(cu[b + 1]), int(seqlens[b])
        npages = -(-n // PAGE)
        ids = [int(table[b, j]) if j < table.shape[1] else -1 for j in range(npages)]
        good = np.repeat([0 <= i < P for i in ids], PAGE)[:n] if npages else np.zeros(0, bool)
        for h in range(hkv):
            if npages:
                K = np.concatenate([val(kcache[i if 0 <= i < P else 0, h]) for i in ids])[:n]
                V = np.concatenate([val(vcache[i if 0 <= i < P else 0, h]).T for i in ids])[:n]
            for t in range(lo, hi):
                see = n - (hi - lo) + (t - lo) + 1
                for x in range(h * g, (h + 1) * g):
                    keep = np.nonzero(good[:max(see, 0)])[0]
                    if len(keep) == 0:
                        out[t, x] = spread[t, x] = 0.0
                        continue
                    s = (K[keep] @ qf[t, x]) * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    f = 1.0 if gate is None else 1.0 / (1.0 + np.exp(-np.float64(gate[t, x])))
                    out[t, x] = (p @ V[keep]) * f
                    spread[t, x] = (p @ np.abs(V[keep])) * np.abs(f)
    return out, spread
