"""CPU restatement of the paged KV cache operators in 64 bits (TEST INFRASTRUCTURE).

Only tests/ import this; the product path is vllm_gr_ehaleva_b200/attention/paged.py.
Written from the definitions: loops over requests and tokens, no tiling."""
from __future__ import annotations

import numpy as np


def extend_block_tables(table, cached, fresh, free, block_size, num_tokens):
    """Returns (table, cu, seq_lens, slots, positions, used, no_block)."""
    table = table.copy()
    slots = np.full(num_tokens, -1, np.int64)
    positions = np.zeros(num_tokens, np.int64)
    cu, used, no_block, t = [0], 0, False, 0
    for r in range(len(cached)):
        c, f = int(cached[r]), int(fresh[r])
        have, need = -(-c // block_size), -(-(c + f) // block_size)
        for j in range(have, need):
            if used < len(free) and j < table.shape[1]:
                table[r, j] = free[used]
            else:
                no_block = True
            used += 1
        for i in range(f):
            p = c + i
            j = p // block_size
            ok = j < table.shape[1]
            if ok and j >= have:
                ok = used - (need - have) + (j - have) < len(free)
            if ok and table[r, j] >= 0:
                slots[t] = int(table[r, j]) * block_size + p % block_size
            else:
                no_block = True
            positions[t] = p
            t += 1
        cu.append(cu[-1] + f)
    return (table, np.array(cu, np.int32), (np.asarray(cached) + np.asarray(fresh)).astype(np.int32), slots, positions,
            used, no_block)


def seen(n, length, causal, tail=0, steps=0):
    """bool [n, length]: which keys each of a request's n query tokens sees."""
    p = (length - n + np.arange(n))[:, None]
    k = np.arange(length)[None]
    ok = (k <= p) if causal else np.ones((n, length), bool)
    if steps > 0:
        first = length - n + tail
        own = first + (p - first) // steps * steps
        ok = ok & np.where(p >= first, (k < first) | (k >= own), True)
    return ok


def attention(q, k_cache, v_cache, table, cu, seq_lens, *, causal=True, scale=None, tail=None, steps=None):
    """float64 arrays in; returns (out, lse, absv): absv = sum_k w_k |v_k| per output, the
    size of the sum that rounding errors of the weights act on.  Rows of no request are NaN."""
    T, H, D = q.shape
    HK = k_cache.shape[2]
    G = H // HK
    bs = k_cache.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = np.full((T, H, D), np.nan)
    lse = np.full((T, H), np.nan)
    absv = np.full((T, H, D), np.nan)
    for r in range(len(seq_lens)):
        a, b, L = int(cu[r]), int(cu[r + 1]), int(seq_lens[r])
        n = b - a
        if n == 0:
            continue
        pos = np.arange(L)
        kr = k_cache[table[r, pos // bs], pos % bs] if L else np.zeros((0, HK, D))
        vr = v_cache[table[r, pos // bs], pos % bs] if L else np.zeros((0, HK, D))
        ok = seen(n, L, causal, 0 if tail is None else int(tail[r]), 0 if steps is None else int(steps[r]))
        for h in range(H):
            s = np.where(ok, scale * (q[a:b, h] @ kr[:, h // G].T), -np.inf)
            m = s.max(1, initial=-np.inf)
            w = np.exp(s - np.where(np.isinf(m), 0, m)[:, None])
            l = w.sum(1)
            with np.errstate(divide="ignore", invalid="ignore"):
                lse[a:b, h] = m + np.log(l)
                w = np.where(l[:, None] > 0, w / l[:, None], 0)
            out[a:b, h] = w @ vr[:, h // G]
            absv[a:b, h] = w @ np.abs(vr[:, h // G])
    return out, lse, absv
