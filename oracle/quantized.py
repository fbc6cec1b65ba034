"""Plain 64-bit forms of the 8-bit KV pool's operators and of the block tables (tests only).

Codes are given as the numbers they are (float64 [pages, 16, kv_heads, head_dim]); scales
[pages, kv_heads, 2] float64 (K, V)."""
from __future__ import annotations

import numpy as np

PAGE = 16


def append_scales(scale, x, slots, qmax, tiny=2.0 ** -100):
    """(new scales, written) of one tensor: `scale` [pages, kv_heads], rows x [tokens, kv_heads,
    head_dim] at `slots`; `written` maps a page to {row: token}.  Of two tokens with one slot the
    later is kept; slots outside the pool are left out."""
    new = scale.copy()
    written = {}
    for t, s in enumerate(slots):
        if 0 <= s < scale.shape[0] * PAGE:
            written.setdefault(int(s) // PAGE, {})[int(s) % PAGE] = t
    for page, rows in written.items():
        vals = np.abs(x[list(rows.values())])
        top = np.where(np.isfinite(vals), vals, 0.0).max(axis=(0, 2)) / qmax
        top[top < tiny] = 0.0
        new[page] = np.maximum(0.0 if 0 in rows else scale[page], top)
    return new, written


def attention(q, k, v, scales, tables, seqs, positions, sm_scale):
    """(out, weight) per token and head: softmax(q.k * sm_scale).v, and the same sum over |v|,
    which bounds what an error of the probabilities can do.  Rows without keys are zeros."""
    T, H, D = q.shape
    N, _, KVH, _ = k.shape
    B, W = tables.shape
    out, weight = np.zeros((T, H, D)), np.zeros((T, H, D))
    for t in range(T):
        s, p = int(seqs[t]), int(positions[t])
        if not 0 <= s < B or p < 0:
            continue
        n = min(p + 1, W * PAGE)
        pages = tables[s, :(n + PAGE - 1) // PAGE].astype(np.int64)
        ok = (pages >= 0) & (pages < N)
        safe = np.where(ok, pages, 0)

        def rows(pool, which):
            x = pool[safe] * scales[safe][:, None, :, which, None]
            x[~ok] = 0.0
            return x.reshape(-1, KVH, D)[:n]

        kk, vv = rows(k, 0), rows(v, 1)
        for h in range(H):
            g = h // (H // KVH)
            x = kk[:, g] @ q[t, h] * sm_scale
            e = np.exp(x - x.max())
            e /= e.sum()
            out[t, h] = e @ vv[:, g]
            weight[t, h] = e @ np.abs(vv[:, g])
    return out, weight


def block_tables(cached, new, tables, free, head, tokens):
    """What build_block_tables returns, row by row."""
    tables = tables.copy()
    seqs = np.full(tokens, -1, np.int32)
    pos, slots = np.full(tokens, -1, np.int64), np.full(tokens, -1, np.int64)
    last = np.full(len(cached), -1, np.int64)
    lens = np.zeros(len(cached), np.int32)
    head = max(int(head), 0)
    t = 0
    W = tables.shape[1]
    for r in range(len(cached)):
        c, n = max(int(cached[r]), 0), max(int(new[r]), 0)
        lens[r] = c + n
        for j in range((c + PAGE - 1) // PAGE, min((c + n + PAGE - 1) // PAGE, W)):
            tables[r, j] = free[head] if head < len(free) else -1
            head += 1
        for p in range(c, c + n):
            if t < tokens:
                seqs[t], pos[t] = r, p
                if p // PAGE < W and tables[r, p // PAGE] >= 0:
                    slots[t] = int(tables[r, p // PAGE]) * PAGE + p % PAGE
                last[r] = t
                t += 1
    return dict(tables=tables, seqs=seqs, positions=pos, slots=slots, last=last, lens=lens,
                free_head=np.array([min(head, max(len(free), 0))], np.int32))
