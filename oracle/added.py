"""CPU oracle of the operators without a counterpart in the reference -- TEST INFRASTRUCTURE ONLY.

Only ``tests/`` may import it; the shipped operators run the HIP kernels in
``libfemto_attn.so``.  Float64 numpy, from the operators' definitions:

* window attention: a query at position p of a sequence of L keys sees key j
  iff j < L, j <= p and (j > p - window or j < sinks);
* shared-prefix decode: key j of a sequence is in block ``prefix_pages[j //
  16]`` for j < 16 * len(prefix_pages), else in its own table's column j // 16;
* rotation: dims (a, b) of a pair become (a c - b s, b c + a s).

A block id outside the pool reads as zeros, and a key that is not seen has no
part in the result whatever it holds.
"""

from __future__ import annotations

import numpy as np

PAGE = 16


def gather(pool, table, kv_len):
    """(n_kv_heads, kv_len, D) float64 of one sequence; columns past the table and ids outside the pool: zeros."""
    n = -(-kv_len // PAGE)
    out = np.zeros((n, *pool.shape[1:]), dtype=np.float64)
    for c, blk in enumerate(list(table)[:n]):
        if 0 <= int(blk) < pool.shape[0]:
            out[c] = pool[int(blk)]
    return out.transpose(1, 0, 2, 3).reshape(pool.shape[1], n * PAGE, pool.shape[3])[:, :kv_len]


def attend(q, k, v, seen):
    """One head: q (T, D), k and v (L, D), seen (T, L) -> (T, D); a row that sees nothing is NaN."""
    out = np.full(q.shape, np.nan)
    for t in range(q.shape[0]):
        j = np.nonzero(seen[t])[0]
        if j.size == 0:
            continue
        s = k[j] @ q[t] / np.sqrt(q.shape[1])
        w = np.exp(s - s.max())
        out[t] = w @ v[j] / w.sum()
    return out


def window_seen(pos, kv_len, window, sinks):
    """(T, kv_len) truth values of the window rule for queries at ``pos`` (T,)."""
    j = np.arange(kv_len)[None, :]
    p = np.asarray(pos, dtype=np.int64)[:, None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def window_decode(q, k_pool, v_pool, tables, kv_lens, window, sinks):
    """(H, B, D); an empty context gives zeros."""
    H, B, D = q.shape
    rep = H // k_pool.shape[1]
    out = np.zeros((H, B, D))
    for b in range(B):
        L = int(kv_lens[b])
        if L <= 0:
            continue
        k, v = gather(k_pool, tables[b], L), gather(v_pool, tables[b], L)
        seen = window_seen([L - 1], L, window, sinks)
        for h in range(H):
            out[h, b] = attend(q[h, b : b + 1], k[h // rep], v[h // rep], seen)[0]
    return out


def window_prefill(q, k_pool, v_pool, cu_seqlens, tables, kv_lens, positions, window, sinks, rows=None):
    """(H, T, D); ``rows``: the tokens to compute (others NaN)."""
    H, T, D = q.shape
    rep = H // k_pool.shape[1]
    out = np.full((H, T, D), np.nan)
    cu = [int(x) for x in cu_seqlens]
    for b in range(len(cu) - 1):
        t = np.array([i for i in range(cu[b], cu[b + 1]) if rows is None or i in rows], dtype=np.int64)
        if t.size == 0:
            continue
        L = max(0, int(kv_lens[b]))
        k, v = gather(k_pool, tables[b], L), gather(v_pool, tables[b], L)
        seen = window_seen(np.asarray(positions)[t], L, window, sinks)
        for h in range(H):
            out[h, t] = attend(q[h, t], k[h // rep], v[h // rep], seen)
    return out


def shared_prefix_decode(q, k_pool, v_pool, prefix_pages, tables, kv_lens):
    """(H, B, D); an empty context gives zeros."""
    own = [list(prefix_pages) + list(t)[len(prefix_pages) :] for t in tables]
    return window_decode(q, k_pool, v_pool, own, kv_lens, 1 << 40, 0)


def rotate(x, cos, sin, positions, interleaved):
    """(T, heads, D) rotated at each token's position; cos / sin (rows, R / 2); a position outside them: NaN."""
    x = np.array(x, dtype=np.float64)
    half = cos.shape[1]
    for t, p in enumerate(positions):
        ok = 0 <= p < cos.shape[0]
        c = cos[p].astype(np.float64) if ok else np.full(half, np.nan)
        s = sin[p].astype(np.float64) if ok else np.full(half, np.nan)
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            u, w = x[t, :, a].copy(), x[t, :, b].copy()
            x[t, :, a], x[t, :, b] = u * c[i] - w * s[i], w * c[i] + u * s[i]
    return x
