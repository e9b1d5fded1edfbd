"""CPU oracle of the 4-bit KV cache -- TEST INFRASTRUCTURE ONLY.

Only ``tests/`` may import it.  Float64 numpy from the format's definition: blocks of 32 dims share a scale
2^(byte - 127), values are +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} of it; the scale is the smallest power of two of which no
magnitude of the block is more than 7, from 2^-119 to 2^125; rounding to the nearest, ties to the even index; a block that
holds an infinity or a NaN has the byte 255 and stands for NaN.
"""

from __future__ import annotations

import numpy as np

from oracle.added import attend

PAGE, BLOCK = 16, 32
LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(dim):
    return -(-dim // BLOCK)


def page_bytes(dim):
    return 512 * blocks(dim) + 128


def quantize(x):
    """x (..., D) -> codes (..., 32 N) and scale bytes (..., N)."""
    x = np.asarray(x, dtype=np.float64)
    n = blocks(x.shape[-1])
    y = np.zeros((*x.shape[:-1], 32 * n))
    y[..., : x.shape[-1]] = x
    y = y.reshape(*x.shape[:-1], n, 32)
    code, byte = np.zeros(y.shape, dtype=np.uint8), np.zeros(y.shape[:-1], dtype=np.uint8)
    for at in np.ndindex(*y.shape[:-1]):
        row = y[at]
        if not np.isfinite(row).all():
            byte[at] = 255
            continue
        e, top = -119, np.abs(row).max()
        if top > 0:
            e = max(-119, int(np.floor(np.log2(top))) - 4)
            while top > 7 * 2.0**e and e < 125:
                e += 1
        byte[at] = e + 127
        far = np.abs(np.abs(row)[:, None] / 2.0**e - LEVELS)
        near = far == far.min(axis=1, keepdims=True)
        for i in range(32):
            c = [j for j in range(8) if near[i, j]]
            c = c[0] if len(c) == 1 else next(j for j in c if j % 2 == 0)
            code[at][i] = c + (8 if np.signbit(row[i]) else 0)
    return code.reshape(*x.shape[:-1], 32 * n), byte


def dequantize(code, byte, dim):
    s = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    v = np.where(code >= 8, -1.0, 1.0) * LEVELS[code & 7]
    return (v * np.repeat(s, BLOCK, axis=-1))[..., :dim]


def put(page, row, k, v, dim):
    """Codes and scales of one token into a page (bytes)."""
    n = blocks(dim)
    P = 256 * n
    for (code, byte), is_k in ((quantize(k), True), (quantize(v), False)):
        for d in range(32 * n):
            at = 256 * (d // 32) + 16 * row + d % 32 // 2 if is_k else P + row // 4 * 64 * n + 16 * (d // 8) + 4 * (row % 4) + d % 8 // 2
            shift = 4 * (d % 2)
            page[at] = (int(page[at]) & ~(15 << shift)) | (int(code[d]) << shift)
        for b in range(n):
            page[2 * P + 4 * row + b if is_k else 2 * P + 64 + 16 * (row // 4) + 4 * b + row % 4] = byte[b]


def rows(pool, dim):
    """K and V (num_blocks, n_kv_heads, 16, dim) float64 of a pool (num_blocks, n_kv_heads, page_bytes)."""
    pool = np.asarray(pool)
    n = blocks(dim)
    P = 256 * n
    d, r, b = np.arange(32 * n), np.arange(PAGE)[:, None], np.arange(n)
    k = pool[..., 256 * (d // 32) + 16 * r + d % 32 // 2] >> (4 * (d % 2)) & 15
    v = pool[..., P + r // 4 * 64 * n + 16 * (d // 8) + 4 * (r % 4) + d % 8 // 2] >> (4 * (d % 2)) & 15
    return (dequantize(k, pool[..., 2 * P + 4 * r + b], dim),
            dequantize(v, pool[..., 2 * P + 64 + 16 * (r // 4) + 4 * b + r % 4], dim))


def write(pool, k, v, positions, tables, cu_seqlens, dim):
    """pool with the tokens k, v (T, n_kv_heads, dim) written; placement as oracle.attention.cache_write."""
    pool = np.array(pool)
    cu = range(len(tables) + 1) if cu_seqlens is None else [int(x) for x in cu_seqlens]
    for b in range(len(tables)):
        for t in range(cu[b], cu[b + 1]):
            blk = block_of(pool.shape[0], tables[b], int(positions[cu[b]]), t - cu[b])
            if blk < 0:
                break
            row = (int(positions[cu[b]]) + t - cu[b]) % PAGE
            for h in range(pool.shape[1]):
                put(pool[blk, h], row, k[t, h], v[t, h], dim)
    return pool


def block_of(num_blocks, table, p0, i):
    """Block of position p0 + i, -1 where the walk from p0's column ends before it."""
    if p0 < 0:
        return -1
    blk = -1
    for c in range(p0 // PAGE, (p0 + i) // PAGE + 1):
        blk = int(table[c]) if c < len(table) else -1
        if not 0 <= blk < num_blocks:
            return -1
    return blk


def read(pool, positions, tables, cu_seqlens, dim):
    """(k, v) (T, n_kv_heads, dim) float64; zeros where the walk ends."""
    K, V = rows(pool, dim)
    T = len(positions)
    k, v = np.zeros((T, pool.shape[1], dim)), np.zeros((T, pool.shape[1], dim))
    cu = range(len(tables) + 1) if cu_seqlens is None else [int(x) for x in cu_seqlens]
    for b in range(len(tables)):
        for t in range(cu[b], cu[b + 1]):
            p = int(positions[cu[b]]) + t - cu[b]
            blk = block_of(pool.shape[0], tables[b], int(positions[cu[b]]), t - cu[b])
            if blk >= 0:
                k[t], v[t] = K[blk, :, p % PAGE], V[blk, :, p % PAGE]
    return k, v


def prologue(x, weight, eps, cos, sin, positions, interleaved):
    """Norm (weight None: none) and rotation of x (T, heads, D) by the operator's own rounding steps: the norm in float64,
    rounded to float32; the rotation in float32, each product and sum rounded."""
    x = np.asarray(x, dtype=np.float64)
    if weight is not None:
        x = x * (1.0 / np.sqrt((x * x).sum(-1, keepdims=True) / x.shape[-1] + eps)) * np.asarray(weight, dtype=np.float64)
    x = x.astype(np.float32)
    half = cos.shape[1]
    for t, p in enumerate(positions):
        ok = 0 <= p < cos.shape[0]
        c = cos[p].astype(np.float32) if ok else np.full(half, np.nan, np.float32)
        s = sin[p].astype(np.float32) if ok else np.full(half, np.nan, np.float32)
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            u, w = x[t, :, a].copy(), x[t, :, b].copy()
            x[t, :, a], x[t, :, b] = u * c[i] - w * s[i], w * c[i] + u * s[i]
    return x


def gather(X, table, kv_len):
    """(n_kv_heads, kv_len, D) of one sequence from ``rows``; columns past the table and ids outside the pool: zeros."""
    n = -(-kv_len // PAGE)
    out = np.zeros((n, *X.shape[1:]))
    for c, blk in enumerate(list(table)[:n]):
        if 0 <= int(blk) < X.shape[0]:
            out[c] = X[int(blk)]
    return out.transpose(1, 0, 2, 3).reshape(X.shape[1], n * PAGE, X.shape[3])[:, :kv_len]


def decode(q, pool, tables, kv_lens):
    """(H, B, D); an empty context gives zeros."""
    H, B, D = q.shape
    K, V = rows(pool, D)
    rep, out = H // pool.shape[1], np.zeros((H, B, D))
    for b in range(B):
        L = int(kv_lens[b])
        if L <= 0:
            continue
        k, v = gather(K, tables[b], L), gather(V, tables[b], L)
        for h in range(H):
            out[h, b] = attend(q[h, b : b + 1], k[h // rep], v[h // rep], np.ones((1, L), dtype=bool))[0]
    return out


def prefill(q, pool, cu_seqlens, tables, kv_lens, positions, tokens=None):
    """(H, T, D); ``tokens``: those to compute (others NaN); a token that sees no key is NaN."""
    H, T, D = q.shape
    K, V = rows(pool, D)
    rep, out = H // pool.shape[1], np.full((H, T, D), np.nan)
    cu = [int(x) for x in cu_seqlens]
    for b in range(len(cu) - 1):
        t = np.array([i for i in range(cu[b], cu[b + 1]) if tokens is None or i in tokens], dtype=np.int64)
        if t.size == 0:
            continue
        L = max(0, int(kv_lens[b]))
        k, v = gather(K, tables[b], L), gather(V, tables[b], L)
        seen = np.arange(L)[None, :] <= np.asarray(positions)[t][:, None]
        for h in range(H):
            out[h, t] = attend(q[h, t], k[h // rep], v[h // rep], seen)
    return out
