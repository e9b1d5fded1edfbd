"""Attention over the 4-bit cache where its values, queries or hidden rows are not the usual ones, against the 64-bit oracle.

f16 values that round to 65536 in the cache.
"""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from fp4_helpers import Batch, pool_of
from helpers import half_ulp, np64

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def hide(w, byte, code):
    """Every row that no sequence holds: full codes (``code`` twice a byte) under scales of ``byte``."""
    n = of.blocks(w.dim)
    P = 256 * n
    held = np.zeros(w.pool.shape[:1] + (16,), dtype=bool)
    for table, length in zip(w.tables, w.kv_lens):
        for c in range(-(-int(length) // 16)):
            held[table[c], : min(16, int(length) - 16 * c)] = True
    for r in range(16):
        blk = np.nonzero(~held[:, r])[0][:, None]
        i, b = np.arange(16), np.arange(4)
        for x in range(n):
            w.pool[blk, :, 256 * x + 16 * r + i] = code
        c = np.arange(4 * n)
        for x in range(4):
            w.pool[blk, :, P + 64 * n * (r // 4) + 16 * c + 4 * (r % 4) + x] = code
        w.pool[blk, :, 2 * P + 4 * r + b] = byte
        w.pool[blk, :, 2 * P + 64 + 16 * (r // 4) + 4 * b + r % 4] = byte


def refill(w, K, V):
    w.pool = pool_of(K, V)
    hide(w, 255, 255)


def gemv(ops, gpu, w):
    pool, tables, lens, _, _, q = w.on(gpu)
    return ops.paged_attention_gemv_fp4(q, pool, tables, lens, int(w.kv_lens.max()))


def gemm(ops, gpu, w):
    pool, tables, lens, cu, pos, q = w.on(gpu)
    return ops.paged_attention_gemm_fp4(q, pool, cu, max(n for _, n in w.chunks), tables, lens, pos)


def rows_of(w, decode):
    """(row of q, keys it sees, its sequence)"""
    for b, (p, n) in enumerate(w.chunks):
        for i in range(1 if decode else n):
            yield (b if decode else int(w.cu[b]) + i), (int(w.kv_lens[b]) if decode else p + i + 1), b


def weights(w, decode):
    """want (H, T, D), sum_j w_j |v_j| and sum_j w_j |v_j - want| (the same shape), and |q| . |k| / sqrt(D) of the row's
    largest key with q's magnitudes those of its blocks' largest (H, T)."""
    H, T, D = w.q.shape
    K, V = of.rows(w.pool, D)
    rep, q = H // w.pool.shape[1], np64(w.q)
    top = np.abs(q).reshape(H, T, -1, min(32, D)).max(-1).repeat(min(32, D), -1)
    want, size, spread = np.zeros((3, H, T, D))
    reach = np.zeros((H, T))
    for t, length, b in rows_of(w, decode):
        k, v = of.gather(K, w.tables[b], length), of.gather(V, w.tables[b], length)
        for h in range(H):
            s = k[h // rep] @ q[h, t] / np.sqrt(D)
            p = np.exp(s - s.max())
            p /= p.sum()
            x = v[h // rep]
            want[h, t] = p @ x
            size[h, t], spread[h, t] = p @ np.abs(x), p @ np.abs(x - want[h, t])
            reach[h, t] = (np.abs(k[h // rep]) @ top[h, t]).max() / np.sqrt(D)
    return want, size, spread, reach


LENS = [1, 17, 64, 100, 333, 1000]
CHUNKS = [(0, 130), (200, 70), (90, 1), (900, 40), (40, 1)]


@pytest.mark.parametrize("decode", [True, False])
def test_f16_values_that_round_to_65536(ops, gpu, decode):
    """Finite f16 values past 57344 are held as 65536, which f16 has no number for: attention's averages of it are finite."""
    chunks = [(n - 1, 1) for n in (9, 40, 300)] if decode else [(8, 60), (100, 130), (20, 1)]
    w = Batch(chunks, 4, 2, 64, F16, 5, decode=decode, scale=0.25)
    rng = np.random.default_rng(6)
    K, V = rng.standard_normal((2, len(w.pool), 2, 16, 64))
    big = rng.random(V.shape[:3]) < 0.2
    V[big, 7] = 60000.0 * rng.choice([-1.0, 1.0], size=big.sum())
    V[big, 40] = 65504.0
    w.pool = pool_of(0.25 * K, V)
    hide(w, 254, 0x77)
    assert (np.abs(of.rows(w.pool, 64)[1]) == 65536.0).any()
    got = np64(gemv(ops, gpu, w) if decode else gemm(ops, gpu, w))
    want, size, _, _ = weights(w, decode)
    assert np.isfinite(got).all() and np.abs(want).max() > 10000
    # weights off by 2^-11 each, rounded, their sum's and the query's as much again
    assert (np.abs(got - want) <= size * 2.0**-9 + half_ulp(np.abs(want), F16) + 2.0**-11).all()
