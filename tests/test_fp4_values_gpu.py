"""Attention over the 4-bit cache where its values, queries or hidden rows are not the usual ones, against the 64-bit oracle.

* Queries whose blocks of 32 dims hold one large channel: what the other dims hold has to arrive all the same.  The values
  here need at most 18 bits below a block's largest magnitude's exponent, which a split of q into four terms holds exactly in
  decode; a prefill query is split after it took the softmax scale, and is off by at most 2^-18 of the largest magnitude of
  its block.
* Sharp scores, where one key's weight is near 1 and a score's error moves outputs by as much: bounds per row, from the row's
  own weights, and far below the spread of its values.
* f16 values that round to 65536 in the cache; rows that no sequence holds, with full codes under large scales and NaN.
"""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from fp4_helpers import Batch, pool_of
from helpers import assert_close, half_ulp, np64

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
    """want (H, T, D), sum_j w_j |v_j| and sum_j w_j |v_j - want| (the same shape); and of the row's largest key, (H, T) each,
    the sum over dims of |k| and the root of that of k^2, times the largest |q| of the dim's block, over sqrt(D)."""
    H, T, D = w.q.shape
    K, V = of.rows(w.pool, D)
    rep, q = H // w.pool.shape[1], np64(w.q)
    top = np.abs(q).reshape(H, T, -1, min(32, D)).max(-1).repeat(min(32, D), -1)
    want, size, spread = np.zeros((3, H, T, D))
    reach, root = np.zeros((2, H, T))
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
            root[h, t] = np.sqrt((k[h // rep] ** 2 @ top[h, t] ** 2).max() / D)
    return want, size, spread, reach, root


LENS = [1, 17, 64, 100, 333, 1000]
CHUNKS = [(0, 130), (200, 70), (90, 1), (900, 40), (40, 1)]


def large_channels(chunks, heads, dim, dtype, top, seed, decode):
    """q: N(0, 1) past 1/8, and ``top`` in dims 5, 37, ..; K zero there, else of size 4; V of size 1."""
    w = Batch(chunks, *heads, dim, dtype, seed, decode=decode)
    rng = np.random.default_rng(seed)
    K, V = rng.standard_normal((2, len(w.pool), heads[1], 16, dim))
    K *= 4
    K[..., 5::32] = 0
    refill(w, K, V)
    q = w.q.float()
    q = torch.where(q < 0, q.clamp(max=-0.125), q.clamp(min=0.125))
    q[..., 5::32] = top * torch.sign(q[..., 5::32])
    w.q = q.to(dtype)
    return w


@pytest.mark.parametrize("dtype,top", [(BF16, 512.0), (F16, 64.0)])
@pytest.mark.parametrize("dim", [128, 64, 80])
@pytest.mark.parametrize("heads", [(8, 2), (4, 4)])
def test_decode_of_queries_with_large_channels(ops, gpu, heads, dim, dtype, top):
    w = large_channels([(n - 1, 1) for n in LENS], heads, dim, dtype, top, dim + sum(heads), True)
    assert_close(gemv(ops, gpu, w), of.decode(np64(w.q), w.pool, w.tables, w.kv_lens), dtype, f"channels of {top}")


@pytest.mark.parametrize("dtype,top", [(BF16, 512.0), (F16, 64.0)])
@pytest.mark.parametrize("dim", [128, 64, 80])
@pytest.mark.parametrize("heads", [(8, 2), (4, 4), (4, 2)])
def test_prefill_of_queries_with_large_channels(ops, gpu, heads, dim, dtype, top):
    """The split's error here: at most 2^-18 * 512 of a dim of q, so some 2^-9 / sqrt(3) * 4 of a score, in f16 an eighth."""
    w = large_channels(CHUNKS, heads, dim, dtype, top, dim + sum(heads), False)
    assert_close(gemm(ops, gpu, w), of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos), dtype, f"channels of {top}")


@pytest.mark.parametrize("top", [64.0, 1000.0])
def test_a_query_of_large_channels_beside_others(ops, gpu, top):
    """Few of a tile's queries have them, in one block each: no other row's result depends on them."""
    w = Batch([(300, 200), (50, 1), (0, 64)], 8, 2, 128, BF16, 3)
    pool, tables, lens, cu, pos, q = w.on(gpu)
    plain = ops.paged_attention_gemm_fp4(q, pool, cu, 200, tables, lens, pos)
    rows = [3, 70, 199, 200, 230]
    w.q[:, rows, 40] = top
    got = gemm(ops, gpu, w)
    want = of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos)
    others = [t for t in range(q.size(1)) if t not in rows]
    assert_close(got[:, others], want[:, others], BF16, "others")
    assert_close(got[:, others], np64(plain[:, others]), BF16, "others as before")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("decode,scale", [(d, s) for d in (True, False) for s in (1.0, 4.0, 12.0, 30.0, 200.0) if d or s < 200])
def test_sharp_scores_row_by_row(ops, gpu, decode, scale, dtype):
    """K of size ``scale``.  A weight is off by its rounding (eps / 2 of P, and as much of the sum) and by e^(2 ds) - 1, ds
    a score's error: q's split (decode: none, q's values are held exactly; prefill, three terms: at most 2^-14 of the
    blocks' largest magnitudes in each dim, six times its random sum) and 32-bit sums of some 130 terms (each at most 2^-24
    of the sum of magnitudes, ten times their random sum)."""
    chunks = [(n - 1, 1) for n in LENS] if decode else CHUNKS
    w = Batch(chunks, 8, 2, 128, dtype, int(10 * scale), decode=decode, scale=scale)
    hide(w, 255, 255)
    q = w.q.float()
    w.q = torch.where(q < 0, q.clamp(max=-2.0**-5), q.clamp(min=2.0**-5)).to(dtype)
    got = np64(gemv(ops, gpu, w) if decode else gemm(ops, gpu, w))
    want, size, spread, reach, root = weights(w, decode)
    ds = ((0 if decode else 6 * 2.0**-14 / np.sqrt(3)) * root + 2.0**-24 * 10 * np.sqrt(130) * reach)[..., None]
    step = torch.finfo(dtype).eps / 2
    bound = spread * np.expm1(2 * ds) + size * 2 * step + half_ulp(np.abs(want), dtype) + 2.0**-20
    K, V = of.rows(w.pool, 128)
    assert np.median(bound) < 0.02 * np.nanstd(V) and bound.max() < np.nanstd(V), (np.median(bound), bound.max())
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


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
    want, size, _, _, _ = weights(w, decode)
    assert np.isfinite(got).all() and np.abs(want).max() > 10000
    # weights off by 2^-11 each, rounded, their sum's and the query's as much again
    assert (np.abs(got - want) <= size * 2.0**-9 + half_ulp(np.abs(want), F16) + 2.0**-11).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [128, 48])
@pytest.mark.parametrize("byte,code", [(254, 0x77), (254, 0xFF), (255, 0x00), (255, 0xFF), (1, 0x99)])
def test_rows_that_no_sequence_holds(ops, gpu, byte, code, dim, dtype):
    """Full codes under the largest scale, NaN with any codes: nothing of them arrives."""
    w = Batch([(n - 1, 1) for n in LENS + [15, 16, 31]], 4, 2, dim, dtype, 7, decode=True)
    hide(w, byte, code)
    assert_close(gemv(ops, gpu, w), of.decode(np64(w.q), w.pool, w.tables, w.kv_lens), dtype, "decode")
    w = Batch(CHUNKS + [(0, 15), (0, 63), (17, 48)], 4, 2, dim, dtype, 8)
    hide(w, byte, code)
    assert_close(gemm(ops, gpu, w), of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos), dtype, "prefill")


@pytest.mark.parametrize("dtype,top", [(BF16, 512.0), (F16, 64.0)])
@pytest.mark.parametrize("dim", [128, 112, 48, 16])
def test_large_channels_of_a_split_tile_and_beside_rows(ops, gpu, dim, dtype, top):
    """A long context's tile in pieces, which split q each for themselves, and decode rows in the same launch."""
    w = large_channels([(6000, 64), (100, 20)] + [(n, 1) for n in (0, 40, 700)], (8, 2), dim, dtype, top, dim, False)
    want = of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos)
    first = gemm(ops, gpu, w)
    assert_close(first, want, dtype, f"channels of {top}, dim {dim}")
    assert torch.equal(gemm(ops, gpu, w), first)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_zeros_infinities_and_nan_in_queries(ops, gpu, dtype):
    """Rows of zeros (plain averages), rows with most dims zero, and an infinity or a NaN in one row, which stays its own."""
    w = Batch([(100, 70), (0, 33), (64, 1)], 4, 2, 128, dtype, 11)
    w.q[:, 3] = 0
    w.q[:, 7, 1:] = 0
    w.q[:, 40, 33:] = 0
    w.q[1, 10, 70], w.q[2, 75, 0], w.q[3, 103, 127] = float("inf"), float("nan"), float("-inf")
    got = gemm(ops, gpu, w)
    want = of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos)
    for h, t in ((1, 10), (2, 75), (3, 103)):
        want[h, t] = np.nan  # (infinite scores of both signs, or of one and NaN for those of zero: the row is NaN)
    assert_close(got, want, dtype, "zeros and infinities")
