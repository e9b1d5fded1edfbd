"""Decode over the 4-bit cache against the 64-bit oracle.

Bounds: helpers.assert_close's, as of the 16-bit operators.  The kernel rounds P to q's type (at most eps / 2 relative
per weight, as there) and the output once; q enters to 2^-14 of the largest magnitude of its 32 dims, so a score is off by
at most 2^-14 max|q| sum|k| / sqrt(D), below 2^-14 * 4 * 128 / 11.3 = 2.8e-3 at worst and its random sum far below that,
where bf16's half step of P alone is 3.9e-3.
"""

import threading

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from fp4_helpers import Batch, poison
from helpers import assert_close, np64

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
LENS = [1, 2, 15, 16, 17, 31, 32, 33, 48, 64, 65, 129, 300, 1000]


def run(ops, gpu, w, max_kv_len=None):
    pool, tables, lens, _, _, q = w.on(gpu)
    return ops.paged_attention_gemv_fp4(q, pool, tables, lens, int(w.kv_lens.max()) if max_kv_len is None else max_kv_len)


def check(ops, gpu, w, what, **kw):
    out = run(ops, gpu, w, **kw)
    want = of.decode(np64(w.q), w.pool, w.tables, w.kv_lens)
    assert_close(out, want, w.dtype, what)
    return out


@pytest.mark.usefixtures("decode_path")
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [(8, 8), (16, 8), (32, 8), (64, 8), (6, 2), (20, 1), (34, 2), (1, 1)])
def test_heads(ops, gpu, heads, dtype):
    w = Batch([(n - 1, 1) for n in LENS], *heads, 128, dtype, sum(heads), decode=True)
    check(ops, gpu, w, f"heads {heads} {dtype}")


@pytest.mark.usefixtures("decode_path")
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112])
def test_dims(ops, gpu, dim, dtype):
    w = Batch([(n - 1, 1) for n in LENS], 8, 2, dim, dtype, dim, decode=True)
    check(ops, gpu, w, f"dim {dim} {dtype}")


@pytest.mark.usefixtures("decode_path")
def test_long_and_many(ops, gpu):
    """More sequences than a wave has lanes, very uneven, a context past 16k keys, empty slots with tables of -1."""
    rng = np.random.default_rng(5)
    lens = [17000, 5000] + [int(x) for x in rng.integers(1, 900, size=70)]
    chunks = [(n - 1, 1) for n in lens]
    for b in (3, 40, 71):
        chunks[b] = (0, 0)
    w = Batch(chunks, 4, 2, 128, BF16, 6, decode=True)
    out = check(ops, gpu, w, "long and many")
    assert (out[:, [3, 40, 71]] == 0).all()


@pytest.mark.parametrize("max_kv_len", [0, 1, 100, 1000, 5000, 2**31 - 1])
def test_max_kv_len_only_plans(ops, gpu, max_kv_len):
    w = Batch([(n - 1, 1) for n in (1000, 3, 500)], 8, 2, 128, BF16, 7, decode=True)
    check(ops, gpu, w, f"max_kv_len {max_kv_len}", max_kv_len=max_kv_len)


@pytest.mark.parametrize("lens", [[3000], [16384, 20, 17], [500, 1, 0, 2047], [33000] + [40] * 15, [17000] + [300] * 31])
def test_rows_in_parts_and_split_calls(ops, gpu, lens):
    """Few long rows are cut into parts (short ones among them into fewer), many of the longest contexts run split."""
    w = Batch([(max(n - 1, 0), min(n, 1)) for n in lens], 16, 8, 128, BF16, sum(lens), decode=True)
    a = check(ops, gpu, w, f"lens {lens[:3]}")
    for _ in range(5):  # parts are merged in order, whoever comes last
        assert torch.equal(run(ops, gpu, w), a)


@pytest.mark.usefixtures("decode_path")
def test_blocks_outside_the_pool_and_short_tables(ops, gpu):
    """A block id outside the pool and a column past the table read as zeros, with their weight."""
    w = Batch([(n - 1, 1) for n in (200, 100, 64, 33)], 8, 2, 128, BF16, 8, decode=True)
    w.tables[0, 3], w.tables[0, 7], w.tables[1, 0], w.tables[3, 2] = -1, len(w.pool), 2**31 - 1, -(2**31)
    check(ops, gpu, w, "ids outside")
    w.tables = np.ascontiguousarray(w.tables[:, :9])
    check(ops, gpu, w, "a table of 9 columns")


@pytest.mark.usefixtures("decode_path")
@pytest.mark.parametrize("scale", [2.0**-20, 0.02, 12.0, 200.0])
def test_flat_and_sharp_scores(ops, gpu, scale):
    """All weights alike, and one key that takes all (a score's error grows with it: the bound of assert_close times the
    largest score's share, see the module's text)."""
    w = Batch([(n - 1, 1) for n in (300, 77, 16)], 8, 2, 128, BF16, 9, decode=True, scale=scale)
    out = run(ops, gpu, w)
    want = of.decode(np64(w.q), w.pool, w.tables, w.kv_lens)
    # 2^-14 max|q| sum_d |k_d| / sqrt(D) of a score, e^that - 1 of a weight, twice that of the outputs' range
    K, V = of.rows(w.pool, 128)
    k = np.concatenate([K[t[: -(-n // 16)]].transpose(1, 0, 2, 3).reshape(2, -1, 128)[:, :n] for t, n in zip(w.tables, w.kv_lens)], axis=1)
    off = 2.0**-14 * np.abs(np64(w.q)).max() * np.abs(k).sum(-1).max() / np.sqrt(128)
    top = np.nanmax(np.abs(V))
    bound = top * (2 * np.expm1(2 * off) + 2.0**-7) + 1e-2
    assert np.isfinite(np64(out)).all() and np.abs(np64(out) - want).max() <= bound
    if scale < 1:
        assert_close(out, want, BF16, f"scale {scale}")


@pytest.mark.usefixtures("decode_path")
def test_nan_and_infinities(ops, gpu):
    """A NaN key makes its sequence's heads NaN, a NaN block of V those dims; other sequences and heads are not touched."""
    w = Batch([(n - 1, 1) for n in (100, 100, 100, 37)], 4, 2, 128, BF16, 10, decode=True)
    P = 1024
    w.pool[w.tables[0, 2], 1, 2 * P + 4 * 5 + 2] = 255  # K of key 37, head 1
    w.pool[w.tables[1, 6], 0, 2 * P + 64 + 4 * 1 + 3] = 255  # V of key 99, head 0, dims 32 .. 63
    w.q[3, 2, 5] = float("inf")
    out = check(ops, gpu, w, "NaN")
    nan = torch.isnan(out).cpu()
    assert nan[2:, 0].all() and nan[:2, 1, 32:64].all() and nan[3, 2].all() and nan.sum() == 2 * 128 + 2 * 32 + 128


def test_strided_q_and_q_of_another_type_than_the_writer(ops, gpu):
    w = Batch([(n - 1, 1) for n in LENS], 8, 2, 64, F16, 11, decode=True)
    pool, tables, lens, _, _, q = w.on(gpu)
    wide = torch.zeros(len(LENS), 3, 8, 64, dtype=F16, device=gpu)
    wide[:, 1] = q.transpose(0, 1)
    a = ops.paged_attention_gemv_fp4(wide[:, 1].transpose(0, 1), pool, tables, lens, 1000)
    b = ops.paged_attention_gemv_fp4(q, pool, tables, lens, 1000)
    assert torch.equal(a, b)
    assert_close(a, of.decode(np64(w.q), w.pool, w.tables, w.kv_lens), F16, "strided")


def test_f16_values_near_its_range(ops, gpu):
    """V of 2^-14 and less, and up to 6 * 2^13, in f16."""
    for shift in (-16, 13):
        w = Batch([(39, 1), (15, 1)], 2, 1, 64, F16, 12, decode=True)
        n = of.blocks(64)
        at = slice(512 * n + 64, 512 * n + 128)
        s = w.pool[..., at].astype(int)
        w.pool[..., at] = np.where(s == 255, 255, 127 + shift)
        out = run(ops, gpu, w)
        want = of.decode(np64(w.q), w.pool, w.tables, w.kv_lens)
        # weights off by 2^-11 each (rounded, and their sum's), subnormal outputs by half a step of 2^-24
        assert (np.abs(np64(out) - want) <= 6 * 2.0**shift * 2.0**-9 + 2.0**-25).all()


def test_far_pool_and_wide_batch(ops, gpu):
    """A pool past 4 GiB: blocks beyond 32-bit byte offsets."""
    blocks = (5 << 30) // (8 * 2176)
    w = Batch([(n - 1, 1) for n in (70, 500, 33)], 16, 8, 128, BF16, 13, decode=True)
    pool = torch.empty((blocks, 8, 2176), dtype=torch.uint8, device=gpu)
    shift = blocks - len(w.pool)
    pool[shift:] = torch.tensor(w.pool, device=gpu)
    _, tables, lens, _, _, q = w.on(gpu)
    out = ops.paged_attention_gemv_fp4(q, pool, torch.where(tables >= 0, tables + shift, tables), lens, 500)
    assert_close(out, of.decode(np64(w.q), w.pool, w.tables, w.kv_lens), BF16, "far pool")


def test_graphs_streams_and_threads(ops, gpu):
    """Captured calls replayed between eager ones, two streams at once, two host threads: each result is the eager one's."""
    ws = [Batch([(n - 1, 1) for n in lens], 16, 8, 128, BF16, 20 + i, decode=True) for i, lens in enumerate(([4000], [700, 9, 64], [33] * 40))]
    sets = [w.on(gpu) for w in ws]
    call = lambda s, w: ops.paged_attention_gemv_fp4(s[5], s[0], s[1], s[2], int(w.kv_lens.max()))
    want = [call(s, w).clone() for s, w in zip(sets, ws)]
    graphs, outs = [], []
    for s, w in zip(sets, ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(s, w))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        assert torch.equal(call(sets[1], ws[1]), want[1])
        torch.cuda.synchronize()
        for o, x in zip(outs, want):
            assert torch.equal(o, x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, s, w in zip(streams, sets, ws):
            with torch.cuda.stream(st):
                got.append(call(s, w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    bad = []

    def work(i):
        for _ in range(30):
            if not torch.equal(call(sets[i], ws[i]), want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_refusals(ops, gpu):
    w = Batch([(9, 1), (20, 1)], 4, 2, 64, BF16, 30, decode=True)
    pool, tables, lens, _, _, q = w.on(gpu)
    call = lambda **kw: ops.paged_attention_gemv_fp4(**{**dict(q=q, kv_pool=pool, kv_page_tables=tables, kv_lens=lens, max_kv_len=21), **kw})
    for kw, message in ((dict(q=q.float()), "not implemented"), (dict(q=q[:3]), "multiple of n_kv_heads"), (dict(q=q[0]), "3-D"),
                        (dict(q=q[:, :1]), "kv_page_tables.size"), (dict(kv_lens=lens[:1]), "kv_lens.size"),
                        (dict(kv_lens=lens.long()), "kv_lens"), (dict(kv_page_tables=tables.long()), "kv_page_tables"),
                        (dict(kv_pool=pool[..., :-1]), "contiguous"), (dict(kv_pool=pool.cpu()), "kv_pool must be on"),
                        (dict(q=torch.zeros(4, 2, 72, dtype=BF16, device=gpu)), "head_dim"), (dict(max_kv_len=-1), "negative"),
                        (dict(max_kv_len=2**31), "out of range"), (dict(kv_lens=lens.cpu()), "kv_lens")):
        with pytest.raises(RuntimeError, match=message):
            call(**kw)
    with pytest.raises(ValueError):
        call(q=q.cpu())
    assert call(q=q[:, :0], kv_page_tables=tables[:0], kv_lens=lens[:0]).shape == (4, 0, 64)
