"""The 4-bit cache without a GPU: its format in the oracle, pool shapes, and what the entry points refuse."""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from femtovllm import fp4


@pytest.fixture(scope="module")
def C():
    from femtovllm import _C

    return _C


def test_pool_shapes(C):
    for dim in range(-16, 161):
        ok = 0 < dim <= 128 and dim % 16 == 0
        assert C._lib.femto_fp4_page_bytes(dim) == (of.page_bytes(dim) if ok else 0)
        if ok:
            assert fp4.page_bytes(dim) == of.page_bytes(dim) and of.page_bytes(dim) % 128 == 0
        else:
            with pytest.raises(ValueError):
                fp4.page_bytes(dim)
    pool = fp4.new_pool(3, 2, 80, device="cpu")
    assert pool.shape == (3, 2, 1664) and pool.dtype == torch.uint8 and not pool.any()


def test_oracle_rounding():
    """Each value of a block is the nearest of its list; ties, saturation, scales and NaN by hand."""
    x = np.zeros((1, 32))
    x[0, :16] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.25, -0.3, -5.01, 6.9, 0.2, -0.0]
    code, byte = of.quantize(x)
    assert byte[0, 0] == 127
    assert of.dequantize(code, byte, 32)[0, :16].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, 6, 6, 0, -0.5, -6, 6, 0, 0]
    assert code[0, 10] == 8 and code[0, 15] == 8  # the sign stays
    assert of.quantize(np.full((1, 32), 7.0))[1][0, 0] == 127 and of.quantize(np.full((1, 32), 7.001))[1][0, 0] == 128
    assert of.quantize(np.zeros((1, 32)))[1][0, 0] == 8 and of.quantize(np.full((1, 32), 2.0**-130))[1][0, 0] == 8
    big = of.quantize(np.full((1, 40), 3.3895e38))
    assert big[1].tolist() == [[252, 252]] and (of.dequantize(*big, 40) == 1.5 * 2.0**127).all()
    for bad in (np.inf, -np.inf, np.nan):
        y = np.ones((2, 64))
        y[1, 40] = bad
        code, byte = of.quantize(y)
        assert byte[0].tolist() == [125, 125] and byte[1].tolist() == [125, 255] and not code[1, 32:].any()
        assert np.isnan(of.dequantize(code, byte, 64)[1, 32:]).all()
    rng = np.random.default_rng(0)
    z = rng.standard_normal((50, 96)) * np.exp(rng.standard_normal((50, 96)))
    code, byte = of.quantize(z)
    back, step = of.dequantize(code, byte, 96), np.repeat(2.0 ** (byte.astype(float) - 127), 32, -1)
    assert (np.abs(back - z) <= step).all() and (np.abs(back) <= 6 * step).all()
    assert np.abs(back - z).max() > 0.2 * step.min()  # (it does round)


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 112, 128])
def test_oracle_layout(dim):
    """Rows come back from the page, every byte of it belongs to one row, and rows leave their neighbours alone."""
    rng = np.random.default_rng(dim)
    n = of.blocks(dim)
    pool = rng.integers(0, 256, (2, 3, of.page_bytes(dim)), dtype=np.uint8)
    start = pool.copy()
    k, v = rng.standard_normal((2, 16, 3, dim))
    changed = np.zeros(pool.shape[2], dtype=int)
    for r in rng.permutation(16):
        before = pool.copy()
        pool = of.write(pool, k[r : r + 1], v[r : r + 1], [16 + int(r)], [[0, 1]], None, dim)
        assert (pool[0] == start[0]).all()
        inv = 255 - before
        other = of.write(inv, k[r : r + 1], v[r : r + 1], [16 + int(r)], [[0, 1]], None, dim)
        changed += (pool[1, 0] == other[1, 0]) | ((pool[1, 0] ^ other[1, 0]) != 255)
        K, V = of.rows(pool, dim)
        assert np.array_equal(K[1, :, r], of.dequantize(*of.quantize(k[r]), dim))
        assert np.array_equal(V[1, :, r], of.dequantize(*of.quantize(v[r]), dim))
    assert (changed[: 512 * n] == 1).all() and changed[512 * n :].sum() == 2 * 16 * n
    K, V = of.rows(pool, dim)
    assert np.array_equal(K[1], of.dequantize(*of.quantize(k.transpose(1, 0, 2)), dim))
    got = of.read(pool, [16, 17], [[0, 1]], [0, 2], dim)
    assert np.array_equal(got[0], K[1].transpose(1, 0, 2)[:2]) and np.array_equal(got[1], V[1].transpose(1, 0, 2)[:2])


def _write(C, **kw):
    a = dict(dtype=2, k=16, kst=256, ksh=128, v=16, vst=256, vsh=128, pool=16, nb=8, kvh=2, d=128, cu=16, nseq=2, ntok=10,
             maxq=5, pos=16, tab=16, npages=4, ts=4, stream=None)
    a.update(kw)
    return C._lib.femto_kv_cache_write_fp4(*a.values())


def _read(C, **kw):
    a = dict(dtype=2, pool=16, nb=8, kvh=2, d=128, k=16, v=16, cu=16, nseq=2, ntok=10, maxq=5, pos=16, tab=16, npages=4, ts=4,
             stream=None)
    a.update(kw)
    return C._lib.femto_kv_cache_read_fp4(*a.values())


def _rope(C, **kw):
    a = dict(dtype=2, q=16, qst=512, qsh=128, k=16, kst=256, ksh=128, v=16, vst=256, vsh=128, out=16, ost=512, osh=128,
             qw=None, kw=None, eps=1e-6, cos=16, sin=16, rs=64, rows=100, r=128, il=0, pool=16, nb=8, h=4, kvh=2, d=128,
             cu=16, nseq=2, ntok=10, maxq=5, pos=16, tab=16, npages=4, ts=4, stream=None)
    a.update(kw)
    return C._lib.femto_rope_cache_write_fp4(*a.values())


@pytest.mark.parametrize("call", [_write, _read, _rope])
def test_library_refusals(C, call):
    """Each is refused before anything touches the (fake) pointers."""
    last = lambda: C._lib.femto_attn_last_error().decode()
    for dtype in (0, 5):
        assert call(C, dtype=dtype) == 2 and "not implemented" in last()
    for d in (0, 8, 100, 136, 144, -16):
        assert call(C, d=d) == 2 and "head_dim" in last()
    assert call(C, nseq=-1) == 1 and call(C, ntok=-1) == 1 and call(C, maxq=0) == 1 and "max_q_len" in last()
    assert call(C, cu=None) == 1 and "one token" in last()
    assert call(C, nseq=70000) == 1 and call(C, kvh=0) == 1 and call(C, nb=0) == 1 and call(C, ts=3) == 1
    for name in ("k", "v", "pool", "pos", "tab"):
        assert call(C, **{name: None}) == 1 and "null" in last()
    for name in ("k", "v", "pool"):
        assert call(C, **{name: 8}) == 1 and "aligned" in last()
    assert call(C, ntok=0) == 0 and call(C, nseq=0) == 0


def test_library_refusals_of_strides_and_tables(C):
    last = lambda: C._lib.femto_attn_last_error().decode()
    assert _write(C, ksh=100) == 1 and "strides" in last() and _write(C, vst=4) == 1
    for r in (0, 1, 63, 130, -2):
        assert _rope(C, r=r) == 1 and "rotary_dim must be even" in last()
    assert _rope(C, rs=32) == 1 and "tables too small" in last() and _rope(C, rows=0) == 1
    assert _rope(C, qw=16) == 1 and "both or not at all" in last()
    assert _rope(C, qw=16, kw=16, eps=-1.0) == 1 and "eps" in last() and _rope(C, qw=16, kw=16, eps=float("nan")) == 1
    assert _rope(C, qw=16, kw=24) == 1 and "aligned" in last() and _rope(C, cos=18) == 1 and _rope(C, qsh=100) == 1
    assert _rope(C, h=0) == 1 and _rope(C, q=None) == 1 and _rope(C, out=8) == 1


def test_ops_refuse_cpu_tensors():
    from femtovllm import ops

    x, t, i, pool = torch.zeros(2, 4, 64), torch.zeros(8, 32), torch.zeros(2, dtype=torch.int32), fp4.new_pool(2, 4, 64, "cpu")
    with pytest.raises(ValueError):
        ops.kv_cache_write_fp4(x, x, pool, i, i[:, None])
    with pytest.raises(ValueError):
        ops.kv_cache_read_fp4(pool, 64, torch.bfloat16, i, i[:, None])
    with pytest.raises(ValueError):
        ops.rope_cache_write_fp4(x, x, x, t, t, i, pool, i[:, None])
