"""Writes to and reads of the 4-bit cache on the GPU, byte for byte against the oracle.

A write's bytes are whole numbers and have to be equal, those around it too.  The prologue's norm is formed in float64
and its rotation step by step in float32, so its bytes are equal as well, and q is that float32 value rounded once.
"""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from femtovllm import fp4
from helpers import np64

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def rows(shape, dtype, gen, spread=1.0):
    x = torch.randn(shape, generator=gen) * torch.exp(spread * torch.randn((*shape[:-1], 1), generator=gen))
    return x.to(dtype)


def some_pool(num_blocks, heads, dim, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 256, (num_blocks, heads, fp4.page_bytes(dim)), generator=g, dtype=torch.uint8)


# (position of the first token, tokens) of each sequence
CHUNKS = [(0, 5), (15, 1), (7, 30), (0, 0), (33, 17), (16, 16)]


def batch(chunks, num_blocks, seed):
    order = np.random.default_rng(seed).permutation(num_blocks).tolist()
    tables, width = [], max(-(-(p + n) // 16) for p, n in chunks)
    for p, n in chunks:
        t = [order.pop() for _ in range(-(-(p + n) // 16))]
        tables.append(t + [-1] * (width - len(t)))
    cu = np.cumsum([0] + [n for _, n in chunks])
    pos = np.concatenate([np.arange(p, p + n) for p, n in chunks])
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32)
    return i32(tables), i32(cu), i32(pos), max(n for _, n in chunks)


def check_write(ops, gpu, k, v, dim, chunks, tables, cu, pos, max_q, seed):
    pool = some_pool(16, k.shape[1], dim, seed)
    dev = pool.to(gpu)
    ops.kv_cache_write_fp4(k.to(gpu), v.to(gpu), dev, pos.to(gpu), tables.to(gpu), None if cu is None else cu.to(gpu), max_q)
    want = of.write(pool.numpy(), np64(k), np64(v), pos.tolist(), tables.tolist(), None if cu is None else cu.tolist(), dim)
    assert np.array_equal(dev.cpu().numpy(), want)
    return dev, want


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 112, 128])
def test_write_chunks_and_read_back(ops, gpu, dim, dtype):
    gen = torch.Generator().manual_seed(dim)
    tables, cu, pos, max_q = batch(CHUNKS, 16, dim)
    k, v = (rows((len(pos), 3, dim), dtype, gen) for _ in range(2))
    dev, want = check_write(ops, gpu, k, v, dim, CHUNKS, tables, cu, pos, max_q, dim)
    for out in (BF16, F16):
        got = ops.kv_cache_read_fp4(dev, dim, out, pos.to(gpu), tables.to(gpu), cu.to(gpu), max_q)
        for x, y in zip(got, of.read(want, pos.tolist(), tables.tolist(), cu.tolist(), dim)):
            assert x.dtype == out and x.shape == (len(pos), 3, dim)
            assert torch.equal(x.cpu(), torch.tensor(y).to(out))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_write_one_token_each(ops, gpu, dtype):
    gen = torch.Generator().manual_seed(3)
    chunks = [(p, 1) for p in (0, 1, 15, 16, 31, 40, 2)]
    tables, _, pos, _ = batch(chunks, 16, 3)
    k, v = (rows((7, 5, 128), dtype, gen) for _ in range(2))
    dev, want = check_write(ops, gpu, k, v, 128, chunks, tables, None, pos, 1, 3)
    got = ops.kv_cache_read_fp4(dev, 128, BF16, pos.to(gpu), tables.to(gpu))
    for x, y in zip(got, of.read(want, pos.tolist(), tables.tolist(), None, 128)):
        assert np.array_equal(np64(x), y)


def test_values_at_the_borders(ops, gpu):
    """Ties, saturation, signs, subnormals, the largest numbers, infinities and NaN, whole blocks of zeros."""
    special = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0, 0.0]
    k = torch.zeros(10, 2, 128)
    for t in range(10):
        for b in range(4):
            s = 2.0 ** (t - 5) * (1.0, 2.0**20, 2.0**-20, 1.0)[b]
            k[t, 0, 32 * b : 32 * b + 10] = torch.tensor(special) * s
            k[t, 1, 32 * b : 32 * b + 10] = -torch.tensor(special) * s * (1 + 2.0**-6)
    k[3, 0, 5], k[4, 0, 40], k[5, 1, 127], k[6, 1, 64:96] = float("nan"), float("inf"), float("-inf"), 0.0
    k[7, 0, :32], k[7, 0, 32:64], k[7, 0, 64:96], k[7, 1] = 3.38e38, 1e-38, 2.0**-133, -0.0
    v = k.flip(0).flip(2)
    tables, cu, pos, max_q = batch([(3, 10)], 16, 1)
    dev, want = check_write(ops, gpu, k.to(BF16), v.to(BF16), 128, None, tables, cu, pos, max_q, 5)
    got = ops.kv_cache_read_fp4(dev, 128, BF16, pos.to(gpu), tables.to(gpu), cu.to(gpu), max_q)
    for x, y in zip(got, of.read(want, pos.tolist(), tables.tolist(), cu.tolist(), 128)):
        assert np.array_equal(np64(x), y, equal_nan=True)
    h = (k * 2.0**8).clamp(-65504, 65504)
    h[8, 0, 3], h[9, 1, 90] = 65504.0, 2.0**-24
    check_write(ops, gpu, h.to(F16), h.flip(1).to(F16), 128, None, tables, cu, pos, max_q, 6)


def test_reads_of_every_scale(ops, gpu):
    """Pages of random codes under scale bytes 1 to 255, as both types; a fresh pool reads as zeros."""
    pool = some_pool(8, 2, 112, 9)
    pool[..., 2048:] = (torch.arange(8 * 2 * 128) % 255 + 1).to(torch.uint8).reshape(8, 2, 128)
    tables, pos = torch.arange(8, dtype=torch.int32)[None], torch.arange(128, dtype=torch.int32)
    cu = torch.tensor([0, 128], dtype=torch.int32)
    for out in (BF16, F16):
        got = ops.kv_cache_read_fp4(pool.to(gpu), 112, out, pos.to(gpu), tables.to(gpu), cu.to(gpu), 128)
        for x, y in zip(got, of.read(pool.numpy(), pos.tolist(), tables.tolist(), cu.tolist(), 112)):
            want = torch.tensor(y).to(out)
            assert torch.equal(torch.isnan(x).cpu(), torch.isnan(want)) and torch.equal(x.cpu().nan_to_num(), want.nan_to_num())
        fresh = ops.kv_cache_read_fp4(fp4.new_pool(8, 2, 112, gpu), 112, out, pos.to(gpu), tables.to(gpu), cu.to(gpu), 128)
        assert not fresh[0].any() and not fresh[1].any()


@pytest.mark.parametrize("case", ["hole", "outside", "short", "negative", "far"])
def test_where_the_walk_ends(ops, gpu, case):
    """A token is written only if its column and all from the first token's on hold blocks; others read as zeros."""
    gen = torch.Generator().manual_seed(8)
    tables, cu, pos, max_q = batch([(5, 40), (0, 3)], 16, 8)
    if case == "hole":
        tables[0, 1] = -1
    elif case == "outside":
        tables[0, 1] = 16
    elif case == "short":
        tables = tables[:, :1]
    elif case == "negative":
        pos[:40] -= 6
    else:
        pos[:40] += 2**31 - 1 - 5 - 20  # wraps past the largest position
    k, v = (rows((43, 2, 64), BF16, gen) for _ in range(2))
    if case == "far":
        pool = some_pool(16, 2, 64, 1)
        dev = pool.to(gpu)
        ops.kv_cache_write_fp4(k.to(gpu), v.to(gpu), dev, pos.to(gpu), tables.to(gpu), cu.to(gpu), max_q)
        want = of.write(pool.numpy(), np64(k)[40:], np64(v)[40:], [0, 1, 2], tables[1:].tolist(), [0, 3], 64)
        assert np.array_equal(dev.cpu().numpy(), want)
        return
    dev, want = check_write(ops, gpu, k, v, 64, None, tables, cu, pos, max_q, 1)
    got = ops.kv_cache_read_fp4(dev, 64, BF16, pos.to(gpu), tables.to(gpu), cu.to(gpu), max_q)
    for x, y in zip(got, of.read(want, pos.tolist(), tables.tolist(), cu.tolist(), 64)):
        assert np.array_equal(np64(x), y)


def test_strided_sources_tables_and_an_understated_max_q_len(ops, gpu):
    """k and v as views of one projection, a table inside a wider array, max_q_len far below and above the longest chunk."""
    gen = torch.Generator().manual_seed(12)
    tables, cu, pos, _ = batch(CHUNKS, 16, 12)
    fused = rows((len(pos), 9, 128), BF16, gen).to(gpu)
    wide = torch.full((len(CHUNKS), 9), -1, dtype=torch.int32)
    wide[:, 2 : 2 + tables.shape[1]] = tables
    table = wide.to(gpu)[:, 2 : 2 + tables.shape[1]]
    pool = some_pool(16, 2, 128, 2)
    want = of.write(pool.numpy(), np64(fused[:, 5:7]), np64(fused[:, 7:9]), pos.tolist(), tables.tolist(), cu.tolist(), 128)
    for max_q in (1, 7, 30, 2**31 - 1):
        dev = pool.to(gpu)
        ops.kv_cache_write_fp4(fused[:, 5:7], fused[:, 7:9], dev, pos.to(gpu), table, cu.to(gpu), max_q)
        assert np.array_equal(dev.cpu().numpy(), want), max_q
        got = ops.kv_cache_read_fp4(dev, 128, BF16, pos.to(gpu), table, cu.to(gpu), max_q)
        for x, y in zip(got, of.read(want, pos.tolist(), tables.tolist(), cu.tolist(), 128)):
            assert np.array_equal(np64(x), y), max_q


def tables_for(rotary, rows_, seed=0):
    angle = np.random.default_rng(seed).uniform(0, 6.3, (rows_, rotary // 2))
    return torch.tensor(np.cos(angle), dtype=torch.float32), torch.tensor(np.sin(angle), dtype=torch.float32)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (128, 48), (64, 64), (80, 80), (112, 50), (48, 2), (16, 16), (96, 36)])
def test_prologue(ops, gpu, dim, rotary, interleaved, norm, dtype):
    gen = torch.Generator().manual_seed(dim + rotary)
    tables, cu, pos, max_q = batch(CHUNKS, 16, dim + rotary)
    T = len(pos)
    q, k, v = rows((T, 6, dim), dtype, gen), rows((T, 2, dim), dtype, gen), rows((T, 2, dim), dtype, gen)
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype) for _ in range(2))
    cos, sin = tables_for(rotary, 52, dim)
    pool = some_pool(16, 2, dim, 4)
    dev = pool.to(gpu)
    weights = dict(q_norm_weight=wq.to(gpu), k_norm_weight=wk.to(gpu), eps=1e-5) if norm else {}
    out = ops.rope_cache_write_fp4(q.to(gpu), k.to(gpu), v.to(gpu), cos.to(gpu), sin.to(gpu), pos.to(gpu), dev,
                                   tables.to(gpu), cu.to(gpu), max_q, interleaved, **weights)
    turned = lambda x, w: of.prologue(np64(x), np64(w) if norm else None, 1e-5, cos.numpy(), sin.numpy(), pos.tolist(), interleaved)
    assert torch.equal(out.cpu(), torch.tensor(turned(q, wq)).to(dtype))
    want = of.write(pool.numpy(), turned(k, wk), np64(v), pos.tolist(), tables.tolist(), cu.tolist(), dim)
    assert np.array_equal(dev.cpu().numpy(), want)


def test_prologue_in_place_strided_and_outside_the_tables(ops, gpu):
    """q, k and v as columns of one projection, out the q of it, one token each; a position past the tables gives NaN."""
    gen = torch.Generator().manual_seed(21)
    chunks = [(p, 1) for p in (0, 17, 3, 40)]
    tables, _, pos, _ = batch(chunks, 16, 21)
    fused = rows((4, 8, 128), BF16, gen)
    cos, sin = tables_for(128, 30)
    dev = some_pool(16, 2, 128, 6)
    start, dev, x = dev.numpy(), dev.to(gpu), fused.to(gpu)
    q = x[:, :4]
    out = ops.rope_cache_write_fp4(q, x[:, 4:6], x[:, 6:], cos.to(gpu), sin.to(gpu), pos.to(gpu), dev, tables.to(gpu), out=q)
    assert out.data_ptr() == x.data_ptr() and torch.equal(x[:, 4:].cpu(), fused[:, 4:])
    turned = lambda y: of.prologue(np64(y), None, 0, cos.numpy(), sin.numpy(), pos.tolist(), False)
    want_q = torch.tensor(turned(fused[:, :4])).to(BF16)
    assert torch.isnan(want_q[3]).all() and torch.isnan(out[3]).all() and torch.equal(out[:3].cpu(), want_q[:3])
    want = of.write(start, turned(fused[:, 4:6]), np64(fused[:, 6:]), pos.tolist(), tables.tolist(), None, 128)
    assert np.array_equal(dev.cpu().numpy(), want)


def test_refusals(ops, gpu):
    T, dim = 4, 64
    z = lambda *s, dt=BF16: torch.zeros(s, dtype=dt, device=gpu)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)
    pool, k, tab, pos, cu = fp4.new_pool(4, 2, dim, gpu), z(T, 2, dim), i32(1, 2), i32(T), torch.tensor([0, T], dtype=torch.int32, device=gpu)
    bad = [
        (dict(k=z(T, 2, dim, dt=torch.float32), v=z(T, 2, dim, dt=torch.float32)), "not implemented"),
        (dict(v=z(T, 2, dim, dt=F16)), "share a dtype"), (dict(v=z(T, 2, 32)), "one shape"),
        (dict(k=z(T, 1, dim), v=z(T, 1, dim)), "heads differ"), (dict(pool=pool[:, :, :-1]), "contiguous"),
        (dict(pool=pool[::2]), "contiguous"), (dict(pool=pool.view(torch.int8)), "uint8"),
        (dict(pool=fp4.new_pool(4, 2, dim, "cpu")), "kv_pool must be on"), (dict(pos=pos.long()), "positions"),
        (dict(pos=pos[:2]), "positions.numel"), (dict(tab=tab.long()), "kv_page_tables"), (dict(cu=cu.long()), "cu_seqlens"),
        (dict(cu=cu[:1]), "cu_seqlens"), (dict(cu=None), "one token"), (dict(max_q=2**40), "out of range"),
        (dict(max_q=0), "max_q_len"), (dict(k=z(T, 2, 136), v=z(T, 2, 136)), "head_dim"),
        (dict(k=z(T, 2, dim + 8)[..., 4 : 4 + dim]), "aligned"),
    ]
    for change, message in bad:
        a = dict(k=k, v=k, pool=pool, pos=pos, tab=tab, cu=cu, max_q=T)
        a.update(change)
        with pytest.raises(RuntimeError, match=message):
            ops.kv_cache_write_fp4(a["k"], a["v"], a["pool"], a["pos"], a["tab"], a["cu"], a["max_q"])
        with pytest.raises(RuntimeError, match=message):
            ops.rope_cache_write_fp4(a["k"], a["k"], a["v"], z(9, 32, dt=torch.float32), z(9, 32, dt=torch.float32), a["pos"],
                                     a["pool"], a["tab"], a["cu"], a["max_q"])
    for args in ((pool, 128, BF16), (pool, 64, torch.float32), (pool, 60, BF16)):
        with pytest.raises(RuntimeError):
            ops.kv_cache_read_fp4(*args, pos, tab, cu, T)
    q, t = z(T, 4, dim), z(9, 32, dt=torch.float32)
    rope = lambda **kw: ops.rope_cache_write_fp4(**{**dict(q=q, k=k, v=k, cos=t, sin=t, positions=pos, kv_pool=pool,
                                                           kv_page_tables=tab, cu_seqlens=cu, max_q_len=T), **kw})
    for kw, message in ((dict(q=z(T, 4, 32)), "q must be"), (dict(cos=t[:4]), "cos / sin"), (dict(cos=t.half()), "float32"),
                        (dict(q_norm_weight=z(dim)), "both or not at all"),
                        (dict(q_norm_weight=z(dim), k_norm_weight=z(32)), "k_norm_weight"),
                        (dict(q_norm_weight=z(dim), k_norm_weight=z(dim), eps=-1.0), "eps"), (dict(out=z(T, 4, 32)), "out must match"),
                        (dict(q=k, out=k), "no memory with"), (dict(cos=z(9, 40, dt=torch.float32), sin=z(9, 40, dt=torch.float32)), "rotary_dim")):
        with pytest.raises(RuntimeError, match=message):
            rope(**kw)
    empty = dict(q=z(0, 4, dim), k=z(0, 2, dim), v=z(0, 2, dim), positions=i32(0), cu_seqlens=i32(2))
    assert rope(**empty).shape == (0, 4, dim)
    assert not pool.any()
