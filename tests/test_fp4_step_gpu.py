"""The 4-bit cache's operators in a row, as a serving step has them: prologue, attention over what it wrote, and reads.

What is cached is compared byte for byte, attention within the bounds of tests/test_fp4_decode_gpu.py.
"""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from femtovllm import fp4
from fp4_helpers import Batch
from helpers import assert_close, np64, sample_rows

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
H, KVH, D = 8, 2, 128


class Model:
    """Rows of q, k and v, norm weights and tables, on the CPU."""

    def __init__(self, tokens, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g)
        self.q, self.k, self.v = r(tokens, H, D).to(dtype), r(tokens, KVH, D).to(dtype), r(tokens, KVH, D).to(dtype)
        self.qw, self.kw = (1 + 0.1 * r(D)).to(dtype), (1 + 0.1 * r(D)).to(dtype)
        angle = torch.arange(400)[:, None] / 10000 ** (torch.arange(D // 2) / (D // 2))
        self.cos, self.sin = angle.cos().float(), angle.sin().float()

    def prologue(self, pool, rows, pos, tables, cu, dtype):
        """(q rotated, rounded to the type (T, H, D), pool with the tokens)"""
        cos, sin = self.cos.numpy(), self.sin.numpy()
        rot = lambda x, w: of.prologue(np64(x[rows]), np64(w), 1e-6, cos, sin, pos, False)
        q = np64(torch.tensor(rot(self.q, self.qw)).to(dtype))
        return q, of.write(pool, rot(self.k, self.kw), np64(self.v[rows]), pos, tables, cu, D)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_steps(ops, gpu, dtype):
    """A prompt; its second chunk beside a new prompt and an empty slot; decode rows beside a chunk; decode, padded."""
    m = Model(160, dtype, 1)
    pool = np.zeros((24, KVH, of.page_bytes(D)), dtype=np.uint8)
    dev = fp4.new_pool(24, KVH, D, gpu)
    assert dev.shape == pool.shape
    dev.zero_()
    order = np.random.default_rng(2).permutation(24).astype(np.int32)
    tables = np.full((4, 8), -1, dtype=np.int32)
    for b in range(3):
        tables[b] = order[8 * b:8 * b + 8]
    w = {k: getattr(m, k).to(gpu) for k in ("cos", "sin", "qw", "kw")}
    t = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=gpu)
    have, used = np.zeros(4, dtype=int), 0
    for new in ([41, 0, 0, 0], [20, 33, 0, 0], [1, 1, 29, 0], [1, 1, 1, 0], [1, 1, 1, 0]):
        decode = max(new) == 1
        n = [1] * 4 if decode else new  # a padded slot has a row of its own in decode
        rows = np.arange(used, used + sum(n))
        used += sum(n)
        cu = np.concatenate([[0], np.cumsum(n)])
        pos = np.concatenate([have[b] + np.arange(n[b]) for b in range(4)])
        if decode:
            pos[3] = -1
        lens = have + np.array(new)
        q, pool = m.prologue(pool, rows, pos, tables, cu, dtype)
        got = ops.rope_cache_write_fp4(m.q[rows].to(gpu), m.k[rows].to(gpu), m.v[rows].to(gpu), w["cos"], w["sin"], t(pos), dev,
                                       t(tables), None if decode else t(cu), max(n), q_norm_weight=w["qw"], k_norm_weight=w["kw"])
        live = len(rows) - decode  # the padded row's q is NaN
        assert np.array_equal(np64(got)[:live], q[:live]) and np.array_equal(dev.cpu().numpy(), pool)
        heads = got.transpose(0, 1)
        if decode:
            out = ops.paged_attention_gemv_fp4(heads, dev, t(tables), t(lens), int(lens.max()))
            q[3] = 0
            want = of.decode(q.transpose(1, 0, 2), pool, tables, lens)
            assert not np64(out)[:, 3].any()
        else:
            out = ops.paged_attention_gemm_fp4(heads, dev, t(cu), max(n), t(tables), t(lens), t(pos))
            want = of.prefill(q.transpose(1, 0, 2), pool, cu, tables, lens, pos)
        assert_close(out, want, dtype, f"new {new}")
        k, v = ops.kv_cache_read_fp4(dev, D, dtype, t(pos), t(tables), None if decode else t(cu), max(n))
        wk, wv = of.read(pool, pos, tables, cu, D)
        assert np.array_equal(np64(k), wk) and np.array_equal(np64(v), wv)
        have = lens


def test_captured_steps(ops, gpu):
    """A decode step of a padded batch and a mixed step, captured side by side and replayed at other positions, with eager
    calls between: pools and outputs are the eager ones', bit by bit."""
    m = Model(200, BF16, 3)
    x = {k: getattr(m, k).to(gpu) for k in ("q", "k", "v", "cos", "sin", "qw", "kw")}
    t = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)
    perm = torch.randperm(96, generator=torch.Generator().manual_seed(4)).to(torch.int32)
    tables = perm.view(6, 16).to(gpu)
    tables[4:] = -1
    cu = t([0, 40, 41, 42, 43, 43, 43])

    def decode(pool, pos, lens):
        q = ops.rope_cache_write_fp4(x["q"][:6], x["k"][:6], x["v"][:6], x["cos"], x["sin"], pos, pool, tables, q_norm_weight=x["qw"],
                                     k_norm_weight=x["kw"])
        return ops.paged_attention_gemv_fp4(q.transpose(0, 1), pool, tables, lens, 256)

    def mixed(pool, pos, lens):
        ops.kv_cache_write_fp4(x["k"][50:93], x["v"][50:93], pool, pos, tables, cu, 40)
        k, v = ops.kv_cache_read_fp4(pool, D, BF16, pos, tables, cu, 40)
        return ops.paged_attention_gemm_fp4(x["q"][50:93].transpose(0, 1), pool, cu, 40, tables, lens, pos), k, v

    def state(step):
        first = [20 + step, 7, 100 + 3 * step, 15 + step, -1, -1]
        pos = [100 + step + i for i in range(40)] + [30 + step, 140 + step, 16 + step]
        return (t(first), t([p + 1 for p in first[:4]] + [0, 0])), (t(pos), t([140 + step, 31 + step, 141 + step, 17 + step, 0, 0]))

    start = torch.randint(0, 100, (96, KVH, fp4.page_bytes(D)), dtype=torch.uint8, generator=torch.Generator().manual_seed(5)).to(gpu)
    start[..., 2048:] = 120
    mine, theirs = start.clone(), start.clone()
    a, b = state(0)
    da, db = [y.clone() for y in a], [y.clone() for y in b]
    decode(start.clone(), *da)
    mixed(start.clone(), *db)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        out_d = decode(mine, *da)
    with torch.cuda.graph(graphs[1]):
        out_m = mixed(mine, *db)
    for step in (0, 1, 5, 2, 9):
        a, b = state(step)
        for to, y in zip((*da, *db), (*a, *b)):
            to.copy_(y)
        for g in graphs:
            g.replay()
        want_d, want_m = decode(theirs, *a), mixed(theirs, *b)
        torch.cuda.synchronize()
        assert torch.equal(mine, theirs), step
        assert torch.equal(out_d, want_d) and all(torch.equal(p, q) for p, q in zip(out_m, want_m)), step
        assert not out_d[:, 4:].any()


def test_a_pool_past_4_gib(ops, gpu):
    """Writes, reads and chunks beyond 32-bit byte offsets are those of a small pool."""
    blocks = (5 << 30) // (KVH * 8 * 2176) * 2  # 8 KV heads
    g = torch.Generator().manual_seed(6)
    r = lambda *s: torch.randn(s, generator=g).to(BF16).to(gpu)
    k, v, q = r(200, 8, D), r(200, 8, D), r(200, 16, D)
    cos, sin = r(200, D // 2).float(), r(200, D // 2).float()
    far = torch.empty((blocks, 8, 2176), dtype=torch.uint8, device=gpu)
    small = torch.zeros((32, 8, 2176), dtype=torch.uint8, device=gpu)
    assert far.numel() > 4 << 30
    far[-32:].zero_()
    tables = torch.randperm(32, generator=g).to(torch.int32).view(2, 16).to(gpu)
    cu = torch.tensor([0, 150, 200], dtype=torch.int32, device=gpu)
    pos = torch.cat([torch.arange(150), torch.arange(50)]).to(torch.int32).to(gpu)
    lens = torch.tensor([150, 50], dtype=torch.int32, device=gpu)
    got = []
    for pool, tab in ((far, tables + (blocks - 32)), (small, tables)):
        out = ops.rope_cache_write_fp4(q, k, v, cos, sin, pos, pool, tab, cu, 150)
        first = pool[-32:].clone()
        ops.kv_cache_write_fp4(v, k, pool, pos, tab, cu, 150)
        got.append([out, first, pool[-32:], *ops.kv_cache_read_fp4(pool, D, BF16, pos, tab, cu, 150),
                    ops.paged_attention_gemm_fp4(out.transpose(0, 1), pool, cu, 150, tab, lens, pos)])
    assert all(torch.equal(a, b) for a, b in zip(*got)) and got[1][1].any()


@pytest.mark.parametrize("new,rows", [(1100, 4), (1100, 40), (300, 40), (40, 60)])
def test_rows_and_tiles_in_every_order(ops, gpu, new, rows):
    """Rows that start before the tiles, all of them or the first 256 workgroups, tiles for both slots of a CU or for one,
    with their keys split or not (32/8 heads)."""
    rng = np.random.default_rng(new + rows)
    chunks = [(130, new)] + [(int(n), 1) for n in rng.integers(0, 700, size=rows)]
    w = Batch(chunks, 32, 8, D, BF16, new + rows)
    pool, tables, lens, cu, pos, q = w.on(gpu)
    out = ops.paged_attention_gemm_fp4(q, pool, cu, new, tables, lens, pos)
    tokens = set(sample_rows(w.cu[:2], 6, rng)) | set(range(new, new + rows))
    want = of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos, tokens)
    mask = np.zeros(want.shape, dtype=bool)
    mask[:, sorted(tokens)] = True
    assert_close(out, want, BF16, f"{new} beside {rows}", mask=mask)
    again = ops.paged_attention_gemm_fp4(q, pool, cu, new, tables, lens, pos)
    assert torch.equal(again, out)  # partials are merged in order


@pytest.mark.parametrize("count", [63, 64, 65, 300, 5000])
def test_many_sequences(ops, gpu, count):
    """A wave finds its token's sequence among many, empty ones too (at both ends); rows behind the last sequence and before
    the first stay as they were."""
    rng = np.random.default_rng(count)
    n = rng.choice([0, 1, 2, 17], size=count, p=[0.4, 0.3, 0.2, 0.1])
    n[0] = n[-1] = n[-2] = 0
    cu = np.concatenate([[3], 3 + np.cumsum(n)])
    T, dim = int(cu[-1]) + 4, 16
    pos = np.concatenate([[0] * 3, *(np.arange(m) + int(rng.integers(0, 14)) for m in n), [0] * 4])
    tables = rng.permutation(2 * count).reshape(count, 2)
    g = torch.Generator().manual_seed(count)
    k, v, q = (torch.randn((T, 1, dim), generator=g).to(F16) for _ in range(3))
    cos, sin = torch.randn((40, 8), generator=g), torch.randn((40, 8), generator=g)
    start = rng.integers(0, 100, size=(2 * count, 1, of.page_bytes(dim))).astype(np.uint8)
    t = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=gpu)
    mine = slice(3, T - 4)
    dev = torch.tensor(start, device=gpu)
    ops.kv_cache_write_fp4(k.to(gpu), v.to(gpu), dev, t(pos), t(tables), t(cu), 17)
    want = of.write(start, np64(k), np64(v), pos, tables, cu, dim)
    assert np.array_equal(dev.cpu().numpy(), want)
    rk, rv = ops.kv_cache_read_fp4(dev, dim, F16, t(pos), t(tables), t(cu), 17)
    wk, wv = of.read(want, pos, tables, cu, dim)
    assert np.array_equal(np64(rk)[mine], wk[mine]) and np.array_equal(np64(rv)[mine], wv[mine])
    dev = torch.tensor(start, device=gpu)
    out = torch.full((T, 1, dim), 7.0, dtype=F16, device=gpu)
    ops.rope_cache_write_fp4(q.to(gpu), k.to(gpu), v.to(gpu), cos.to(gpu), sin.to(gpu), t(pos), dev, t(tables), t(cu), 17, out=out)
    turned = lambda x: of.prologue(np64(x), None, 0, cos.numpy(), sin.numpy(), pos, False)
    assert np.array_equal(np64(out)[mine], np64(torch.tensor(turned(q)).to(F16))[mine])
    assert (out[:3] == 7).all() and (out[-4:] == 7).all()
    assert np.array_equal(dev.cpu().numpy(), of.write(start, turned(k), np64(v), pos, tables, cu, dim))


@pytest.mark.parametrize("heads", [(8, 8), (4, 2), (8, 2)])
def test_nan_values_of_later_tokens(ops, gpu, heads):
    """V of a later token that is NaN: no token of an earlier query tile (at most 128 tokens) changes, those that see it are
    NaN in its 32 dims."""
    w = Batch([(50, 400), (7, 1)], *heads, D, BF16, sum(heads))
    pool, tables, lens, cu, pos, q = w.on(gpu)
    run = lambda p: ops.paged_attention_gemm_fp4(q, p, cu, 400, tables, lens, pos)
    want = run(pool)
    for token in (390, 399, 200):
        key = 50 + token
        bad = w.pool.copy()
        bad[w.tables[0, key // 16], :, 2 * 1024 + 64 + 16 * (key % 16 // 4) + 4 * 2 + key % 4] = 255  # V's block 2
        got = run(torch.tensor(bad, device=gpu))
        first = token // 128 * 128
        assert torch.equal(got[:, :first], want[:, :first]) and torch.equal(got[:, 400], want[:, 400])
        assert torch.isnan(got[:, token:400, 64:96]).all()
        assert torch.equal(got[:, :400, :64], want[:, :400, :64]) and torch.equal(got[:, :400, 96:], want[:, :400, 96:])
