"""Prefill over the 4-bit cache against the 64-bit oracle.  Bounds: as tests/test_fp4_decode_gpu.py."""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from fp4_helpers import Batch
from helpers import assert_close, np64, sample_rows

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
CHUNKS = [(0, 200), (100, 65), (333, 1), (1000, 130), (0, 1), (63, 64), (2000, 33), (5, 2)]


def run(ops, gpu, w, max_q_len=None):
    pool, tables, lens, cu, pos, q = w.on(gpu)
    return ops.paged_attention_gemm_fp4(q, pool, cu, max(n for _, n in w.chunks) if max_q_len is None else max_q_len, tables, lens, pos)


def check(ops, gpu, w, what, tokens=None, **kw):
    out = run(ops, gpu, w, **kw)
    want = of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos, tokens)
    mask = None
    if tokens is not None:
        mask = np.zeros(want.shape, dtype=bool)
        mask[:, sorted(tokens)] = True
    assert_close(out, want, w.dtype, what, mask=mask)
    return out


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", [(8, 8), (16, 8), (8, 2), (32, 4), (6, 2), (20, 1), (1, 1)])
def test_heads(ops, gpu, heads, dtype):
    check(ops, gpu, Batch(CHUNKS, *heads, 128, dtype, sum(heads)), f"heads {heads} {dtype}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112])
def test_dims(ops, gpu, dim, dtype):
    check(ops, gpu, Batch(CHUNKS, 8, 2, dim, dtype, dim), f"dim {dim} {dtype}")


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300])
def test_single_prompts(ops, gpu, n):
    check(ops, gpu, Batch([(0, n)], 4, 2, 128, BF16, n), f"prompt {n}")


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_key_split_and_many_sequences(ops, gpu, dtype):
    """One long sequence beside short ones (its query tiles are cut over their keys), more than 64 and than 256 sequences."""
    chunks = [(9000, 40)] + [(int(p), 3 + int(p) % 7) for p in np.random.default_rng(0).integers(0, 300, size=20)]
    w = Batch(chunks, 8, 2, 128, dtype, 1)
    check(ops, gpu, w, f"split {dtype}")
    rng = np.random.default_rng(2)
    for count in (80, 300):
        w = Batch([(int(rng.integers(0, 60)), int(rng.integers(0, 5))) for _ in range(count)] + [(400, 70)], 4, 2, 64, dtype, count)
        check(ops, gpu, w, f"{count} sequences {dtype}")


def test_repeated_calls_of_a_split_agree(ops, gpu):
    w = Batch([(6000, 64), (100, 20)], 8, 2, 128, F16, 4)
    first = run(ops, gpu, w)
    for _ in range(10):  # partials are merged in order, whoever comes last
        assert torch.equal(run(ops, gpu, w), first)


@pytest.mark.parametrize("max_q_len", [0, 1, 7, 2**31 - 1])
def test_max_q_len_only_plans(ops, gpu, max_q_len):
    check(ops, gpu, Batch(CHUNKS, 8, 2, 128, BF16, 5), f"max_q_len {max_q_len}", max_q_len=max_q_len)


def test_rows_beside_a_chunk(ops, gpu):
    """A chunk beside decode rows of uneven contexts, some empty chunks; only rows; more heads than a wave holds."""
    rng = np.random.default_rng(6)
    rows = [(int(n), 1) for n in rng.integers(0, 1500, size=40)]
    check(ops, gpu, Batch([(300, 150)] + rows + [(0, 0), (64, 0)], 16, 8, 128, BF16, 7), "rows beside a chunk")
    check(ops, gpu, Batch(rows, 20, 1, 80, F16, 8), "only rows")
    check(ops, gpu, Batch([(5000, 1), (0, 30), (20, 1)], 4, 1, 128, BF16, 9), "a long row")


def test_positions_of_their_own(ops, gpu):
    """Positions that are not the last ones: some past kv_len, some that see nothing (NaN), in no order."""
    w = Batch([(100, 90), (40, 1), (70, 1)], 8, 2, 128, BF16, 10)
    rng = np.random.default_rng(11)
    w.pos[:90] = rng.permutation(np.concatenate([np.arange(-5, 60), np.arange(170, 195)]))
    w.pos[90], w.pos[91] = -1, 10
    out = check(ops, gpu, w, "positions")
    assert torch.isnan(out[:, 90]).all() and torch.isnan(out[:, 0]).all() == bool(w.pos[0] < 0)


def test_kv_len_zero_and_blocks_outside(ops, gpu):
    w = Batch([(100, 40), (0, 9), (200, 70), (50, 1)], 8, 2, 128, BF16, 12)
    w.kv_lens[1] = 0
    w.tables[0, 2], w.tables[0, 8], w.tables[2, 0], w.tables[2, 16], w.tables[3, 1] = -1, len(w.pool), 2**31 - 1, -(2**31), -7
    out = check(ops, gpu, w, "outside")
    assert torch.isnan(out[:, 40:49]).all()
    w.tables = np.ascontiguousarray(w.tables[:, :10])
    check(ops, gpu, w, "a table of 10 columns")


@pytest.mark.parametrize("scale", [2.0**-20, 4.0, 30.0])
def test_flat_and_sharp_scores(ops, gpu, scale):
    """As the decode test of this name."""
    w = Batch([(100, 200), (0, 70), (300, 1)], 8, 2, 128, BF16, 13, scale=scale)
    out = run(ops, gpu, w)
    want = of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos)
    K, V = of.rows(w.pool, 128)
    off = 2.0**-14 * np.abs(np64(w.q)).max() * np.nanmax(np.abs(K).sum(-1)) / np.sqrt(128)
    bound = np.nanmax(np.abs(V)) * (2 * np.expm1(2 * off) + 2.0**-7) + 1e-2
    assert np.isfinite(np64(out)).all() and np.abs(np64(out) - want).max() <= bound
    if scale < 1:
        assert_close(out, want, BF16, f"scale {scale}")


def test_nan_keys(ops, gpu):
    """A NaN key of K reaches the heads of tokens that see it, and no other."""
    w = Batch([(100, 60), (10, 30)], 4, 2, 128, BF16, 14)
    w.pool[w.tables[0, 130 // 16], 1, 2048 + 4 * (130 % 16) + 1] = 255
    out = check(ops, gpu, w, "NaN key")
    nan = torch.isnan(out).cpu()
    assert nan[2:, 30:60].all() and nan.sum() == 2 * 30 * 128


def test_large_sampled(ops, gpu):
    w = Batch([(1500, 600), (0, 700), (4000, 300)], 16, 8, 128, BF16, 15)
    check(ops, gpu, w, "large", tokens=set(sample_rows(w.cu, 6, np.random.default_rng(0))))


def test_strided_q(ops, gpu):
    w = Batch(CHUNKS, 8, 2, 64, F16, 16)
    pool, tables, lens, cu, pos, q = w.on(gpu)
    wide = torch.zeros(q.size(1), 3, 8, 64, dtype=F16, device=gpu)
    wide[:, 1] = q.transpose(0, 1)
    a = ops.paged_attention_gemm_fp4(wide[:, 1].transpose(0, 1), pool, cu, 200, tables, lens, pos)
    assert torch.equal(a, ops.paged_attention_gemm_fp4(q, pool, cu, 200, tables, lens, pos))


def test_captured_calls(ops, gpu):
    ws = [Batch(c, 16, 8, 128, BF16, 20 + i) for i, c in enumerate(([(3000, 64), (10, 5)], [(0, 100)] + [(90, 1)] * 9))]
    sets = [w.on(gpu) for w in ws]
    call = lambda s, w: ops.paged_attention_gemm_fp4(s[5], s[0], s[3], max(n for _, n in w.chunks), s[1], s[2], s[4])
    want = [call(s, w) for s, w in zip(sets, ws)]
    graphs, outs = [], []
    for s, w in zip(sets, ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(s, w))
        graphs.append(g)
    for _ in range(4):
        for g in graphs:
            g.replay()
        again = call(sets[1], ws[1])
        torch.cuda.synchronize()
        for o, x in zip((*outs, again), (*want, want[1])):
            assert torch.equal(o, x)


def test_refusals(ops, gpu):
    w = Batch([(9, 10), (20, 1)], 4, 2, 64, BF16, 30)
    pool, tables, lens, cu, pos, q = w.on(gpu)
    call = lambda **kw: ops.paged_attention_gemm_fp4(**{**dict(q=q, kv_pool=pool, cu_seqlens=cu, max_q_len=10, kv_page_tables=tables,
                                                               kv_lens=lens, positions=pos), **kw})
    for kw, message in ((dict(q=q.float()), "not implemented"), (dict(q=q[:3]), "multiple of n_kv_heads"),
                        (dict(cu_seqlens=cu.long()), "cu_seqlens"), (dict(cu_seqlens=cu[:2]), "kv_page_tables.size"),
                        (dict(kv_lens=lens[:1]), "kv_lens.size"), (dict(positions=pos[:5]), "positions.numel"),
                        (dict(positions=pos.cpu()), "positions"), (dict(kv_pool=pool[..., :-1]), "contiguous"),
                        (dict(max_q_len=-1), "negative"), (dict(max_q_len=2**31), "out of range")):
        with pytest.raises(RuntimeError, match=message):
            call(**kw)
    with pytest.raises(ValueError):
        call(q=q.cpu())
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)
    assert call(q=q[:, :0], positions=pos[:0], cu_seqlens=i32(3)).shape == (4, 0, 64)
