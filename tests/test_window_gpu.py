"""Window attention (paged_attention_gemv_window / paged_attention_gemm_window) against the 64-bit oracle.

Bounds: those of the operators without a window (helpers.assert_close).  The kernels compute the same sums over
fewer keys: P rounds to the storage type (at most eps / 2 relative per weight), the output once more.
"""

import threading

import numpy as np
import pytest
import torch

import oracle.added as oa
from femtovllm import workloads
from femtovllm.metadata import build_varlen_metadata
from helpers import assert_agree, assert_close, np32, np64, np_tables

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def free_hidden_blocks(w, window, sinks):
    """Table entries of blocks that no token of the batch sees become -1 (a serving engine hands those blocks
    back), and rows that no token sees in the blocks that stay become NaN."""
    for b, (p, n) in enumerate(w.chunks):
        first = max(0, p - window + 1)
        hidden = [j for j in range(first) if j >= sinks]
        for j in hidden:
            blk = w.raw_block_tables[b][j // 16]
            if blk >= 0:
                w.k_pool[blk, :, j % 16] = float("nan")
                w.v_pool[blk, :, j % 16] = float("nan")
        for c in range(len(w.raw_block_tables[b])):
            if all(j >= sinks and j < first for j in range(16 * c, 16 * c + 16)):
                w.raw_block_tables[b][c] = -1
    return w


def run_decode(ops, w, device, window, sinks):
    q, meta = w.gemv_call(device=device)
    wd = w.to(device)
    out = ops.paged_attention_gemv_window(q.to(device), wd.k_pool, wd.v_pool, meta.block_tables, meta.kv_lens,
                                          meta.max_kv_len, window, sinks)
    want = oa.window_decode(np64(q), np32(w.k_pool), np32(w.v_pool), np_tables(meta), meta.kv_lens.tolist(), window, sinks)
    return out, want


LENS = [1, 2, 15, 16, 17, 64, 65, 129, 300, 1000]


@pytest.mark.usefixtures("decode_path")
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (15, 0), (16, 16), (17, 3), (64, 4), (100, 33), (257, 0),
                                          (999, 1), (5000, 4), (40, 2000)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_decode_windows(ops, gpu, dtype, window, sinks):
    w = workloads.make_paged_workload("window", [(L - 1, 1) for L in LENS], 8, 4, dtype=dtype, seed=window + sinks)
    out, want = run_decode(ops, free_hidden_blocks(w, window, sinks), gpu, window, sinks)
    assert_close(out, want, dtype, f"window {window} sinks {sinks} {dtype}")


@pytest.mark.usefixtures("decode_path")
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads", [(8, 8), (32, 8), (64, 8), (6, 1), (12, 4)])
@pytest.mark.parametrize("dim", [128, 80, 8])
def test_decode_heads_and_dims(ops, gpu, heads, dim, dtype):
    w = workloads.make_paged_workload("heads", [(L - 1, 1) for L in (1, 40, 700, 333)], *heads, head_dim=dim,
                                      dtype=dtype, seed=sum(heads))
    out, want = run_decode(ops, free_hidden_blocks(w, 150, 5), gpu, 150, 5)
    assert_close(out, want, dtype, f"heads {heads} dim {dim}")


@pytest.mark.usefixtures("decode_path")
def test_decode_long_contexts_and_empty_slots(ops, gpu):
    """Contexts past 8192 keys, more sequences than a wave has lanes, and slots without keys (zeros)."""
    rng = np.random.default_rng(3)
    lens = [20000, 9000] + [int(x) for x in rng.integers(1, 1500, size=70)]
    w = workloads.make_paged_workload("long", [(L - 1, 1) for L in lens], 4, 2, seed=4)
    window, sinks = 600, 20
    free_hidden_blocks(w, window, sinks)
    q, meta = w.gemv_call(device=gpu)
    wd, kv_lens = w.to(gpu), meta.kv_lens.clone()
    kv_lens[5] = kv_lens[66] = kv_lens[71] = 0
    meta.block_tables[5] = meta.block_tables[66] = meta.block_tables[71] = -1
    out = ops.paged_attention_gemv_window(q.to(gpu), wd.k_pool, wd.v_pool, meta.block_tables, kv_lens, 20000, window, sinks)
    want = oa.window_decode(np64(q), np32(w.k_pool), np32(w.v_pool), np_tables(meta), kv_lens.tolist(), window, sinks)
    assert (out[:, [5, 66, 71]] == 0).all()
    assert_close(out, want, BF16, "long contexts")


@pytest.mark.usefixtures("decode_path")
def test_decode_whole_context_agrees_with_the_plain_call(ops, gpu):
    """A window past the context: two kernels, each within the bounds of the exact value."""
    w = workloads.make_paged_workload("whole", [(L - 1, 1) for L in LENS], 16, 8, seed=9)
    q, meta = w.gemv_call(device=gpu)
    wd, q = w.to(gpu), q.to(gpu)
    a = ops.paged_attention_gemv(q, wd.k_pool, wd.v_pool, meta.block_tables, meta.kv_lens, meta.max_kv_len)
    for window, sinks in ((1000, 0), (1 << 40, 0), (3, 1000)):
        b = ops.paged_attention_gemv_window(q, wd.k_pool, wd.v_pool, meta.block_tables, meta.kv_lens, meta.max_kv_len,
                                            window, sinks)
        assert_agree(b, a, BF16, f"window {window}")


@pytest.mark.usefixtures("decode_path")
def test_decode_infinities_of_visible_keys(ops, gpu):
    """An infinite V of a visible key is an infinite output, also in the last row of a context."""
    w = workloads.make_paged_workload("inf", [(L - 1, 1) for L in (100, 37, 16)], 4, 2, seed=10)
    for b, j in ((0, 99), (1, 30), (2, 15)):
        w.v_pool[w.raw_block_tables[b][j // 16], :, j % 16, 3] = float("inf")
    for b, j in ((0, 60), (1, 3)):  # hidden
        w.v_pool[w.raw_block_tables[b][j // 16], :, j % 16] = float("-inf")
    out, want = run_decode(ops, w, gpu, 12, 2)
    assert torch.isinf(out[:, :, 3]).all() and (out[:, :, 3] > 0).all()
    keep = [d for d in range(128) if d != 3]
    assert_close(out[:, :, keep], want[:, :, keep], BF16, "beside an infinity")


def run_prefill(ops, w, device, window, sinks, rows=None, meta=None):
    q, m = w.gemm_call(device=device)
    meta = meta or m
    wd = w.to(device)
    out = ops.paged_attention_gemm_window(q.to(device), wd.k_pool, wd.v_pool, meta.cu_seqlens, meta.max_q_len,
                                          meta.block_tables, meta.kv_lens, meta.positions, window, sinks)
    want = oa.window_prefill(np64(q), np32(w.k_pool), np32(w.v_pool), meta.cu_seqlens.tolist(), np_tables(meta),
                             meta.kv_lens.tolist(), meta.positions.cpu().numpy(), window, sinks, rows)
    return out, want


CHUNKS = [(0, 200), (100, 65), (333, 1), (1000, 130), (0, 1), (63, 64), (2000, 33)]


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 4), (16, 0), (63, 1), (64, 64), (65, 70), (128, 4), (200, 0),
                                          (700, 17), (5000, 4), (30, 3000)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_windows(ops, gpu, dtype, window, sinks):
    w = workloads.make_paged_workload("pre", CHUNKS, 8, 4, dtype=dtype, seed=100 + window + sinks)
    out, want = run_prefill(ops, free_hidden_blocks(w, window, sinks), gpu, window, sinks)
    assert_close(out, want, dtype, f"window {window} sinks {sinks} {dtype}")


@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (16, 2), (6, 2), (3, 1)])
@pytest.mark.parametrize("dim", [128, 80, 16])
def test_prefill_heads_and_dims(ops, gpu, heads, dim):
    w = workloads.make_paged_workload("pre", CHUNKS, *heads, head_dim=dim, seed=sum(heads) + dim)
    out, want = run_prefill(ops, free_hidden_blocks(w, 90, 5), gpu, 90, 5)
    assert_close(out, want, BF16, f"heads {heads} dim {dim}")


@pytest.mark.parametrize("window,sinks", [(1500, 0), (4000, 100), (700, 4)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefill_key_split(ops, gpu, dtype, window, sinks):
    """Few query tiles over many keys: the call splits its keys over workgroups and merges them."""
    w = workloads.make_paged_workload("split", [(6000, 70), (20, 40)], 4, 2, dtype=dtype, seed=window)
    for _ in range(2):  # the counters are left zero
        out, want = run_prefill(ops, free_hidden_blocks(w, window, sinks), gpu, window, sinks)
        assert_close(out, want, dtype, f"split, window {window}")


@pytest.mark.parametrize("heads", [(16, 8), (32, 8), (16, 2)])
def test_mixed_batch(ops, gpu, heads):
    """One chunk beside decode rows: 70 of them (more than a wave's lanes), then few."""
    rng = np.random.default_rng(5)
    for rows in (70, 3):
        chunks = [(900, 100)] + [(int(x) - 1, 1) for x in rng.integers(1, 1500, size=rows)]
        w = workloads.make_paged_workload("mixed", chunks, *heads, seed=rows)
        out, want = run_prefill(ops, free_hidden_blocks(w, 200, 5), gpu, 200, 5)
        assert_close(out, want, BF16, f"mixed {heads} {rows} rows")


def test_prefill_other_positions(ops, gpu):
    """Positions that are not the consecutive ones up to kv_len - 1: shuffled, repeated, past the context (only the
    sinks, or nothing: NaN), a decode row past its context."""
    w = workloads.make_paged_workload("pos", [(500, 140), (80, 40), (100, 1)], 4, 2, seed=8)
    rng = np.random.default_rng(8)
    for sinks in (0, 9):
        _, meta = w.gemm_call(device=gpu)
        pos = meta.positions.cpu().numpy().copy()
        pos[:140] = rng.integers(0, 640, size=140)
        pos[140:160] = 90
        pos[160:170] = 2000
        pos[180] = 175 if sinks else 400
        meta.positions = torch.from_numpy(pos).to(gpu)
        out, want = run_prefill(ops, w, gpu, 77, sinks, meta=meta)
        assert_close(out, want, BF16, f"positions, sinks {sinks}")
        assert np.isnan(np64(out[:, 160:170])).all() == (sinks == 0)


def test_prefill_whole_context_agrees_with_the_plain_call(ops, gpu):
    """Two kernels, each within the bounds of the exact value: they differ by at most twice those."""
    w = workloads.make_paged_workload("whole", CHUNKS, 8, 4, seed=12)
    q, meta = w.gemm_call(device=gpu)
    wd, q = w.to(gpu), q.to(gpu)
    a = ops.paged_attention_gemm(q, wd.k_pool, wd.v_pool, meta.cu_seqlens, meta.max_q_len, 32, meta.cu_q_tiles,
                                 meta.q_tile_to_seq_idx, meta.block_tables, meta.kv_lens, meta.positions)
    for window, sinks in ((3000, 0), (1 << 35, 0)):
        b = ops.paged_attention_gemm_window(q, wd.k_pool, wd.v_pool, meta.cu_seqlens, meta.max_q_len, meta.block_tables,
                                            meta.kv_lens, meta.positions, window, sinks)
        assert_agree(b, a, BF16, f"window {window}")


def test_long_prompt(ops, gpu):
    """The last chunk of a 32k prompt, sampled rows."""
    w = workloads.make_paged_workload("long", [(30720, 2048)], 4, 1, seed=13)
    rows = {0, 1, 31, 32, 63, 64, 1000, 1023, 1024, 2046, 2047}
    out, want = run_prefill(ops, free_hidden_blocks(w, 4096, 4), gpu, 4096, 4, rows=rows)
    idx = sorted(rows)
    assert_close(out[:, idx], want[:, idx], BF16, "32k prompt")


@pytest.mark.usefixtures("decode_path")
@pytest.mark.parametrize("heads", [(17, 1), (48, 2), (40, 1)])
def test_decode_more_query_heads_than_a_wave_holds(ops, gpu, heads):
    """Ratios above 16: a KV head's query heads in two or three groups, the last one smaller."""
    w = workloads.make_paged_workload("ratio", [(L - 1, 1) for L in (900, 33, 1)], *heads, seed=sum(heads))
    out, want = run_decode(ops, free_hidden_blocks(w, 420, 3), gpu, 420, 3)
    assert_close(out, want, BF16, f"heads {heads}")
    w = workloads.make_paged_workload("ratio", [(300, 40), (899, 1), (0, 1)], *heads, seed=sum(heads) + 1)
    out, want = run_prefill(ops, free_hidden_blocks(w, 420, 3), gpu, 420, 3)
    assert_close(out, want, BF16, f"prefill, heads {heads}")


@pytest.mark.parametrize("window", [385, 4000, 20000])
@pytest.mark.parametrize("lens", [[30000], [21000, 700], [5000, 5001, 1, 16]])
def test_decode_rows_in_parts(ops, gpu, lens, window):
    """Few rows over many pages: parts of a row in several workgroups, ends anywhere in a part, sequences shorter than
    the parts; the same bits every time, whichever part ends last."""
    w = workloads.make_paged_workload("parts", [(L - 1, 1) for L in lens], 8, 2, dtype=F16, seed=len(lens) + window)
    free_hidden_blocks(w, window, 5)
    out, want = run_decode(ops, w, gpu, window, 5)
    assert_close(out, want, F16, f"window {window} lens {lens}")
    again, _ = run_decode(ops, w, gpu, window, 5)
    assert torch.equal(again, out)


@pytest.mark.parametrize("chunk", [(2000, 100), (0, 5)])
def test_mixed_batch_rows_in_parts(ops, gpu, chunk):
    """Two rows of many pages beside a chunk: the rows are cut too."""
    w = workloads.make_paged_workload("parts", [(9000, 1), chunk, (4500, 1)], 8, 2, seed=chunk[1])
    free_hidden_blocks(w, 6000, 20)
    first, want = run_prefill(ops, w, gpu, 6000, 20)
    assert_close(first, want, BF16, f"rows in parts beside {chunk}")
    again, _ = run_prefill(ops, w, gpu, 6000, 20)
    assert torch.equal(again, first)


def test_rows_behind_the_last_sequence_stay(ops, gpu):
    """Queries past cu_seqlens[-1] (a padded batch): no kernel writes their rows, whatever they hold."""
    w = workloads.make_paged_workload("pad", [(300, 50), (700, 1), (0, 9)], 8, 4, seed=30)
    q, meta = w.gemm_call(device=gpu)
    wd = w.to(gpu)
    n = q.size(1)
    padded = torch.full((8, n + 20, 128), float("nan"), dtype=BF16, device=gpu)
    padded[:, :n] = q.to(gpu)
    pos = torch.full((n + 20,), -7, dtype=torch.int32, device=gpu)
    pos[:n] = meta.positions
    out = ops.paged_attention_gemm_window(padded, wd.k_pool, wd.v_pool, meta.cu_seqlens, meta.max_q_len, meta.block_tables,
                                          meta.kv_lens, pos, 100, 2)
    want = oa.window_prefill(np64(q), np32(w.k_pool), np32(w.v_pool), meta.cu_seqlens.tolist(), np_tables(meta),
                             meta.kv_lens.tolist(), meta.positions.cpu().numpy(), 100, 2)
    assert out.shape == padded.shape
    assert_close(out[:, :n], want, BF16, "padded batch")


def test_pools_past_4_gib(ops, gpu):
    """The same blocks in a compact pool and at the end of one of 4.3 GiB: equal bits, decode and prefill."""
    w = workloads.make_paged_workload("big", [(2048, 1), (4000, 1), (900, 200), (30, 1)], 16, 8, seed=31, poison=False)
    blocks, n = 140_000, w.k_pool.size(0)
    outs = []
    for base in (0, blocks - n):
        pools = []
        for pool in (w.k_pool, w.v_pool):
            big = torch.empty((base + n,) + tuple(pool.shape[1:]), dtype=BF16, device=gpu)
            big[base:] = pool.to(gpu)
            pools.append(big)
        q, meta = w.gemm_call(device=gpu)
        q, tables = q.to(gpu), torch.where(meta.block_tables >= 0, meta.block_tables + base, meta.block_tables)
        outs.append([ops.paged_attention_gemm_window(q, *pools, meta.cu_seqlens, meta.max_q_len, tables, meta.kv_lens,
                                                     meta.positions, 700, 16),
                     ops.paged_attention_gemv_window(q[:, :4].contiguous(), *pools, tables, meta.kv_lens, 4001, 700, 16)])
        torch.cuda.synchronize()
        del pools
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_calls_of_two_threads(ops, gpu):
    """Two host threads, a stream each, calls whose rows are cut into parts: every result is the one alone."""
    calls, want = [], []
    for i, lens in enumerate(([20000], [9000, 12000])):
        w = workloads.make_paged_workload("threads", [(L - 1, 1) for L in lens], 8, 4, seed=40 + i)
        q, meta = w.gemv_call(device=gpu)
        wd, q = w.to(gpu), q.to(gpu)
        calls.append(lambda q=q, wd=wd, m=meta: ops.paged_attention_gemv_window(q, wd.k_pool, wd.v_pool, m.block_tables,
                                                                                m.kv_lens, m.max_kv_len, 8000, 4))
        want.append(calls[-1]())
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i].append(calls[i]())
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20 and all(torch.equal(x, want[i]) for x in got[i])


def test_strided_and_other_stream(ops, gpu):
    """q as the projection leaves it, a table that is a slice of a wider one, and a stream of its own."""
    w = workloads.make_paged_workload("strides", [(300, 90), (50, 1)], 8, 4, seed=14)
    q, meta = w.gemm_call(device=gpu)
    wd = w.to(gpu)
    q3 = q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    wide = torch.full((2, meta.block_tables.size(1) + 7), -5, dtype=torch.int32, device=gpu)
    wide[:, : meta.block_tables.size(1)] = meta.block_tables
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.paged_attention_gemm_window(q3, wd.k_pool, wd.v_pool, meta.cu_seqlens, meta.max_q_len,
                                              wide[:, : meta.block_tables.size(1)], meta.kv_lens, meta.positions, 60, 2)
    side.synchronize()
    want = oa.window_prefill(np64(q), np32(w.k_pool), np32(w.v_pool), meta.raw_cu_seqlens, np_tables(meta),
                             meta.kv_lens.tolist(), np.array(meta.raw_positions), 60, 2)
    assert_close(out, want, BF16, "strides")


@pytest.mark.usefixtures("decode_path")
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_blocks_of_seen_pages_read_as_zeros(ops, gpu, dtype):
    """Table entries that are -1, past the pool or past a narrow table, in pages that queries see."""
    w = workloads.make_paged_workload("bad", [(L - 1, 1) for L in (400, 77, 33, 250)], 8, 4, dtype=dtype, seed=17)
    for b, c, x in ((0, 24, -1), (0, 20, 10**6), (0, 0, 2**31 - 1), (1, 4, -7), (2, 2, -(2**31))):
        w.raw_block_tables[b][c] = x
    out, want = run_decode(ops, w, gpu, 90, 5)
    assert_close(out, want, dtype, "bad blocks")
    q, meta = w.gemv_call(device=gpu)
    wd, narrow = w.to(gpu), meta.block_tables[:, :14].contiguous()
    out = ops.paged_attention_gemv_window(q.to(gpu), wd.k_pool, wd.v_pool, narrow, meta.kv_lens, meta.max_kv_len, 90, 5)
    want = oa.window_decode(np64(q), np32(w.k_pool), np32(w.v_pool), narrow.cpu().numpy(), meta.kv_lens.tolist(), 90, 5)
    assert_close(out, want, dtype, "narrow table")
    if dtype == F32:
        return
    w = workloads.make_paged_workload("bad", [(300, 100), (76, 1), (0, 33), (240, 10)], 8, 4, dtype=dtype, seed=18)
    for b, c, x in ((0, 24, -1), (0, 20, 10**6), (0, 0, 2**31 - 1), (1, 4, -7), (2, 2, -(2**31))):
        w.raw_block_tables[b][c] = x
    out, want = run_prefill(ops, w, gpu, 90, 5)
    assert_close(out, want, dtype, "bad blocks, prefill")


@pytest.mark.parametrize("window", [1, 70, 2**31 - 1])
def test_prefill_negative_positions(ops, gpu, window):
    """A token before the sequence's start sees nothing, in a chunk and as a decode row: NaN; its neighbours as always."""
    w = workloads.make_paged_workload("neg", [(100, 40), (50, 1), (60, 1)], 4, 2, seed=15)
    _, meta = w.gemm_call(device=gpu)
    pos = meta.positions.cpu().numpy().copy()
    pos[[3, 20]] = [-1, -(2**31)]
    pos[40] = -9
    meta.positions = torch.from_numpy(pos).to(gpu)
    out, want = run_prefill(ops, w, gpu, window, 5, meta=meta)
    assert torch.isnan(out[:, [3, 20, 40]]).all()
    assert_close(out, want, BF16, f"negative positions, window {window}")


def test_decode_many_sequences(ops, gpu):
    """More (sequence, KV head) pairs than a call has counters: whole rows, whatever their length."""
    rng = np.random.default_rng(16)
    w = workloads.make_paged_workload("many", [(int(x), 1) for x in rng.integers(0, 60, size=2100)], 4, 2, dtype=F16, seed=16)
    out, want = run_decode(ops, free_hidden_blocks(w, 25, 3), gpu, 25, 3)
    assert_close(out, want, F16, "2100 sequences")


@pytest.mark.parametrize("entry", ["decode", "decode_f32", "prefill"])
def test_captured_calls_share_no_workspace(ops, gpu, entry):
    """Two graphs captured on one stream and eager calls of other sizes between their replays, also on two streams
    at once: every replay gives its eager result, with new inputs too."""
    chunks = {"decode": [[(2999, 1), (1700, 1)], [(5000, 1)] * 3], "decode_f32": [[(2999, 1)], [(5000, 1)] * 2], "prefill": [[(3000, 40), (300, 1)], [(5000, 60), (20, 1), (77, 1)]]}
    window, sinks = 1500, 4
    calls, graphs = [], []
    side = torch.cuda.Stream()
    for i, c in enumerate(chunks[entry]):
        w = workloads.make_paged_workload("graph", c, 8, 4, dtype=F32 if entry == "decode_f32" else BF16, seed=20 + i)
        q, meta = w.gemm_call(device=gpu)
        wd, q = w.to(gpu), q.to(gpu)
        if entry != "prefill":
            f = lambda q=q, wd=wd, m=meta: ops.paged_attention_gemv_window(q, wd.k_pool, wd.v_pool, m.block_tables, m.kv_lens,
                                                                           m.max_kv_len, window, sinks)
        else:
            f = lambda q=q, wd=wd, m=meta: ops.paged_attention_gemm_window(q, wd.k_pool, wd.v_pool, m.cu_seqlens, m.max_q_len,
                                                                           m.block_tables, m.kv_lens, m.positions, window, sinks)
        f()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = f()
        calls.append((f, q))
        graphs.append((g, out))
    other = torch.cuda.Stream()
    for turn in range(4):
        for f, q in calls:
            q.copy_(torch.randn_like(q))
        want = [f() for f, _ in calls]
        torch.cuda.synchronize()
        for g, out in graphs:
            out.fill_(7)
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        again = calls[1][0]()
        torch.cuda.synchronize()
        for (_, out), x in zip(graphs, want):
            assert torch.equal(out, x), f"turn {turn}"
        assert torch.equal(again, want[1])


def test_empty_calls(ops, gpu):
    pool = torch.zeros(2, 4, 16, 128, dtype=BF16, device=gpu)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)
    out = ops.paged_attention_gemv_window(torch.zeros(8, 0, 128, dtype=BF16, device=gpu), pool, pool, i32(0, 1), i32(0), 0, 5)
    assert out.shape == (8, 0, 128)
    out = ops.paged_attention_gemm_window(torch.zeros(8, 0, 128, dtype=BF16, device=gpu), pool, pool, i32(1), 0, i32(0, 1),
                                          i32(0), i32(0), 5)
    assert out.shape == (8, 0, 128)


def test_refusals(ops, gpu):
    w = workloads.make_paged_workload("bad", [(30, 4)], 8, 4, seed=1)
    q, m = w.gemm_call(device=gpu)
    wd, q = w.to(gpu), q.to(gpu)
    call = lambda q=q, window=5, sinks=0, positions=m.positions: ops.paged_attention_gemm_window(
        q, wd.k_pool, wd.v_pool, m.cu_seqlens, m.max_q_len, m.block_tables, m.kv_lens, positions, window, sinks)
    for kw, message in (({"window": 0}, "window must be"), ({"sinks": -1}, "sinks must be"),
                        ({"q": q.float()}, "share a dtype"), ({"positions": m.positions.long()}, "int32"),
                        ({"positions": m.positions[:2]}, "positions.numel"), ({"q": q[:7]}, "multiple of n_kv_heads")):
        with pytest.raises(RuntimeError, match=message):
            call(**kw)
    with pytest.raises(TypeError):
        call(window=2.5)
