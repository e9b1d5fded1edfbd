"""paged_attention_gemv_shared_prefix against the 64-bit oracle; bounds as for the plain decode call (the prefix's
weights round to the storage type, as the prefill kernel's do, and the output once)."""

import numpy as np
import pytest
import torch

import oracle.added as added
from femtovllm import workloads
from helpers import assert_close, np32, np64, np_tables

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def batch(prefix, tails, heads, kv_heads, dim=128, dtype=BF16, seed=0):
    """A workload whose sequences share ``prefix`` (whole pages) keys and have ``tails`` keys of their own; a negative
    tail ends inside the prefix.  The shared columns of the tables are then spoilt: nothing may read them."""
    lens = [max(1, prefix + t) for t in tails]
    w = workloads.make_paged_workload("shared", [(L - 1, 1) for L in lens], heads, kv_heads, head_dim=dim, dtype=dtype, seed=seed,
                                      shared_seqs=range(len(lens)), shared_blocks=prefix // 16)
    full = max(w.raw_block_tables, key=len)[: prefix // 16]
    if max(lens) < prefix:  # no sequence holds the whole prefix
        used = {x for t in w.raw_block_tables for x in t}
        full = full + [x for x in range(w.k_pool.size(0)) if x not in used][: prefix // 16 - len(full)]
    for x in full:  # rows past every context: read for the longer ones only
        for pool in (w.k_pool, w.v_pool):
            pool[x] = torch.nan_to_num(pool[x], nan=0.25)
    for i, t in enumerate(w.raw_block_tables):
        t[: prefix // 16] = [(-1, 10**6, 0)[i % 3]] * min(len(t), prefix // 16)
    return w, torch.tensor(full, dtype=torch.int32)


def run(ops, gpu, w, prefix_pages, max_kv_len=None, empty=(), call=None):
    q, meta = w.gemv_call(device=gpu)
    wd, kv_lens = w.to(gpu), meta.kv_lens.clone()
    for b in empty:
        kv_lens[b] = 0
        meta.block_tables[b] = -1
    args = (q.to(gpu), wd.k_pool, wd.v_pool, prefix_pages.to(gpu), meta.block_tables, kv_lens,
            meta.max_kv_len if max_kv_len is None else max_kv_len)
    out = ops.paged_attention_gemv_shared_prefix(*args)
    want = added.shared_prefix_decode(np64(q), np32(w.k_pool), np32(w.v_pool), prefix_pages.tolist(), np_tables(meta),
                                      kv_lens.tolist())
    return out, want, args


@pytest.mark.parametrize("prefix", [0, 16, 48, 64, 80, 400, 1024])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prefixes_and_tails(ops, gpu, dtype, prefix):
    """Tails of none, one and many keys, contexts that end inside the prefix."""
    tails = [0, 1, 5, 16, 17, 200, 700, -1, -15, -16, -17, -prefix // 2, -prefix + 1]
    w, pages = batch(prefix, tails, 8, 4, dtype=dtype, seed=prefix)
    out, want, _ = run(ops, gpu, w, pages)
    assert_close(out, want, dtype, f"prefix {prefix}")


@pytest.mark.parametrize("heads", [(4, 4), (16, 8), (32, 8), (64, 8), (6, 1), (12, 4)])
@pytest.mark.parametrize("dim", [128, 80, 16])
def test_heads_and_dims(ops, gpu, heads, dim):
    w, pages = batch(208, [3, 40, 0, 1, 90], *heads, dim=dim, seed=sum(heads) + dim)
    out, want, _ = run(ops, gpu, w, pages)
    assert_close(out, want, BF16, f"{heads} dim {dim}")


@pytest.mark.parametrize("seqs", [1, 31, 32, 33, 65, 130, 300])
def test_batches(ops, gpu, seqs):
    """Row tiles that end inside a wave, more sequences than lanes; empty slots give zeros."""
    rng = np.random.default_rng(seqs)
    w, pages = batch(320, [int(x) for x in rng.integers(0, 60, size=seqs)], 4, 2, seed=seqs)
    empty = [] if seqs == 1 else [0, seqs // 2, seqs - 1]
    out, want, _ = run(ops, gpu, w, pages, empty=empty)
    assert (out[:, empty] == 0).all()
    assert_close(out, want, BF16, f"{seqs} sequences")


@pytest.mark.parametrize("heads", [(17, 1), (48, 2), (40, 1)])
def test_more_query_heads_than_a_wave_holds(ops, gpu, heads):
    w, pages = batch(336, [100, 0, 45, -20], *heads, seed=sum(heads))
    out, want, _ = run(ops, gpu, w, pages)
    assert_close(out, want, BF16, f"heads {heads}")


def test_bad_blocks_read_as_zeros(ops, gpu):
    """Blocks that are -1 or past the pool, in the prefix and in the tails; a table that ends inside a tail."""
    w, pages = batch(336, [100, 3, 45, 64], 8, 4, seed=9)
    pages[2], pages[20], pages[7] = -1, 10**6, -(2**31)
    w.raw_block_tables[0][22], w.raw_block_tables[0][26], w.raw_block_tables[2][21] = -1, 2**31 - 1, -5
    out, want, args = run(ops, gpu, w, pages)
    assert_close(out, want, BF16, "bad blocks")
    narrow = args[4][:, :24].contiguous()
    out = ops.paged_attention_gemv_shared_prefix(*args[:4], narrow, *args[5:])
    want = added.shared_prefix_decode(np64(args[0]), np32(w.k_pool), np32(w.v_pool), pages.tolist(), narrow.cpu().numpy(),
                                      args[5].tolist())
    assert_close(out, want, BF16, "narrow table")


def test_no_key_past_the_prefix(ops, gpu):
    """Every context ends inside the prefix, and the largest one is understated to the call."""
    w, pages = batch(640, [-1, -100, -320, -639, -64, -63], 8, 4, seed=2)
    out, want, _ = run(ops, gpu, w, pages)
    assert_close(out, want, BF16, "no tails")
    w, pages = batch(320, [900, 3, 1500], 8, 4, seed=3)
    out, want, _ = run(ops, gpu, w, pages, max_kv_len=10)
    assert_close(out, want, BF16, "understated max_kv_len")


def test_long_prefix(ops, gpu):
    w, pages = batch(16 * 700, [100, 20, 3000, 0], 8, 4, seed=4)
    out, want, _ = run(ops, gpu, w, pages)
    assert_close(out, want, BF16, "11200 keys")


def test_agrees_with_the_plain_call_and_growing_scores(ops, gpu):
    """Sharp scores, whose maxima move from piece to piece, and the largest key in the tail or in the prefix."""
    w, pages = batch(512, [40, 1, 130], 8, 4, dtype=F16, seed=5)
    ramp = torch.linspace(0.2, 6.0, pages.numel())
    for i, x in enumerate(pages.tolist()):
        w.k_pool[x] *= ramp[i]
    out, want, _ = run(ops, gpu, w, pages)
    assert_close(out, want, F16, "sharp scores")


def test_one_dominant_key_is_exact(ops, gpu):
    """A key of far the largest score returns its V row, for keys of the prefix and of the tails."""
    w, pages = batch(64, [20] * 84, 4, 2, seed=6)
    w.k_pool[:] = 0
    w.q.zero_()
    w.q[:, :, 0] = 2000.0
    out = None
    tables = [pages.tolist() + t[4:] for t in w.raw_block_tables]
    # key b of sequence b; a shared block's key dominates for every sequence, so the prefix is checked one key a call
    for b in range(64, 84):
        w.k_pool[tables[b][b // 16], :, b % 16, 0] = 1.0
    out, _, _ = run(ops, gpu, w, pages)
    for b in range(64, 84):
        for h in range(4):
            assert torch.equal(out[h, b].cpu(), w.v_pool[tables[b][b // 16], h // 2, b % 16])
    for j in (0, 15, 16, 33, 63):
        w.k_pool[:] = 0
        w.k_pool[tables[0][j // 16], :, j % 16, 0] = 1.0
        out, _, _ = run(ops, gpu, w, pages)
        for h in range(4):
            assert torch.equal(out[h].cpu(), w.v_pool[tables[0][j // 16], h // 2, j % 16].expand(84, -1))


def test_pools_past_4_gib(ops, gpu):
    """The same blocks in a compact pool and at the end of one of 4.3 GiB: equal bits."""
    w, pages = batch(512, [100, 3, 900], 16, 8, seed=31)
    for pool in (w.k_pool, w.v_pool):
        pool.nan_to_num_(nan=0.5)
    blocks, n, outs = 140_000, w.k_pool.size(0), []
    q, meta = w.gemv_call(device=gpu)
    for base in (0, blocks - n):
        pools = []
        for pool in (w.k_pool, w.v_pool):
            big = torch.empty((base + n,) + tuple(pool.shape[1:]), dtype=BF16, device=gpu)
            big[base:] = pool.to(gpu)
            pools.append(big)
        tables = torch.where(meta.block_tables >= 0, meta.block_tables + base, meta.block_tables)
        outs.append(ops.paged_attention_gemv_shared_prefix(q.to(gpu), *pools, (pages + base).to(gpu), tables, meta.kv_lens,
                                                           meta.max_kv_len))
        torch.cuda.synchronize()
        del pools
    assert torch.equal(*outs)


def test_captured_calls_and_other_streams(ops, gpu):
    """Two graphs and an eager call on one stream's workspace, replayed on two streams at once: bit-equal results."""
    graphs = []
    for i, (prefix, tails) in enumerate(((512, [100, 3, 900]), (64, [700] * 9))):
        w, pages = batch(prefix, tails, 8, 4, seed=20 + i)
        _, _, args = run(ops, gpu, w, pages)
        f = lambda args=args: ops.paged_attention_gemv_shared_prefix(*args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out, f, args[0]))
    other = torch.cuda.Stream()
    for turn in range(3):
        for *_, q in graphs:
            q.copy_(torch.randn_like(q))
        want = [f() for _, _, f, _ in graphs]
        for _, out, _, _ in graphs:
            out.fill_(9)
        torch.cuda.synchronize()
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
            third = graphs[0][2]()
        again = graphs[1][2]()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], want[0]) and torch.equal(graphs[1][1], want[1]), turn
        assert torch.equal(third, want[0]) and torch.equal(again, want[1])


def test_refusals(ops, gpu):
    w, pages = batch(32, [4, 5], 4, 2, seed=1)
    _, _, args = run(ops, gpu, w, pages)
    swap = lambda i, x: args[:i] + (x,) + args[i + 1 :]
    for bad, message in ((swap(0, args[0].float()), "share a dtype"), (swap(3, args[3].long()), "must be int32"),
                         (swap(3, args[3][None]), "1-D"), (swap(3, pages), "must be on"), (swap(5, args[5][:1]), "kv_lens"),
                         (swap(6, 1 << 40), "out of range"), (swap(6, -1), "negative")):
        with pytest.raises(RuntimeError, match=message):
            ops.paged_attention_gemv_shared_prefix(*bad)
    f32 = tuple(t.float() if torch.is_tensor(t) and t.is_floating_point() else t for t in args)
    with pytest.raises(RuntimeError, match="not implemented for 'Float'"):
        ops.paged_attention_gemv_shared_prefix(*f32)
    empty = ops.paged_attention_gemv_shared_prefix(args[0][:, :0], args[1], args[2], args[3], args[4][:0], args[5][:0], 0)
    assert empty.shape == (4, 0, 128)
