"""rope_cache_write against the 64-bit oracle, its placement against kv_cache_write's rule.

Bound of a rotated element y = a c - b s (|c|, |s| <= 1): two roundings in fp32, of the product and of the sum,
2^-24 (|b| + |y|), then half a step of the output type relative to y (an fp16 below 2^-14: 2^-25).  Everything
else is copied: equal.
"""

import numpy as np
import pytest
import torch

import oracle.added as added
import oracle.attention as oa
from femtovllm import workloads
from femtovllm.rope import scaled_rope_tables
from helpers import np64

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0**-8, F16: 2.0**-11, F32: 2.0**-24}


def check_rotated(got, x, cos, sin, pos, interleaved, what):
    dtype = got.dtype
    got, x64 = np64(got), np64(x)
    want = added.rotate(x64, cos, sin, pos, interleaved)
    half = cos.shape[1]
    assert np.array_equal(got[..., 2 * half :], x64[..., 2 * half :]), f"{what}: dims past the rotated ones changed"
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN pattern"
    mag = np.abs(x64)
    pair = mag.copy()
    if interleaved:
        pair[..., 0 : 2 * half : 2] += mag[..., 1 : 2 * half : 2]
        pair[..., 1 : 2 * half : 2] += mag[..., 0 : 2 * half : 2]
    else:
        pair[..., :half] += mag[..., half : 2 * half]
        pair[..., half : 2 * half] += mag[..., :half]
    tol = HALF_STEP[dtype] * np.abs(want) + 2.0**-23 * pair + (2.0**-25 if dtype == F16 else 0.0)
    ok = ~np.isnan(want)
    assert (np.abs(got - want)[ok] <= tol[ok]).all(), f"{what}: {np.abs(got - want)[ok].max()}"


def step(chunks, heads, kv_heads, dim, dtype, seed=0):
    """(q, k, v of the new tokens; pools, metadata) of a paged batch, without poison."""
    w = workloads.make_paged_workload("rope", chunks, heads, kv_heads, head_dim=dim, dtype=dtype, seed=seed, poison=False)
    gen = torch.Generator().manual_seed(seed + 1)
    t = w.num_tokens
    draw = lambda h: torch.randn((t, h, dim), generator=gen).to(dtype)
    return w, draw(heads), draw(kv_heads), draw(kv_heads)


def run(ops, gpu, w, q, k, v, tables, interleaved, decode=False, out=None, **change):
    _, meta = w.gemm_call(device=gpu)
    wd = w.to(gpu)
    cos, sin = (t.to(gpu) for t in tables)
    args = dict(positions=meta.positions, kv_page_tables=meta.block_tables, max_q_len=meta.max_q_len)
    args.update(change)
    got = ops.rope_cache_write(q, k, v, cos, sin, args["positions"], wd.k_pool, wd.v_pool, args["kv_page_tables"],
                               cu_seqlens=None if decode else meta.cu_seqlens, max_q_len=args["max_q_len"],
                               interleaved=interleaved, out=out)
    return got, wd, meta


CHUNKS = [(0, 37), (15, 1), (100, 130), (0, 1), (31, 18)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (128, 2), (128, 24), (64, 64), (64, 32), (64, 50), (80, 80),
                                        (80, 40), (96, 72), (16, 16), (8, 6), (8, 8), (112, 112), (120, 118)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_layouts(ops, gpu, dtype, dim, rotary, interleaved):
    w, q, k, v = step(CHUNKS, 6, 2, dim, dtype, seed=dim + rotary)
    tables = scaled_rope_tables(300, rotary, base=1000.0)
    got, wd, meta = run(ops, gpu, w, q.to(gpu), k.to(gpu), v.to(gpu), tables, interleaved)
    cos, sin = (t.numpy() for t in tables)
    pos = meta.positions.cpu().numpy()
    check_rotated(got, q, cos, sin, pos, interleaved, "q")
    # The pools: what the plain write of the same rows leaves, the written k rows within the bound.
    marks = torch.arange(k.size(0)).to(torch.float64)[:, None, None].expand(k.shape).numpy() + 1
    where, _ = oa.cache_write(np.zeros(w.k_pool.shape), np.zeros(w.k_pool.shape), marks, marks, meta.block_tables.cpu().numpy(),
                              meta.raw_cu_seqlens, pos)
    token = where[:, :, :, 0].astype(int)  # 0: not written
    new_k, new_v = wd.k_pool.cpu(), wd.v_pool.cpu()
    keep = torch.from_numpy(token == 0)
    assert torch.equal(new_k[keep], w.k_pool[keep]) and torch.equal(new_v[keep], w.v_pool[keep])
    blk, head, row = np.nonzero(token)
    rows_k = new_k[blk, head, row]
    src_k = k[token[blk, head, row] - 1, head]
    assert torch.equal(new_v[blk, head, row], v[token[blk, head, row] - 1, head])
    assert blk.size == k.size(0) * 2
    check_rotated(rows_k[:, None], src_k[:, None], cos, sin, pos[token[blk, head, row] - 1], interleaved, "k")


@pytest.mark.parametrize("heads", [(64, 8), (1, 1), (16, 16), (5, 5)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_decode_tokens_heads_and_in_place(ops, gpu, heads, interleaved):
    """One token per sequence (no cu_seqlens), q rotated in place from a wider projection, k and v strided."""
    H, KVH = heads
    w, _, _, _ = step([(L - 1, 1) for L in (1, 16, 17, 90)], H, KVH, 64, BF16, seed=H)
    fused = torch.randn(4, (H + 2 * KVH) * 64, device=gpu).to(BF16)
    q = fused[:, : H * 64].view(4, H, 64)
    k = fused[:, H * 64 : (H + KVH) * 64].view(4, KVH, 64)
    v = fused[:, (H + KVH) * 64 :].view(4, KVH, 64)
    before = [t.cpu().clone() for t in (q, k, v)]
    tables = scaled_rope_tables(100, 32)
    got, wd, meta = run(ops, gpu, w, q, k, v, tables, interleaved, decode=True, out=q)
    assert got.data_ptr() == q.data_ptr()
    pos = meta.positions.cpu().numpy()
    check_rotated(got, before[0], *(t.numpy() for t in tables), pos, interleaved, "q in place")
    assert torch.equal(k.cpu(), before[1]) and torch.equal(v.cpu(), before[2])
    for b in range(4):
        blk, row = w.raw_block_tables[b][pos[b] // 16], pos[b] % 16
        check_rotated(wd.k_pool[blk, :, row][None], before[1][b : b + 1], *(t.numpy() for t in tables), pos[b : b + 1],
                      interleaved, "k")
        assert torch.equal(wd.v_pool[blk, :, row].cpu(), before[2][b])


def test_in_place_with_unaligned_halves(ops, gpu):
    """Partners that are read from memory one by one (R / 2 = 25), in place."""
    w, q, k, v = step(CHUNKS, 9, 3, 64, F16, seed=3)
    tables = scaled_rope_tables(300, 50)
    qd = q.to(gpu)
    got, _, meta = run(ops, gpu, w, qd, k.to(gpu), v.to(gpu), tables, False, out=qd)
    check_rotated(got, q, *(t.numpy() for t in tables), meta.positions.cpu().numpy(), False, "q")


def test_positions_outside_the_tables_and_blocks_outside_the_pool(ops, gpu):
    """NaN in the rotated dims; the cache write stops at the first bad table column, and an understated max_q_len
    covers every token."""
    w, q, k, v = step([(0, 70), (40, 1)], 4, 2, 64, BF16, seed=4)
    _, meta = w.gemm_call(device=gpu)
    bad = meta.block_tables.clone()
    bad[0, 2] = 10**6
    bad[1, 2] = -1
    pos = meta.positions.clone()
    pos[5] = 500
    pos[6] = -3
    tables = scaled_rope_tables(100, 32)
    got, wd, _ = run(ops, gpu, w, q.to(gpu), k.to(gpu), v.to(gpu), tables, True, positions=pos, kv_page_tables=bad, max_q_len=3)
    check_rotated(got, q, *(t.numpy() for t in tables), pos.cpu().numpy(), True, "q")
    assert torch.isnan(got[5:7, :, :32]).all() and not torch.isnan(got[:, :, 32:]).any()
    for c in range(5):
        blk = w.raw_block_tables[0][c]
        n = min(16, 70 - 16 * c)
        same = torch.equal(wd.v_pool[blk, :, :n].cpu(), v[16 * c : 16 * c + n].transpose(0, 1))
        assert same == (c < 2)
        if c >= 2:
            assert torch.equal(wd.v_pool[blk].cpu(), w.v_pool[blk])
    assert torch.equal(wd.k_pool[w.raw_block_tables[1][2]].cpu(), w.k_pool[w.raw_block_tables[1][2]])


def test_rows_behind_the_last_sequence_stay(ops, gpu):
    """A padded batch: tokens past cu_seqlens[-1] are neither rotated nor written."""
    w, q, k, v = step([(3, 20)], 4, 2, 64, BF16, seed=6)
    pad = lambda t: torch.cat((t, torch.full((5, *t.shape[1:]), float("nan"), dtype=t.dtype)))
    _, meta = w.gemm_call(device=gpu)
    wd = w.to(gpu)
    tables = [t.to(gpu) for t in scaled_rope_tables(64, 64)]
    pos = torch.cat((meta.positions, torch.full((5,), 7, dtype=torch.int32, device=gpu)))
    out = torch.full((25, 4, 64), 3.0, dtype=BF16, device=gpu)
    ops.rope_cache_write(pad(q).to(gpu), pad(k).to(gpu), pad(v).to(gpu), *tables, pos, wd.k_pool, wd.v_pool,
                         meta.block_tables, cu_seqlens=meta.cu_seqlens, max_q_len=20, out=out)
    assert (out[20:] == 3.0).all() and not torch.isnan(out).any()
    assert not torch.isnan(wd.k_pool).any()


def test_pools_past_4_gib(ops, gpu):
    """The same blocks in a compact pool and at the end of one of 4.3 GiB: equal rows written."""
    w, q, k, v = step(CHUNKS, 16, 8, 128, BF16, seed=31)
    blocks, n, written = 140_000, w.k_pool.size(0), []
    tables = [t.to(gpu) for t in scaled_rope_tables(300, 128, base=1000.0)]
    _, meta = w.gemm_call(device=gpu)
    for base in (0, blocks - n):
        pools = [torch.zeros((base + n, 8, 16, 128), dtype=BF16, device=gpu) for _ in range(2)]
        cols = torch.where(meta.block_tables >= 0, meta.block_tables + base, meta.block_tables)
        out = ops.rope_cache_write(q.to(gpu), k.to(gpu), v.to(gpu), *tables, meta.positions, *pools, cols,
                                   cu_seqlens=meta.cu_seqlens, max_q_len=meta.max_q_len)
        torch.cuda.synchronize()
        assert not any(pool[:base].any() for pool in pools)
        written.append([out] + [pool[base:].clone() for pool in pools])
        del pools
    for a, b in zip(*written):
        assert torch.equal(a, b)


def test_captured_and_replayed(ops, gpu):
    w, q, k, v = step(CHUNKS, 8, 4, 128, BF16, seed=7)
    _, meta = w.gemm_call(device=gpu)
    wd = w.to(gpu)
    tables = [t.to(gpu) for t in scaled_rope_tables(300, 128)]
    qd, kd, vd = q.to(gpu), k.to(gpu), v.to(gpu)
    call = lambda: ops.rope_cache_write(qd, kd, vd, *tables, meta.positions, wd.k_pool, wd.v_pool, meta.block_tables,
                                        cu_seqlens=meta.cu_seqlens, max_q_len=meta.max_q_len)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for _ in range(3):
        for t in (qd, kd, vd):
            t.copy_(torch.randn_like(t))
        want, pools = call(), (wd.k_pool.clone(), wd.v_pool.clone())
        out.zero_()
        wd.k_pool.fill_(1)
        wd.v_pool.fill_(1)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for pool, ref in zip((wd.k_pool, wd.v_pool), pools):
            for (p, n), table in zip(w.chunks, w.raw_block_tables):
                for j in range(p, p + n):
                    assert torch.equal(pool[table[j // 16], :, j % 16], ref[table[j // 16], :, j % 16])


def test_refusals(ops, gpu):
    w, q, k, v = step([(0, 8)], 4, 2, 64, BF16, seed=8)
    q, k, v = q.to(gpu), k.to(gpu), v.to(gpu)
    tables = scaled_rope_tables(64, 32)
    both = torch.zeros(9, 4, 64, dtype=BF16, device=gpu)
    for kw, message in ((dict(out=both[:8, :2]), "out must match"), (dict(max_q_len=0), "max_q_len must be")):
        with pytest.raises(RuntimeError, match=message):
            run(ops, gpu, w, q, k, v, tables, False, **kw)
    both[:8] = q
    with pytest.raises(RuntimeError, match="share no memory with q"):
        run(ops, gpu, w, both[:8], k, v, tables, False, out=both[1:])
    with pytest.raises(RuntimeError, match="float32"):
        run(ops, gpu, w, q, k, v, [t.half() for t in tables], False)
    with pytest.raises(RuntimeError, match="rotary_dim must be"):
        run(ops, gpu, w, q, k, v, scaled_rope_tables(64, 66), False)
    with pytest.raises(RuntimeError, match="share a dtype"):
        run(ops, gpu, w, q, k.half(), v, tables, False)
