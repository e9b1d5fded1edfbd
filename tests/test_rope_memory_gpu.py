"""rope_cache_write with an ``out`` that lies beside q, k and v in their buffer, or on them; with a max_q_len far above
the sequences' lengths."""

import pytest
import torch

from femtovllm.rope import scaled_rope_tables
from test_rope_gpu import BF16, check_rotated, run, step

pytestmark = pytest.mark.gpu


def test_out_beside_q_in_its_buffer(ops, gpu):
    """out, q, k and v are columns of one array: out gets the rotated q, the others stay."""
    w, _, _, _ = step([(3, 20), (0, 7)], 4, 2, 64, BF16, seed=1)
    x = torch.randn(27, 12, 64, device=gpu).to(BF16)
    out, q, k, v = x.split([4, 4, 2, 2], dim=1)
    before = x.cpu().clone()
    tables = scaled_rope_tables(64, 64)
    got, _, meta = run(ops, gpu, w, q, k, v, tables, False, out=out)
    assert got.data_ptr() == out.data_ptr()
    check_rotated(got, before[:, 4:8], *(t.numpy() for t in tables), meta.positions.cpu().numpy(), False, "out")
    assert torch.equal(x[:, 4:].cpu(), before[:, 4:])


def test_heads_of_q_k_and_v_in_turn_in_place(ops, gpu):
    w, _, _, _ = step([(3, 20), (0, 7)], 4, 4, 64, BF16, seed=2)
    x = torch.randn(27, 4, 3, 64, device=gpu).to(BF16)
    q, k, v = x.unbind(2)
    before = x.cpu().clone()
    tables = scaled_rope_tables(64, 32)
    got, _, meta = run(ops, gpu, w, q, k, v, tables, True, out=q)
    check_rotated(got, before[:, :, 0], *(t.numpy() for t in tables), meta.positions.cpu().numpy(), True, "in place")
    assert torch.equal(x[:, :, 1:].cpu(), before[:, :, 1:])


def test_out_on_k_or_v_is_refused(ops, gpu):
    """Also where out is q itself: k and v must not change before they are read."""
    w, q, k, v = step([(0, 8)], 4, 2, 64, BF16, seed=8)
    q, k, v = q.to(gpu), k.to(gpu), v.to(gpu)
    tables = scaled_rope_tables(64, 32)
    long = torch.zeros(9, 4, 64, dtype=BF16, device=gpu)
    for args, name in (((q, q[:, :2], v), "k"), ((q, k, q[:, 2:]), "v"), ((long[:8], long[1:, :2], v), "k")):
        with pytest.raises(RuntimeError, match=f"out must share no memory with {name}"):
            run(ops, gpu, w, *args, tables, False, out=args[0])
    with pytest.raises(RuntimeError, match="out must share no memory with v"):
        run(ops, gpu, w, q, k, long[:8, 2:], tables, False, out=long[:8])


def test_out_whose_rows_meet_is_refused(ops, gpu):
    w, q, k, v = step([(0, 8)], 4, 2, 64, BF16, seed=9)
    q, k, v = q.to(gpu), k.to(gpu), v.to(gpu)
    tables = scaled_rope_tables(64, 32)
    row = torch.zeros(1, 4, 64, dtype=BF16, device=gpu).expand(8, -1, -1)
    for args in ((q, k, v, row), (row, k, v, row)):
        with pytest.raises(RuntimeError, match="rows of out share memory"):
            run(ops, gpu, w, *args[:3], tables, False, out=args[3])
    got, _, meta = run(ops, gpu, w, row, k, v, tables, False)  # as an input they may
    check_rotated(got, row, *(t.numpy() for t in tables), meta.positions.cpu().numpy(), False, "one row for all tokens")


def test_heads_ahead_of_tokens(ops, gpu):
    """out and q as (heads, tokens, dim) arrays seen token by token."""
    w, q, k, v = step([(0, 8), (17, 3)], 4, 2, 64, BF16, seed=10)
    tables = scaled_rope_tables(64, 64)
    qd = q.transpose(0, 1).contiguous().to(gpu).transpose(0, 1)
    out = torch.empty(4, 11, 64, dtype=BF16, device=gpu).transpose(0, 1)
    got, _, meta = run(ops, gpu, w, qd, k.to(gpu), v.to(gpu), tables, True, out=out)
    check_rotated(got, q, *(t.numpy() for t in tables), meta.positions.cpu().numpy(), True, "out")
    run(ops, gpu, w, qd, k.to(gpu), v.to(gpu), tables, True, out=qd)
    assert torch.equal(qd, got)


@pytest.mark.parametrize("bound", [100, 1 << 24, 2**31 - 1])
def test_overstated_max_q_len(ops, gpu, bound):
    w, q, k, v = step([(0, 37), (15, 1), (100, 60)], 6, 2, 64, BF16, seed=11)
    q, k, v = q.to(gpu), k.to(gpu), v.to(gpu)
    tables = scaled_rope_tables(300, 64)
    want, pools, _ = run(ops, gpu, w, q, k, v, tables, False)
    got, wd, _ = run(ops, gpu, w, q, k, v, tables, False, max_q_len=bound)
    assert torch.equal(got, want) and torch.equal(wd.k_pool, pools.k_pool) and torch.equal(wd.v_pool, pools.v_pool)
