"""Prefill over the 4-bit cache where a key's V is NaN that some tokens of a query tile see and others do not.

The oracle takes a row's own keys only.  Chunks of any length, so that keys fall in a tile's first and last columns; one and
more query heads per KV head (tiles of 128, 64 and 32 tokens); dims below 128; keys cut over workgroups; beside decode rows.
"""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from fp4_helpers import Batch
from helpers import assert_close, np64

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def nan_value(w, seq, key, head, block):
    n = of.blocks(w.dim)
    w.pool[w.tables[seq, key // 16], head, 512 * n + 64 + 16 * (key % 16 // 4) + 4 * block + key % 4] = 255


def check(ops, gpu, w, what):
    pool, tables, lens, cu, pos, q = w.on(gpu)
    call = lambda: ops.paged_attention_gemm_fp4(q, pool, cu, max(n for _, n in w.chunks), tables, lens, pos)
    out = call()
    want = of.prefill(np64(w.q), w.pool, w.cu, w.tables, w.kv_lens, w.pos)
    assert np.isnan(want).any() and np.isfinite(want).any()
    assert_close(out, want, w.dtype, what)
    for _ in range(3):
        again = call()
        assert torch.equal(torch.isnan(again), torch.isnan(out)) and torch.equal(again.nan_to_num(), out.nan_to_num())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("dim", [16, 48, 64, 112, 128])
@pytest.mark.parametrize("heads", [(4, 4), (4, 2), (8, 2), (6, 2)])
def test_nan_values_inside_a_tile(ops, gpu, heads, dim, dtype):
    w = Batch([(0, 150), (70, 90), (33, 1), (200, 64), (0, 1), (5, 2)], *heads, dim, dtype, dim + sum(heads))
    n = of.blocks(dim)
    for seq, key in ((0, 0), (0, 31), (0, 32), (0, 63), (0, 64), (0, 149), (1, 69), (1, 70), (1, 159), (2, 33), (3, 230), (3, 263),
                     (5, 6)):
        nan_value(w, seq, key, key % heads[1], (key // 16) % n)
    check(ops, gpu, w, f"{heads} {dim} {dtype}")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("key", [0, 3000, 5990, 6000, 6031, 6063])
def test_nan_values_of_a_split_tile(ops, gpu, key, dtype):
    """A long context's query tile in pieces: the key is in one of them, seen by all, by some or by the last token."""
    w = Batch([(6000, 64), (100, 20)], 8, 2, 128, dtype, key)
    nan_value(w, 0, key, 1, 3)
    check(ops, gpu, w, f"key {key} {dtype}")


def test_positions_in_no_order(ops, gpu):
    """Tokens of a tile see the key or not in no order."""
    w = Batch([(100, 90), (20, 100)], 8, 2, 128, BF16, 4)
    rng = np.random.default_rng(5)
    for c in (slice(0, 90), slice(90, 190)):
        w.pos[c] = rng.permutation(w.pos[c])
    for key in (101, 128, 150, 189):
        nan_value(w, 0, key, 0, key % 4)
        nan_value(w, 1, key - 95, 1, key % 4)
    check(ops, gpu, w, "permuted")


def test_every_key_of_a_prompt(ops, gpu):
    """A NaN at each key in turn, and at all of them."""
    for key in list(range(0, 130, 3)) + [128, 129]:
        w = Batch([(0, 130)], 2, 1, 64, F16, 6)
        nan_value(w, 0, key, 0, key % 2)
        check(ops, gpu, w, f"key {key}")
    w = Batch([(0, 130)], 2, 1, 64, F16, 6)
    for key in range(1, 130):
        nan_value(w, 0, key, 0, 1)
    check(ops, gpu, w, "all but the first")
