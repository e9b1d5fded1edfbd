"""Contexts that end inside the shared prefix, in batches of many query rows: few and uneven pieces of the prefix,
the case in which a context's number of pieces follows from the piece's size and not from the number of pieces."""

import numpy as np
import pytest
import torch

from helpers import assert_close
from test_shared_prefix_gpu import BF16, F16, batch, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs,heads,prefix,dtype", [
    (192, (32, 8), 1792, BF16),  # 28 key tiles in 4 pieces
    (256, (16, 8), 1024, F16),   # 16 in 4
    (256, (32, 8), 2048, BF16),  # 32 in 4
    (56, (64, 8), 4096, BF16),   # 64 in 8
])
def test_ends_inside_the_prefix(ops, gpu, seqs, heads, prefix, dtype):
    """Contexts of one key up to the whole prefix and past it, ends at, before and behind every 64-key border."""
    rng = np.random.default_rng(seqs + prefix)
    ends = [1, prefix - 1, prefix, prefix + 1] + [64 * i + d for i in range(1, prefix // 64) for d in (-1, 0, 1, 33)]
    ends = [int(x) for x in rng.permutation(ends)][: seqs - 8]
    ends += [prefix + int(x) for x in rng.integers(0, 40, size=seqs - len(ends))]
    w, pages = batch(prefix, [e - prefix for e in ends], *heads, dtype=dtype, seed=seqs)
    out, want, _ = run(ops, gpu, w, pages)
    assert_close(out, want, dtype, f"{seqs} sequences on {prefix}")


@pytest.mark.parametrize("seed", range(6))
def test_random_ends(ops, gpu, seed):
    rng = np.random.default_rng(seed)
    heads = [(32, 8), (16, 8), (16, 16), (8, 1), (64, 8), (12, 4)][seed]
    seqs, prefix = int(rng.integers(100, 260)), 16 * int(rng.integers(40, 200))
    tails = [int(x) for x in rng.integers(-prefix + 1, 100, size=seqs)]
    w, pages = batch(prefix, tails, *heads, dim=64, seed=seed)
    empty = [int(x) for x in rng.integers(0, seqs, size=3)]
    out, want, _ = run(ops, gpu, w, pages, empty=empty)
    assert (out[:, empty] == 0).all()
    assert_close(out, want, BF16, f"{seqs} sequences of {heads} on {prefix}")
