"""Every head_dim of the windowed and shared-prefix calls, with pages enough for several per wave, in few sequences (eight
waves or parts per row) and in many (four waves)."""

import numpy as np
import pytest
import torch

from helpers import assert_close
from test_shared_prefix_gpu import batch
from test_shared_prefix_gpu import run as run_shared
from test_window_gpu import BF16, F16, F32, free_hidden_blocks, run_decode, run_prefill
from femtovllm import workloads

pytestmark = pytest.mark.gpu


def lens(seqs, seed):
    return [int(x) for x in np.random.default_rng(seed).integers(100, 400, size=seqs)]


@pytest.mark.parametrize("dim", range(8, 129, 8))
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_window_decode(ops, gpu, dtype, dim):
    for seqs in (3, 40):
        w = workloads.make_paged_workload("dims", [(L - 1, 1) for L in lens(seqs, dim)], 8, 4, head_dim=dim, dtype=dtype, seed=dim)
        out, want = run_decode(ops, free_hidden_blocks(w, 300, 5), gpu, 300, 5)
        assert_close(out, want, dtype, f"{seqs} sequences, dim {dim}")


@pytest.mark.parametrize("dim", range(4, 129, 12))
def test_window_decode_f32(ops, gpu, dim):
    w = workloads.make_paged_workload("dims", [(L - 1, 1) for L in lens(40, dim)], 8, 4, head_dim=dim, dtype=F32, seed=dim)
    out, want = run_decode(ops, free_hidden_blocks(w, 300, 5), gpu, 300, 5)
    assert_close(out, want, F32, f"dim {dim}")


@pytest.mark.parametrize("dim", range(16, 129, 16))
@pytest.mark.parametrize("heads", [(4, 4), (8, 4), (8, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_window_prefill_with_rows(ops, gpu, dtype, heads, dim):
    chunks = [(250, 70)] + [(L - 1, 1) for L in lens(12, dim)]
    w = workloads.make_paged_workload("dims", chunks, *heads, head_dim=dim, dtype=dtype, seed=dim)
    out, want = run_prefill(ops, free_hidden_blocks(w, 300, 5), gpu, 300, 5)
    assert_close(out, want, dtype, f"{heads}, dim {dim}")


@pytest.mark.parametrize("dim", range(16, 129, 16))
@pytest.mark.parametrize("heads", [(4, 4), (8, 4), (8, 2)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_shared_prefix(ops, gpu, dtype, heads, dim):
    w, pages = batch(304, [L - 150 for L in lens(40, dim)], *heads, dim=dim, dtype=dtype, seed=dim)
    out, want, _ = run_shared(ops, gpu, w, pages)
    assert_close(out, want, dtype, f"{heads}, dim {dim}")
