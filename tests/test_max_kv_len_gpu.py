"""Decode calls whose max_kv_len is far above the contexts: an upper bound that only plans the call."""

import pytest
import torch

import femtovllm
import oracle.added as added
from femtovllm import workloads
from helpers import assert_close, np32, np64, np_tables
from test_shared_prefix_gpu import batch, run

pytestmark = pytest.mark.gpu

LENS = [1, 40, 700, 333, 2000]
BOUNDS = [2**30, 2**31 - 17, 2**31 - 1]


@pytest.mark.parametrize("bound", BOUNDS)
def test_shared_prefix(ops, gpu, bound):
    w, pages = batch(112, [9, 105, 138, -49, 179, 67], 8, 1, dim=112, seed=6)
    out, want, _ = run(ops, gpu, w, pages, max_kv_len=bound)
    assert_close(out, want, torch.bfloat16, f"bound {bound}")


@pytest.mark.parametrize("bound", BOUNDS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [(8, 1), (16, 8)])
def test_window_and_plain_decode(ops, gpu, monkeypatch, dtype, heads, bound):
    w = workloads.make_paged_workload("bound", [(L - 1, 1) for L in LENS], *heads, dtype=dtype, seed=3)
    q, meta = w.gemv_call(device=gpu)
    wd = w.to(gpu)
    args = (q.to(gpu), wd.k_pool, wd.v_pool, meta.block_tables, meta.kv_lens, bound)
    for window, sinks in ((2**31 - 1, 0), (2**31 - 1, 2**31 - 1), (100, 3)):
        out = ops.paged_attention_gemv_window(*args, window, sinks)
        want = added.window_decode(np64(q), np32(w.k_pool), np32(w.v_pool), np_tables(meta), LENS, window, sinks)
        assert_close(out, want, dtype, f"window {window}, bound {bound}")
    monkeypatch.setattr(femtovllm._DEV, "split_kv_decode", True)
    want = added.window_decode(np64(q), np32(w.k_pool), np32(w.v_pool), np_tables(meta), LENS, 1 << 40, 0)
    assert_close(ops.paged_attention_gemv(*args), want, dtype, f"plain, bound {bound}")
