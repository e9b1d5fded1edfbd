"""Reads of the 4-bit cache: tokens that belong to no sequence give zeros, whatever the memory of the outputs held before."""

import numpy as np
import pytest
import torch

import oracle.fp4 as of
from helpers import np64

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def dirty(gpu, shape, dtype):
    """The allocator's next blocks of these outputs hold NaN."""
    hold = [torch.full(shape, float("nan"), dtype=dtype, device=gpu) for _ in range(4)]
    torch.cuda.synchronize()
    del hold


@pytest.fixture(params=["native", "python"])
def route(request, monkeypatch):
    from femtovllm import _C

    if request.param == "python":
        monkeypatch.setattr(_C, "_native", type("NotHere", (), {"__getattr__": lambda self, name: lambda *a: None})())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("before,n,after", [(3, [4, 0, 17], 5), (0, [1], 70), (130, [2, 1], 0), (9, [0, 0], 1)])
def test_tokens_before_and_behind(ops, gpu, route, before, n, after, dtype):
    rng = np.random.default_rng(before)
    cu = before + np.concatenate([[0], np.cumsum(n)])
    T, dim = int(cu[-1]) + after, 48
    pos = np.concatenate([np.zeros(before), *(np.arange(m) for m in n), np.zeros(after)])
    tables = rng.permutation(2 * len(n)).reshape(len(n), 2)
    pool = rng.integers(0, 120, size=(2 * len(n), 3, of.page_bytes(dim))).astype(np.uint8)
    pool[..., 1024:] = rng.integers(120, 130, size=pool[..., 1024:].shape)
    t = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=gpu)
    dirty(gpu, (T, 3, dim), dtype)
    got = ops.kv_cache_read_fp4(torch.tensor(pool, device=gpu), dim, dtype, t(pos), t(tables), t(cu), 17)
    for x, y in zip(got, of.read(pool, pos.astype(int), tables, cu, dim)):
        assert np.array_equal(np64(x), y)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_sequences(ops, gpu, route, dtype):
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)
    pool = torch.full((2, 3, of.page_bytes(64)), 120, dtype=torch.uint8, device=gpu)
    dirty(gpu, (6, 3, 64), dtype)
    for x in ops.kv_cache_read_fp4(pool, 64, dtype, i32(6), i32(0, 2), i32(1), 1):
        assert x.shape == (6, 3, 64) and not x.any()
