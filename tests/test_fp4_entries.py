"""Refusals of the 4-bit cache's attention entries; nothing is launched and nothing behind the (fake) pointers is touched."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def C():
    from femtovllm import _C

    return _C


def _gemv(C, **kw):
    a = dict(dtype=2, q=16, qh=128, qs=1024, out=16, oh=128, os=1024, pool=16, nb=8, kvh=2, d=128, tab=16, npages=4, ts=4, lens=16,
             nseq=3, h=8, maxkv=64, ws=None, wsb=0, stream=None)
    a.update(kw)
    return C._lib.femto_paged_attention_gemv_fp4(*a.values())


def _gemm(C, **kw):
    a = dict(dtype=2, q=16, qh=128, qs=1024, out=16, oh=128, os=1024, pool=16, nb=8, kvh=2, d=128, cu=16, nseq=3, ntok=9, maxq=5,
             h=8, tab=16, npages=4, ts=4, lens=16, pos=16, ws=None, wsb=0, stream=None)
    a.update(kw)
    return C._lib.femto_paged_attention_gemm_fp4(*a.values())


@pytest.mark.parametrize("call", [_gemv, _gemm])
def test_refusals(C, call):
    last = lambda: C._lib.femto_attn_last_error().decode()
    for dtype in (0, 5, -1):
        assert call(C, dtype=dtype) == 2 and "not implemented" in last()
    for d in (0, 8, 100, 136, 144, -16):
        assert call(C, d=d) == 2 and "head_dim" in last()
    for h, kvh in ((0, 2), (8, 0), (7, 2), (-8, 2), (8, -2), (2, 4)):
        assert call(C, h=h, kvh=kvh) == 1 and "multiple of n_kv_heads" in last()
    assert call(C, nb=0) == 1 and call(C, npages=-1) == 1 and call(C, ts=-1) == 1
    for name in ("q", "out", "pool", "tab"):
        assert call(C, **{name: None}) == 1 and "null" in last()
    assert call(C, lens=None) == 1 and "null" in last()
    for name, at in (("q", 8), ("pool", 8), ("out", 4)):
        assert call(C, **{name: at}) == 1 and "aligned" in last()
    assert call(C, qh=4) == 1 and "q strides" in last() and call(C, qs=1025) == 1
    assert call(C, nseq=-1) == 1 and "negative" in last()
    assert call(C, nseq=0) == 0


def test_refusals_of_one(C):
    last = lambda: C._lib.femto_attn_last_error().decode()
    assert _gemv(C, maxkv=-1) == 1 and "negative" in last()
    assert _gemm(C, ntok=-1) == 1 and _gemm(C, maxq=-1) == 1 and "negative" in last() and _gemm(C, ntok=0) == 0
    assert _gemm(C, cu=None) == 1 and _gemm(C, pos=None) == 1 and "null" in last()
    assert _gemm(C, oh=2) == 1 and "out strides" in last() and _gemm(C, os=1022) == 1


def test_ops_refuse_cpu_tensors(C):
    from femtovllm import fp4, ops

    q, i = torch.zeros(8, 3, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    pool, cu = fp4.new_pool(8, 2, 128, "cpu"), torch.arange(4, dtype=torch.int32)
    with pytest.raises((ValueError, RuntimeError)):
        ops.paged_attention_gemv_fp4(q, pool, i[:, None], i, 16)
    with pytest.raises((ValueError, RuntimeError)):
        ops.paged_attention_gemm_fp4(q, pool, cu, 1, i[:, None], i, i)


def test_no_sequences_need_no_workspace(C):
    size = C._lib.femto_paged_attention_gemv_fp4_workspace_size
    assert size.restype is ctypes.c_size_t and size(0, 8, 2, 64) == 0 and size(3, 8, 0, 64) == 0
