"""The shared-prefix decode call's refusals, without a GPU."""

import pytest
import torch


def _shared(C, **kw):
    a = dict(dtype=2, q=16, qsh=128, qsb=2048, out=16, osh=128, osb=2048, k=16, v=16, nb=8, kvh=8, bs=16, d=128,
             ps0=16384, ps1=2048, ps2=128, pre=16, pages=4, tables=16, npages=4, ts=4, kv_lens=16, nseq=4, h=16, maxkv=90,
             ws=None, wsb=0, stream=None)
    a.update(kw)
    return C._lib.femto_paged_attention_gemv_shared_prefix(*a.values())


def test_library_refusals():
    """Each is refused before anything touches the (fake) pointers."""
    from femtovllm import _C as C

    last = lambda: C._lib.femto_attn_last_error().decode()
    assert _shared(C, dtype=0) == 2 and "not implemented for 'Float'" in last()
    assert _shared(C, d=72, ps2=72) == 2 and "multiple of 16" in last()
    assert _shared(C, d=144) == 2
    assert _shared(C, pages=-1) == 1 and "prefix_pages" in last()
    assert _shared(C, pages=1 << 27) == 1
    assert _shared(C, pre=None) == 1 and "null" in last()
    assert _shared(C, kv_lens=None) == 1 and _shared(C, nseq=-1) == 1 and _shared(C, nseq=70000) == 1
    assert _shared(C, h=12) == 1 and _shared(C, bs=8) == 1 and _shared(C, nb=0) == 1 and _shared(C, q=8) == 1
    assert _shared(C, ps2=1 << 25) == 1 and "stride" in last()
    assert _shared(C, nseq=0) == 0
    assert _shared(C) != 0  # no workspace (or, here, no device to plan for)


def test_ops_refuse_cpu_tensors():
    from femtovllm import ops

    q, pool, t = torch.zeros(16, 2, 128), torch.zeros(4, 8, 16, 128), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_attention_gemv_shared_prefix(q, pool, pool, t[:, 0], t, t[:, 0], 16)
