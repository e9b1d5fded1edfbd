"""The window attention's refusals and its oracle, without a GPU."""

import ctypes

import numpy as np
import pytest
import torch

import oracle.added as added
import oracle.attention as plain


@pytest.fixture(scope="module")
def C():
    from femtovllm import _C

    return _C


def _gemv(C, **kw):
    a = dict(dtype=2, q=16, qsh=128, qsb=2048, out=16, osh=128, osb=2048, k=16, v=16, nb=8, kvh=8, bs=16, d=128,
             ps0=16384, ps1=2048, ps2=128, tables=16, npages=4, ts=4, kv_lens=16, nseq=4, h=16, maxkv=9000, window=5000,
             sinks=4, ws=None, wsb=0, stream=None)
    a.update(kw)
    return C._lib.femto_paged_attention_gemv_window(*a.values())


def _gemm(C, **kw):
    a = dict(dtype=2, q=16, qsh=128, qst=128, out=16, osh=128, ost=128, k=16, v=16, nb=8, kvh=8, bs=16, d=128,
             ps0=16384, ps1=2048, ps2=128, cu=16, nseq=2, ntok=10, maxq=5, h=16, tables=16, npages=4, ts=4,
             kv_lens=16, pos=16, window=5, sinks=0, ws=256, wsb=64, stream=None)
    a.update(kw)
    return C._lib.femto_paged_attention_gemm_window(*a.values())


def test_library_refusals(C):
    """Each is refused before anything touches the (fake) pointers."""
    last = lambda: C._lib.femto_attn_last_error().decode()
    for call, name in ((_gemv, "paged_attention_gemv_window"), (_gemm, "paged_attention_gemm_window")):
        assert call(C, window=0) == 1 and "window must be at least 1" in last() and name in last()
        assert call(C, window=-3) == 1
        assert call(C, sinks=-1) == 1 and "sinks must be >= 0" in last()
        assert call(C, d=136) == 2 and name in last()
        assert call(C, h=12) == 1 and call(C, nb=0) == 1 and call(C, q=8) == 1 and call(C, ps2=100) == 1
        assert call(C, kv_lens=None) == 1
        assert call(C, nseq=0) == 0
    assert _gemm(C, dtype=0) == 2 and "not implemented for 'Float'" in last()
    assert _gemv(C, ps2=1 << 25) == 1 and "row stride" in last()
    assert _gemv(C) != 0  # no workspace (or, without a GPU, no device to plan for)


def test_workspace_sizes_of_refused_calls(C):
    size = C._lib.femto_paged_attention_gemv_window_workspace_size
    assert size(2, 0, 16, 8, 9000, 5, 0) == 0 and size(2, 4, 16, 8, 9000, 0, 0) == 0 and size(2, 4, 12, 8, 9000, 5, 0) == 0
    size = C._lib.femto_paged_attention_gemm_window_workspace_size
    assert size(2, 9, 5, 16, 8, 40, 0, 0) == 0 and size(0, 9, 5, 16, 8, 40, 5, 0) == 0


def test_ops_refuse_cpu_tensors():
    from femtovllm import ops

    q, pool, t = torch.zeros(16, 2, 128), torch.zeros(4, 8, 16, 128), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.paged_attention_gemv_window(q, pool, pool, t, t[:, 0], 16, 4)
    with pytest.raises(ValueError):
        ops.paged_attention_gemm_window(q, pool, pool, t[:, 0], 1, t, t[:, 0], t[:, 0], 4)


def test_a_capture_gets_its_own_workspace(monkeypatch, C):
    """Eager calls share the stream's; a captured call takes new memory with its first bytes cleared."""
    monkeypatch.setattr(C, "_stream", lambda device: 0)
    cpu, cache = torch.device("cpu"), {}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    a = C._call_workspace(cache, cpu, 1000, 64)
    assert C._call_workspace(cache, cpu, 900, 64)[0] == a[0] and a[0] % 256 == 0 and a[1] >= 1000
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    ptr, size, hold = C._call_workspace(cache, cpu, 1000, 64)
    assert ptr != a[0] and ptr % 256 == 0 and size >= 1000 and hold.data_ptr() <= ptr
    assert not any(ctypes.string_at(ptr, 64))
    assert len(cache) == 1 and C._call_workspace(cache, cpu, 0, 64) == (None, 0, None)


def test_oracle_window_rule():
    """Against the causal oracle where the window is whole, a direct reading of the rule, and a planted mistake."""
    rng = np.random.default_rng(0)
    q, pool = rng.standard_normal((4, 9, 16)), rng.standard_normal((6, 2, 16, 16))
    tables, kv, pos, cu = [[0, 2, 4], [5, 1, -1]], [40, 20], np.array([36, 37, 38, 39, 15, 16, 17, 18, 19]), [0, 4, 9]
    want = plain.paged_prefill(q, pool, pool, cu, tables, kv, pos)
    got = added.window_prefill(q, pool, pool, cu, tables, kv, pos, 100, 0)
    assert np.allclose(got, want, rtol=0, atol=1e-13)
    seen = added.window_seen([7], 12, 3, 2)[0]
    assert [j for j in range(12) if seen[j]] == [0, 1, 5, 6, 7]
    assert not np.allclose(added.window_prefill(q, pool, pool, cu, tables, kv, pos, 6, 2),
                           added.window_prefill(q, pool, pool, cu, tables, kv, pos, 7, 2))
    one = added.window_decode(q[:, :2], pool, pool, tables, kv, 1, 0)  # a window of one key: its V row
    assert np.array_equal(one[3, 0], pool[4, 1, 7]) and np.array_equal(one[0, 1], pool[1, 0, 3])


def test_oracle_prefix():
    rng = np.random.default_rng(1)
    q, pool = rng.standard_normal((4, 3, 16)), rng.standard_normal((9, 2, 16, 16))
    tables, kv = [[0, 2, 4], [0, 2, 5], [0, 2, 6]], [40, 48, 33]
    want = plain.paged_decode(q, pool, pool, tables, kv)
    hidden = [[-1, 99, 4], [7, -1, 5], [-1, -1, 6]]
    assert np.allclose(added.shared_prefix_decode(q, pool, pool, [0, 2], hidden, kv), want, rtol=0, atol=1e-13)
