"""The rotary tables and rope_cache_write's refusals, without a GPU."""

import math

import numpy as np
import pytest
import torch

import oracle.added as added
import oracle.prologue as prologue
from femtovllm.rope import rope_tables, scaled_rope_tables


@pytest.fixture(scope="module")
def C():
    from femtovllm import _C

    return _C


def _rope(C, **kw):
    a = dict(dtype=2, q=16, qst=512, qsh=128, k=16, kst=256, ksh=128, v=16, vst=256, vsh=128, out=16, ost=512, osh=128,
             cos=16, sin=16, rs=64, rows=100, r=128, il=0, kp=16, vp=16, nb=8, h=4, kvh=2, bs=16, d=128, ps0=4096, ps1=2048,
             ps2=128, cu=16, nseq=2, ntok=10, maxq=5, pos=16, tab=16, npages=4, ts=4, stream=None)
    a.update(kw)
    return C._lib.femto_rope_cache_write(*a.values())


def test_library_refusals(C):
    """Each is refused before anything touches the (fake) pointers."""
    last = lambda: C._lib.femto_attn_last_error().decode()
    assert _rope(C, dtype=5) == 2 and "dtype" in last()
    for d in (0, 100, 136):
        assert _rope(C, d=d, r=2) == 2 and "head_dim" in last()
    for r in (0, 1, 63, 130, -2):
        assert _rope(C, r=r) == 1 and "rotary_dim must be even" in last()
    assert _rope(C, nseq=-1) == 1 and _rope(C, maxq=0) == 1 and "max_q_len" in last()
    assert _rope(C, cu=None) == 1 and "one token" in last()
    assert _rope(C, nseq=70000) == 1 and _rope(C, bs=32) == 1 and _rope(C, kvh=0) == 1 and _rope(C, nb=0) == 1
    assert _rope(C, q=None) == 1 and "null" in last()
    assert _rope(C, rs=32) == 1 and "tables too small" in last()
    assert _rope(C, rows=0) == 1 and _rope(C, ts=3) == 1
    assert _rope(C, k=8) == 1 and "aligned" in last()
    assert _rope(C, cos=18) == 1 and _rope(C, qsh=100) == 1 and "strides" in last()
    assert _rope(C, ntok=0) == 0


def test_ops_refuse_cpu_tensors():
    from femtovllm import ops

    x, t, i = torch.zeros(2, 4, 64), torch.zeros(8, 32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.rope_cache_write(x, x, x, t, t, i, torch.zeros(2, 4, 16, 64), torch.zeros(2, 4, 16, 64), i[:, None])


def test_overlaps(C):
    x = torch.zeros(10, 4)
    assert C._overlaps(x[:5], x[4:]) and not C._overlaps(x[:5], x[5:]) and not C._overlaps(x[:0], x)
    assert C._overlaps(x[:, :2], x[:, 2:])  # by their spans
    assert not C._overlaps(x, torch.zeros(10, 4))


def test_oracle_rotation():
    """Against the half-layout oracle; the interleaved layout is the half one with the dims dealt out; a planted
    mistake (the other sign) shows."""
    rng = np.random.default_rng(0)
    x, pos = rng.standard_normal((5, 3, 16)), np.array([0, 3, 9, 1, 7])
    cos, sin = (t.numpy() for t in rope_tables(10, 16))
    want = prologue.rope(x, cos, sin, pos)
    assert np.allclose(added.rotate(x, cos[:, :8], sin[:, :8], pos, False), want, rtol=0, atol=1e-14)
    order = [i // 2 + 8 * (i % 2) for i in range(16)]
    dealt = added.rotate(x[..., order], cos[:, :8], sin[:, :8], pos, True)
    assert np.allclose(dealt, want[..., order], rtol=0, atol=1e-14)
    assert not np.allclose(added.rotate(x, cos[:, :8], -sin[:, :8], pos, False), want)
    assert np.isnan(added.rotate(x, cos[:5, :4], sin[:5, :4], pos, False)[2, :, :8]).all()


def test_tables_without_scaling():
    cos, sin = scaled_rope_tables(4000, 128, base=1000000.0)
    old_cos, old_sin = rope_tables(4000, 128)
    assert cos.shape == (4000, 64) and cos.dtype == torch.float32
    # rope_tables forms its angles in float32: off by up to (frequency's 2^-24 twice, product 2^-24) * angle
    tol = 4.0 * 2.0**-24 * torch.arange(4000.0)[:, None] + 2.0**-22
    assert ((cos - old_cos[:, :64]).abs() <= tol).all() and ((sin - old_sin[:, :64]).abs() <= tol).all()
    far = scaled_rope_tables(100001, 2)  # one radian a token
    assert abs(float(far[0][100000, 0]) - math.cos(100000.0)) <= 2.0**-24


def test_scalings():
    """Each against its formula for single pairs, written out."""
    R, base, L, f = 64, 10000.0, 2048, 4.0
    w = [base ** (-2.0 * i / R) for i in range(R // 2)]
    # position 1: the angle is the frequency itself
    freq = lambda **kw: torch.atan2(*reversed([t.double()[1] for t in scaled_rope_tables(2, R, base=base, **kw)])).tolist()
    close = lambda a, b: abs(a - b) <= 2.0**-22
    assert all(close(a, b) for a, b in zip(freq(), w))
    assert all(close(a, b / f) for a, b in zip(freq(scaling="linear", factor=f), w))
    ntk = freq(scaling="ntk", factor=f)
    assert close(ntk[0], w[0]) and close(ntk[-1], w[-1] / f)
    wl = freq(scaling="wavelength", factor=f, original_max_seqlen=L, low_freq_factor=1.0, high_freq_factor=4.0)
    for a, b in zip(wl, w):
        lam = 2 * math.pi / b
        mix = (L / lam - 1.0) / 3.0
        assert close(a, b if lam <= L / 4 else b / f if lam >= L else (1 - mix) * b / f + mix * b)
    y = scaled_rope_tables(2, R, base=base, scaling="yarn", factor=f, original_max_seqlen=L)
    m = 0.1 * math.log(f) + 1
    assert torch.allclose(torch.hypot(*(t.double()[1] for t in y)), torch.tensor(m, dtype=torch.float64), rtol=0, atol=2.0**-22)
    yarn = freq(scaling="yarn", factor=f, original_max_seqlen=L, attention_factor=1.0)
    for a, b in zip(yarn, w):
        turns = L * b / (2 * math.pi)
        assert b / f - 2.0**-22 <= a <= b + 2.0**-22
        if turns > 45:
            assert close(a, b)
        if turns < 0.7:
            assert close(a, b / f)


@pytest.mark.parametrize("kw", [dict(rotary_dim=7), dict(rotary_dim=0), dict(scaling="cubic"), dict(scaling="linear", factor=0.5),
                                dict(scaling="yarn", factor=2.0), dict(scaling="wavelength", factor=2.0),
                                dict(scaling="wavelength", factor=2.0, original_max_seqlen=9, low_freq_factor=4.0)])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        scaled_rope_tables(4, **{"rotary_dim": 8, **kw})
