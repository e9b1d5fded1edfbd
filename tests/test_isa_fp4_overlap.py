"""Static check of the 4-bit cache kernels' gfx950 code (CPU only: hipcc -S): no conversion of 32 values between fp32 and 6 bits
writes over a register of its own sources, which the instruction still reads while it writes."""

import importlib.util
import os
import re
import subprocess

import pytest

from test_isa_prefill import PKG


def registers(text):
    """(first, last) of every vector register operand."""
    return [(int(a), int(b or a)) for a, b in re.findall(r"\bv\[?(\d+)(?::(\d+)\])?", text)]


def overlaps(line):
    (a, b), *sources = registers(line.split(None, 1)[1])
    return any(c <= b and d >= a for c, d in sources)


def test_the_check():
    assert overlaps("v_cvt_scalef32_2xpk16_fp6_f32 v[4:9], v[2:17], v[34:49], v19")
    assert overlaps("v_cvt_scalef32_2xpk16_fp6_f32 v[2:7], v[50:65], v[2:17], v19")
    assert overlaps("v_cvt_scalef32_pk32_f32_fp6 v[2:33], v[28:33], v75") and overlaps("v_cvt_scalef32_pk32_f32_fp6 v[2:33], v[40:45], v5")
    assert not overlaps("v_cvt_scalef32_2xpk16_fp6_f32 v[146:151], v[50:65], v[34:49], v75")
    assert not overlaps("v_cvt_scalef32_pk32_f32_fp6 v[2:33], v[146:151], s4")


@pytest.mark.parametrize("source,kernels", [("fp4_decode.hip", 12), ("fp4_prefill.hip", 24)])
def test_conversions_leave_their_sources(tmp_path, source, kernels):
    spec = importlib.util.spec_from_file_location("femto_build", os.path.join(PKG, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    try:
        hipcc = build.hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    out = tmp_path / "kernels.s"
    flags = [f for f in build.HIPCC_FLAGS if f not in ("-shared", "-fPIC")]
    cmd = [hipcc, *flags, "--cuda-device-only", "-S", "-I", build.INCLUDE, "-I", build.CSRC, os.path.join(build.CSRC, source),
           "-o", str(out)]
    res = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
    assert res.returncode == 0, res.stderr[-2000:]
    bodies = re.split(r"^(_ZN5femto\d+\w+_kernelI\w+):", out.read_text(), flags=re.M)
    assert len(bodies[1::2]) == kernels
    for name, body in zip(bodies[1::2], bodies[2::2]):
        found = re.findall(r"^\s+(v_cvt_scalef32_(?:2xpk16_fp6_f32|pk32_f32_fp6) .*)$", body, flags=re.M)
        assert found, name
        assert not [x for x in found if overlaps(x)], name
