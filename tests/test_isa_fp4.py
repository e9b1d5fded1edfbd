"""Static check of the 4-bit cache kernels' gfx950 code (CPU only: hipcc -S), as test_isa_added.py and test_isa_mfma_waits.py.

No kernel spills to scratch memory or loads by flat addresses (their waits would count LDS traffic too); the copies to LDS
carry their wait states, a tile's K being one of them; no MFMA's result is read too early, the scaled instructions'
included.
"""

import importlib.util
import os
import re
import subprocess

import pytest

import test_isa_mfma_waits as waits
from test_isa_prefill import PKG


@pytest.mark.parametrize("source,kernels", [("fp4_cache.hip", 16), ("fp4_decode.hip", 12), ("fp4_prefill.hip", 24)])
def test_code(tmp_path, monkeypatch, source, kernels):
    # Passes of the scaled instructions with operands of at most 6 bits.
    monkeypatch.setattr(waits, "PASSES", {"16x16x128": 4, "32x32x64": 8, **waits.PASSES})
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
    asm = out.read_text()
    lines = asm.split("\n")
    scratch = dict(re.findall(r"\.set (_ZN5femto\w+)\.private_seg_size, (\S+)", asm))
    found = 0
    for s, line in enumerate(lines):
        name = re.match(r"^(_ZN5femto\d+\w+_kernelI\w+):", line)
        if not name:
            continue
        name = name.group(1)
        body = [x.strip() for x in lines[s + 1:next(j for j in range(s, len(lines)) if lines[j].startswith(".Lfunc_end"))]]
        found += 1
        assert scratch[name] == "0", name
        assert not [x for x in body if x.startswith("flat_")], name
        for k, x in enumerate(body):
            if x.startswith("global_load_lds_dwordx4"):
                before = [y for y in body[max(0, k - 12):k] if y and not y.startswith((";", "."))][-3:]
                assert before[0].startswith("s_nop 4") and re.match(r"s_(mov_b32|add_u32) m0,", before[1]) \
                    and before[2].startswith("s_nop 0"), (name, before)
        if source != "fp4_cache.hip":
            assert [x for x in body if x.startswith("v_mfma_scale_f32")], name
        assert waits.early_reads(body) == [], name
    assert found == kernels
