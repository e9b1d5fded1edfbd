"""Static check of the window and shared-prefix kernels' gfx950 code (CPU only: hipcc -S), as test_isa_prefill.py.

Their direct-to-LDS copies come from inline asm: a tile's eight and a decode page's four (K, then V) each form one run
of s_nop 4, then per copy an m0 write, s_nop 0 and the copy; no vmcnt wait stands between copies of a block, and no
kernel spills to scratch memory (a spill's load would be waited for in the middle of them).
"""

import importlib.util
import os
import re
import subprocess

import pytest

from test_isa_prefill import PKG, _blocks


@pytest.mark.parametrize("source,kernels,run_lengths", [("window_prefill.hip", 24, {4, 8}), ("window_decode.hip", 8, {4}),
                                                        ("shared_prefix.hip", 12, {4, 8})])
def test_copies(tmp_path, source, kernels, run_lengths):
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
    found = set()
    for s, line in enumerate(lines):
        name = re.match(r"^(_ZN5femto\d+\w+_kernelI\w+):", line)
        if not name:
            continue
        name = name.group(1)
        end = next(j for j in range(s, len(lines)) if lines[j].startswith(".Lfunc_end"))
        blocks = [b for _, b in _blocks(lines[s:end])]
        total = sum(t.startswith("global_load_lds_dwordx4") for b in blocks for t in b)
        if total == 0:
            continue
        found.add(name)
        assert scratch[name] == "0", name
        in_runs = 0
        for ins in blocks:
            copies = [k for k, t in enumerate(ins) if t.startswith("global_load_lds_dwordx4")]
            if copies:
                waits = [t for t in ins[copies[0]:copies[-1]] if t.startswith("s_waitcnt") and "vmcnt" in t]
                assert not waits, (name, waits)
            k = 0
            while k < len(ins):
                run, j = 0, k + 1
                while ins[k].startswith("s_nop 4") and j + 2 < len(ins) and re.match(r"s_(mov_b32|add_u32) m0,", ins[j]) \
                        and ins[j + 1].startswith("s_nop 0") and ins[j + 2].startswith("global_load_lds_dwordx4"):
                    run += 1
                    j += 3
                assert run == 0 or run in run_lengths, (name, run)
                in_runs += run
                k = max(j, k + 1) if run else k + 1
        assert in_runs == total, (name, in_runs, total)
    assert len(found) == kernels, sorted(found)
