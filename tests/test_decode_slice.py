"""The split decode workers' slices (csrc/decode_slice.h), built for the CPU."""

import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nano-vllm-practice_amd", "csrc")


@pytest.fixture(scope="module")
def slice_pages(tmp_path_factory):
    d = tmp_path_factory.mktemp("slice")
    (d / "slice.cpp").write_text(
        '#include "decode_slice.h"\n'
        'extern "C" int slice(int wi, int C, int total, int* out) { return femto::slice_pages(wi, C, total, out[0], out[1]); }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=undefined",
                    "-static-libubsan", "-shared", "-fPIC", f"-I{CSRC}", str(d / "slice.cpp"), "-o", str(d / "slice.so")], check=True)
    lib = ctypes.CDLL(str(d / "slice.so"))
    out = (ctypes.c_int * 2)()
    return lambda wi, C, total: (out[0], out[1]) if lib.slice(wi, C, total, out) else None


@pytest.mark.parametrize("C,total", [(1, 1), (4, 4), (4, 5), (66, 67_000), (7, 0), (4194304, 60), (4194304, 9_000_000),
                                     (1 << 30, 5), (2**31 - 1, 2**31 - 1), (2**30, 2**31 - 1)])
@pytest.mark.parametrize("waves", [1, 2, 128, 1024])
def test_slices_cover_the_pages_once(slice_pages, C, total, waves):
    """Up to C * waves pages: consecutive, no longer than C, nothing before 0 or past the end, whatever C is."""
    want = 0
    for wi in range(waves):
        got = slice_pages(wi, C, total)
        if wi * C >= total:
            assert got is None, (wi, got)
            continue
        assert got == (wi * C, min(total, (wi + 1) * C))
        assert got[0] == want
        want = got[1]
    assert want == min(total, C * waves)
