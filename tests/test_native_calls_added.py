"""csrc/native_calls.cpp, the window, shared-prefix and rotary calls, without a GPU: as test_native_calls.py.

Those calls also ask for the current device and whether their stream is being captured: stand-ins here, set by the tests.
"""

import ctypes
import importlib.machinery
import importlib.util
import os
import subprocess

import pytest
import torch

from test_native_calls import HARNESS, PKG

STUBS = r"""
#include <hip/hip_runtime_api.h>
extern "C" { int current_device = -1; int capturing = 0; int capture_error = 0; }
static hipError_t stub_device(int* d) { *d = current_device; return hipSuccess; }
static hipError_t stub_capture(hipStream_t, hipStreamCaptureStatus* s) {
    if (capture_error) return hipErrorInvalidValue;
    *s = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
    return hipSuccess;
}
#define hipGetDevice stub_device
#define hipStreamIsCapturing stub_capture
#include "native_calls.cpp"
"""

FUNCTIONS = ("femto_paged_attention_gemv_window", "femto_paged_attention_gemm_window",
             "femto_paged_attention_gemv_shared_prefix", "femto_rope_cache_write")
REQUIRED = ("femto_paged_attention_gemv", "femto_paged_attention_gemm", "femto_qk_norm_rope_cache_write",
            "femto_flash_attention")


@pytest.fixture(scope="module")
def native(tmp_path_factory):
    """(module, counts, rc, sizes, globals of the stand-ins)"""
    spec = importlib.util.spec_from_file_location("femto_build", os.path.join(PKG, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    d = tmp_path_factory.mktemp("native")
    src, lib = d / "harness.cpp", d / "femto_native.so"
    src.write_text(HARNESS.replace('#include "native_calls.cpp"\n', STUBS))
    cmd = [str(src) if a.endswith("native_calls.cpp") else "-O0" if a == "-O2" else a for a in build.native_command(str(lib))]
    subprocess.run(cmd + [f"-I{PKG}/csrc"], check=True, capture_output=True, text=True)
    loader = importlib.machinery.ExtensionFileLoader("femto_native", str(lib))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("femto_native", loader))
    loader.exec_module(module)
    counts, rc, size, keep = {}, [0], [512], {}

    def entry(name, restype, result):
        def call():
            counts[name] = counts.get(name, 0) + 1
            return result()

        keep[name] = ctypes.CFUNCTYPE(restype)(call)

    message = ctypes.create_string_buffer(b"stand-in refused")
    entry("femto_attn_last_error", ctypes.c_void_p, lambda: ctypes.addressof(message))
    for name in FUNCTIONS + REQUIRED:
        entry(name, ctypes.c_int, lambda: rc[0])
    for name in REQUIRED[:2] + FUNCTIONS[:3]:
        entry(name + "_workspace_size", ctypes.c_size_t, lambda: size[0])
    addresses = {n: ctypes.cast(f, ctypes.c_void_p).value for n, f in keep.items()}
    so = ctypes.CDLL(str(lib))
    flags = {n: ctypes.c_int.in_dll(so, n) for n in ("current_device", "capturing", "capture_error", "fail_wrap")}
    module.bind({n: a for n, a in addresses.items() if n.removesuffix("_workspace_size") not in FUNCTIONS})
    unbound = [call() for _, call in calls(module).values()]
    module.bind(addresses)
    module.keep = keep, message
    return module, counts, rc, size, flags, unbound


def calls(module):
    """entry point -> (library function, call); each call brings a workspace of 4096 bytes"""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    b16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    pool, tab = b16(4, 2, 16, 128), torch.zeros(64, 64)
    spaces = lambda: {(-1, 0): torch.zeros(4096, dtype=torch.uint8)}
    return {
        "gemv_window": (FUNCTIONS[0], lambda q=b16(4, 3, 128), w=5, s=0: module.gemv_window(
            q, pool, pool, i32(3, 2), i32(3), 20, w, s, spaces())),
        "gemm_window": (FUNCTIONS[1], lambda q=b16(4, 5, 128), w=5, s=0: module.gemm_window(
            q, pool, pool, i32(2), 5, i32(1, 2), i32(1), i32(5), w, s, spaces())),
        "gemv_shared": (FUNCTIONS[2], lambda q=b16(4, 3, 128): module.gemv_shared(
            q, pool, pool, i32(1), i32(3, 2), i32(3), 20, spaces())),
        "rope": (FUNCTIONS[3], lambda q=b16(3, 4, 128): module.rope(
            q, b16(3, 2, 128), b16(3, 2, 128), tab, tab, i32(3), pool, pool, i32(3, 2), None, 1, False, None)),
    }


NAMES = ["gemv_window", "gemm_window", "gemv_shared", "rope"]


def test_unbound_functions_decline(native):
    assert native[5] == [None] * 4


@pytest.mark.parametrize("name", NAMES)
def test_call_returns_the_output(native, name):
    module, counts = native[:2]
    fn, call = calls(module)[name]
    before = counts.get(fn, 0)
    out = call()
    assert isinstance(out, torch.Tensor) and out.dtype == torch.bfloat16 and counts[fn] == before + 1


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("how", [1, 2], ids=["throws", "python_error"])
def test_none_means_nothing_was_launched(native, name, how):
    module, counts, *_ = native
    fn, call = calls(module)[name]
    before, flag = counts.get(fn, 0), native[4]["fail_wrap"]
    flag.value = how
    try:
        assert call() is None
    finally:
        flag.value = 0
    assert counts.get(fn, 0) == before


@pytest.mark.parametrize("name", NAMES)
def test_library_errors_raise(native, name):
    module, counts, rc = native[:3]
    fn, call = calls(module)[name]
    before, rc[0] = counts.get(fn, 0), 1
    try:
        with pytest.raises(RuntimeError, match="stand-in refused"):
            call()
    finally:
        rc[0] = 0
    assert counts[fn] == before + 1


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("flag,value", [("current_device", 0), ("capturing", 1), ("capture_error", 1)])
def test_other_devices_and_captured_streams_are_left_to_the_python_path(native, name, flag, value):
    """A rotary call needs no workspace, so capturing does not concern it."""
    module, counts, *_ = native
    fn, call = calls(module)[name]
    var, before = native[4][flag], counts.get(fn, 0)
    old, var.value = var.value, value
    try:
        out = call()
    finally:
        var.value = old
    declined = name != "rope" or flag == "current_device"
    assert (out is None) == declined and counts.get(fn, 0) == before + (not declined)


@pytest.mark.parametrize("name", NAMES)
def test_declined_forms(native, name):
    module, counts, *_ = native
    fn, call = calls(module)[name]
    before = counts.get(fn, 0)

    class Sub(torch.Tensor):
        pass

    q = torch.zeros((3, 4, 128) if name == "rope" else (4, 5 if name == "gemm_window" else 3, 128), dtype=torch.bfloat16)
    for bad in (q.double(), q[0], q.as_subclass(Sub), None, [1.0], q.half(), q[..., ::2], q.transpose(1, 2)):
        assert call(bad) is None
    if name.endswith("window"):
        for kw in ({"w": 0}, {"w": -1}, {"s": -1}, {"w": 2.5}, {"w": True}, {"s": None}):
            assert call(**kw) is None, kw
    assert counts.get(fn, 0) == before


@pytest.mark.parametrize("name", NAMES[:3])
def test_a_workspace_too_small_is_left_to_the_python_path(native, name):
    module, counts, _, size, *_ = native
    fn, call = calls(module)[name]
    before, size[0] = counts.get(fn, 0), 5000
    try:
        assert call() is None
    finally:
        size[0] = 512
    assert counts.get(fn, 0) == before


@pytest.mark.parametrize("name", NAMES[:2])
def test_counts_past_int32_are_the_largest_int32(native, name):
    fn, call = calls(native[0])[name]
    assert call(w=1 << 60, s=1 << 40) is not None
