"""csrc/native_calls.cpp, the calls over a 4-bit cache, without a GPU: as test_native_calls_added.py."""

import ctypes
import importlib.machinery
import importlib.util
import os
import subprocess

import pytest
import torch

from test_native_calls import HARNESS, PKG
from test_native_calls_added import REQUIRED, STUBS

FUNCTIONS = ("femto_kv_cache_write_fp4", "femto_kv_cache_read_fp4", "femto_rope_cache_write_fp4",
             "femto_paged_attention_gemv_fp4", "femto_paged_attention_gemm_fp4")
NAMES = ["write_fp4", "read_fp4", "rope_fp4", "gemv_fp4", "gemm_fp4"]


@pytest.fixture(scope="module")
def native(tmp_path_factory):
    """(module, counts, rc, sizes, globals of the stand-ins, what the unbound calls gave)"""
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
    for name in REQUIRED[:2] + FUNCTIONS[3:]:
        entry(name + "_workspace_size", ctypes.c_size_t, lambda: size[0])
    entry("femto_fp4_page_bytes", ctypes.c_size_t, lambda: 2176)
    addresses = {n: ctypes.cast(f, ctypes.c_void_p).value for n, f in keep.items()}
    so = ctypes.CDLL(str(lib))
    flags = {n: ctypes.c_int.in_dll(so, n) for n in ("current_device", "capturing", "capture_error", "fail_wrap")}
    module.bind({n: a for n, a in addresses.items() if "fp4" not in n})
    unbound = [call() for _, call in calls(module).values()]
    module.bind(addresses)
    module.keep = keep, message
    return module, counts, rc, size, flags, unbound


def calls(module):
    """entry point -> (library function, call of its first tensor); each call brings a workspace of 4096 bytes"""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    b16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    pool, tab = torch.zeros(4, 2, 2176, dtype=torch.uint8), torch.zeros(64, 64)
    spaces = lambda: {(-1, 0): torch.zeros(4096, dtype=torch.uint8)}
    return {
        "write_fp4": (FUNCTIONS[0], lambda x=b16(3, 2, 128), pool=pool: module.write_fp4(x, x, pool, i32(3), i32(3, 2), None, 1)),
        "read_fp4": (FUNCTIONS[1], lambda x=i32(3), pool=pool: module.read_fp4(pool, 128, True, x, i32(3, 2), None, 1)),
        "rope_fp4": (FUNCTIONS[2], lambda x=b16(3, 4, 128), pool=pool, w=None, y=None: module.rope_fp4(
            x, b16(3, 2, 128), b16(3, 2, 128), tab, tab, i32(3), pool, i32(3, 2), None, 1, False, w, y, 1e-6, None)),
        "gemv_fp4": (FUNCTIONS[3], lambda x=b16(4, 3, 128), pool=pool: module.gemv_fp4(x, pool, i32(3, 2), i32(3), 20, spaces())),
        "gemm_fp4": (FUNCTIONS[4], lambda x=b16(4, 5, 128), pool=pool: module.gemm_fp4(
            x, pool, i32(2), 5, i32(1, 2), i32(1), i32(5), spaces())),
    }


def test_unbound_functions_decline(native):
    assert native[5] == [None] * 5


@pytest.mark.parametrize("name", NAMES)
def test_call_returns_the_output(native, name):
    module, counts = native[:2]
    fn, call = calls(module)[name]
    before = counts.get(fn, 0)
    out = call()
    assert counts[fn] == before + 1
    if name == "write_fp4":
        assert out is True
    elif name == "read_fp4":
        assert isinstance(out, tuple) and [tuple(t.shape) for t in out] == [(3, 2, 128)] * 2 and out[0].dtype == torch.bfloat16
    else:
        assert isinstance(out, torch.Tensor) and out.dtype == torch.bfloat16


@pytest.mark.parametrize("name", NAMES[1:])
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
    """Writes and reads need no workspace, so capturing does not concern them."""
    module, counts, *_ = native
    fn, call = calls(module)[name]
    var, before = native[4][flag], counts.get(fn, 0)
    old, var.value = var.value, value
    try:
        out = call()
    finally:
        var.value = old
    declined = name.startswith("gem") or flag == "current_device"
    assert (out is None) == declined and counts.get(fn, 0) == before + (not declined)


@pytest.mark.parametrize("name", NAMES)
def test_declined_forms(native, name):
    module, counts, *_ = native
    fn, call = calls(module)[name]
    before = counts.get(fn, 0)

    class Sub(torch.Tensor):
        pass

    if name == "read_fp4":
        x = torch.zeros(3, dtype=torch.int32)
        bad = (x.long(), x[:2], x.as_subclass(Sub), None, [1], x.repeat(2)[::2])
    else:
        x = torch.zeros({"write_fp4": (3, 2, 128), "rope_fp4": (3, 4, 128), "gemv_fp4": (4, 3, 128), "gemm_fp4": (4, 5, 128)}[name],
                        dtype=torch.bfloat16)
        bad = (x.double(), x.float(), x[0], x.as_subclass(Sub), None, [1.0], x[..., ::2], x.transpose(1, 2), x[..., :72])
    for y in bad:
        assert call(y) is None
    pool = torch.zeros(4, 2, 2176, dtype=torch.uint8)
    for y in (pool[..., :2048], pool.view(torch.int8), pool[::2], pool.float(), pool[:, :0], pool[0], None):
        assert call(pool=y) is None
    if name == "rope_fp4":
        w = torch.zeros(128, dtype=torch.bfloat16)
        for a, b in ((w, None), (None, w), (w, w[:64]), (w, w.float()), (w, torch.zeros(256, dtype=torch.bfloat16)[::2])):
            assert call(w=a, y=b) is None
        assert call(w=w, y=w) is not None
        before += 1
    assert counts.get(fn, 0) == before


@pytest.mark.parametrize("name", NAMES[3:])
def test_a_workspace_too_small_is_left_to_the_python_path(native, name):
    module, counts, _, size, *_ = native
    fn, call = calls(module)[name]
    before, size[0] = counts.get(fn, 0), 5000
    try:
        assert call() is None
    finally:
        size[0] = 512
    assert counts.get(fn, 0) == before
