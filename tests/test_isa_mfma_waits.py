"""Static check of the MFMA kernels' gfx950 code (CPU only: hipcc -S): no instruction reads an MFMA's result too early.

The hardware does not hold up a VALU, LDS or memory instruction, or another MFMA's A or B operand, that reads the result
of an MFMA of P passes: P + 4 wait states have to lie between them, which the compiler fills with s_nop (an instruction
is one, s_nop N is N + 1).  It has left them out across branches: at the target of an early exit from a row of MFMAs.
Every path from every MFMA is followed here, through both sides of each branch.
"""

import importlib.util
import os
import re
import subprocess

import pytest

from test_isa_prefill import PKG

PASSES = {"16x16x16": 4, "16x16x32": 4, "32x32x16": 8}
READERS = ("v_", "ds_", "global_", "buffer_", "flat_", "scratch_")


def registers(operand):
    m = re.match(r"^-?\|?([av])(?:(\d+)|\[(\d+):(\d+)\])\|?$", operand.split()[0] if operand else "")
    if not m:
        return frozenset()
    lo, hi = (m[2], m[2]) if m[2] else (m[3], m[4])
    return frozenset((m[1], i) for i in range(int(lo), int(hi) + 1))


def parse(lines):
    """([(opcode, operands)], {label: index of its instruction})"""
    code, labels = [], {}
    for line in lines:
        line = line.split(";")[0].split("//")[0].strip()
        label = re.match(r"^([.\w$]+):$", line)
        if label:
            labels[label[1]] = len(code)
        elif line and not line.startswith("."):
            op, _, rest = line.partition(" ") if " " in line else line.partition("\t")
            code.append((op.strip(), [x.strip() for x in re.split(r",(?![^\[]*\])", rest)] if rest.strip() else []))
    return code, labels


def early_reads(lines):
    """(MFMA, reader, missing wait states) of every result read too early."""
    code, labels = parse([re.sub(r"^(\s*\S+)\t", r"\1 ", x) for x in lines])
    found = []

    def follow(i):
        op, args = code[i]
        if op == "s_endpgm":
            return ()
        if op == "s_branch":
            return (labels[args[0]],)
        return ((i + 1,) if i + 1 < len(code) else ()) + ((labels[args[0]],) if op.startswith("s_cbranch") else ())

    for i, (op, args) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        result, needed = registers(args[0]), next(p for k, p in PASSES.items() if k in op) + 4
        fewest, todo = {}, [(j, 0) for j in follow(i)]
        while todo:
            j, waited = todo.pop()
            if waited >= needed or fewest.get(j, needed) <= waited:
                continue
            fewest[j] = waited
            op2, args2 = code[j]
            if op2.startswith("v_mfma"):
                if any(registers(x) & result for x in args2[1:3]):
                    found.append((i, j, needed - waited))
                    continue
                if registers(args2[0]) & result:
                    continue  # accumulates on: its own result from here
            elif op2.startswith(READERS) and any(registers(x) & result for x in args2):
                found.append((i, j, needed - waited))
                continue
            todo += [(k, waited + (int(args2[0], 0) + 1 if op2 == "s_nop" else 1)) for k in follow(j)]
    return [(" ".join([code[i][0], *code[i][1]]), " ".join([code[j][0], *code[j][1]]), n) for i, j, n in found]


def test_the_check_sees_an_early_exit():
    straight = ["v_mfma_f32_16x16x16_bf16 a[0:3], v[4:5], v[6:7], a[0:3]", "s_nop 7", "v_accvgpr_read_b32 v1, a3", "s_endpgm"]
    assert early_reads(straight) == []
    assert early_reads([x.replace("s_nop 7", "s_nop 6") for x in straight])[0][2] == 1
    exits = ["v_mfma_f32_16x16x16_bf16 a[0:3], v[4:5], v[6:7], a[0:3]", "s_cbranch_vccnz .L1",
             "v_mfma_f32_16x16x16_bf16 a[4:7], v[4:5], v[6:7], a[4:7]", "s_nop 7", "v_accvgpr_read_b32 v1, a7", ".L1:",
             "v_accvgpr_read_b32 v2, a3", "s_endpgm"]
    assert [x[2] for x in early_reads(exits)] == [7]
    assert early_reads(exits[:6] + ["s_nop 6"] + exits[6:]) == []
    chain = ["v_mfma_f32_32x32x16_f16 v[0:15], v[20:23], v[24:27], 0", "v_mfma_f32_32x32x16_f16 v[0:15], v[28:31], v[24:27], v[0:15]",
             "s_nop 11", "ds_write_b128 v40, v[4:7]", "s_endpgm"]
    assert early_reads(chain) == []  # on into the same registers: no wait
    assert len(early_reads(chain[:1] + ["v_mfma_f32_32x32x16_f16 v[40:55], v[0:3], v[24:27], 0"] + chain[2:])) == 1


@pytest.mark.parametrize("source,kernels", [("window_decode.hip", 8), ("window_prefill.hip", 24), ("shared_prefix.hip", 12),
                                            ("paged_prefill.hip", 30)])
def test_no_result_is_read_early(tmp_path, source, kernels):
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
    lines = out.read_text().split("\n")
    found = 0
    for s, line in enumerate(lines):
        name = re.match(r"^(_ZN5femto\w+):", line)
        if not name or "_kernelI" not in name[1]:
            continue
        body = lines[s + 1:next(j for j in range(s, len(lines)) if lines[j].startswith(".Lfunc_end"))]
        if not any("v_mfma" in x for x in body):
            continue
        found += 1
        early = early_reads(body)
        assert not early, (name[1], len(early), early[:3])
    assert found == kernels
