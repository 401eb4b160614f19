"""The MXFP4 product issues its matrix instructions from inline assembly, where the compiler inserts no wait states.  Its assembly is read here, in the order of
the text, for the two that the instructions need: 2 between a vector instruction and a matrix instruction that reads its result, 8 between a matrix
instruction and another kind of instruction that reads its result."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "autograph_amd", "csrc")
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def registers(operand):
    m = re.fullmatch(r"([va])(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    first, last = (m[2], m[2]) if m[2] else (m[3], m[4])
    return {(m[1], i) for i in range(int(first), int(last) + 1)}


def faults(text):
    """(function, what, wait states, instruction) of every reader that comes too early."""
    found, function, written, results = [], None, [], []
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        if re.fullmatch(r"_Z\w+:", line):
            function, written, results = line[:-1], [], []
        if not line or line[0] == "." or line.endswith(":"):
            continue
        op, _, rest = line.partition(" ")
        args = [a.split()[0] for a in rest.split(",") if a.split()]
        matrix, vector = op.startswith("v_mfma"), op.startswith("v_")
        reads = set().union(*(registers(a) for a in (args[1:6] if matrix else args[1:] if vector else args)), set())
        if matrix:
            found += [(function, "operand", n, line) for n, regs in written if n < 2 and regs & reads]
        else:
            found += [(function, "result", n, line) for n, regs in results if n < 8 and regs & reads]
        passed = int(args[0]) + 1 if op == "s_nop" else 1
        own = registers(args[0]) if vector and args else set()
        written = [(n + passed, regs - own) for n, regs in written if n < 2]
        results = [(n + passed, regs if matrix else regs - own) for n, regs in results if n < 8]
        if own:
            (results if matrix else written).append((0, own))
    return found


def test_the_reader():
    product = "v_mfma_scale_f32_16x16x128_f8f6f4 a[0:3], v[4:7], v[8:11], a[0:3], v1, v2 op_sel:[0,0,0] cbsz:4"
    early = lambda *lines: [f[1:3] for f in faults("\n".join(("_Zk:",) + lines))]  # noqa: E731
    assert early("v_lshrrev_b32 v1, s0, v3", product) == [("operand", 0)]
    assert early("v_lshrrev_b32 v1, s0, v3", "s_nop 0", product) == [("operand", 1)]
    assert early("v_lshrrev_b32 v1, s0, v3", "s_nop 1", product) == []
    assert early("v_mov_b32 v6, v3", "v_mov_b32 v12, v3", product) == [("operand", 1)]
    assert early(product, product) == []
    assert early(product, "v_accvgpr_read_b32 v0, a2") == [("result", 0)]
    assert early(product, "s_nop 7", "v_accvgpr_read_b32 v0, a2") == []
    assert early(product, "s_nop 6", "ds_write_b128 v3, a[0:3]") == [("result", 7)]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_wait_states(tmp_path):
    out = tmp_path / "product.s"
    flags = re.search(r"^HIPFLAGS = ((?:.*\\\n)*.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M)[1].replace("\\\n", " ").replace("$(ARCH)", "gfx950").split()
    subprocess.run([HIPCC, *flags, "-w", "--offload-device-only", "-S", "agh_mx_gemm.hip", "-o", str(out)], cwd=CSRC, check=True, capture_output=True)
    text = out.read_text()
    assert text.count("v_mfma_scale_f32_16x16x128_f8f6f4") > 500
    assert faults(text) == []
