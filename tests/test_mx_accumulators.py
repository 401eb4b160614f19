"""The MXFP4 product's matrix instructions come from inline assembly, without the compiler's wait states.  Its assembly is read here along every path, loops
included: what a matrix instruction writes, nothing may read or write for 8 wait states, but a matrix instruction that adds to exactly the same registers (its
C and D are the earlier D: the hardware hands them over by itself); and no vector instruction may write an operand in the 2 before it."""
import os
import re
import subprocess

import pytest

from test_mx_wait_states import CSRC, HIPCC, registers


class Instruction:
    def __init__(self, line):
        self.line = line
        self.op, _, rest = line.partition(" ")
        args = [a.split()[0] for a in rest.split(",") if a.split()]
        self.args = args
        self.matrix, self.vector = self.op.startswith("v_mfma"), self.op.startswith("v_")
        sets = [registers(a) for a in args]
        self.passed = int(args[0], 0) + 1 if self.op == "s_nop" else 1
        if self.matrix:  # D, A, B, C, and the two scales
            self.writes, self.c = sets[0], sets[3]
            self.reads = set().union(*sets[1:3], *sets[4:6])
        else:  # (a load's destination is among what `touches` names, and the wait for it comes before it is used)
            self.writes = set().union(*sets[: 2 if "swap" in self.op else 1]) if self.vector else set()
            self.touches = set().union(*sets, set())


def functions(text):
    """{name: ([instruction], [indexes that may follow each])}"""
    found, name = {}, None
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        if re.fullmatch(r"_Z\w+:", line):
            name, labels, items = line[:-1], {}, []
            found[name] = items, labels
        elif name and re.fullmatch(r"\.L\w+:", line):
            labels[line[:-1]] = len(items)
        elif name and line and line[0] != "." and not line.endswith(":"):
            items.append(Instruction(line))
    out = {}
    for name, (items, labels) in found.items():
        after = []
        for i, one in enumerate(items):
            to = [labels[one.args[0]]] if one.op.startswith(("s_branch", "s_cbranch")) and one.args[0] in labels else []
            if one.op not in ("s_branch", "s_endpgm"):
                to.append(i + 1)
            after.append([t for t in to if t < len(items)])
        out[name] = items, after
    return out


def faults(text):
    found = set()
    for name, (items, after) in functions(text).items():

        def walk(i, states, regs, limit, check):
            """check(instruction, wait states so far, registers) on every path from i on"""
            todo, seen = [(t, states) for t in after[i]], set()
            while todo:
                at, n = todo.pop()
                if n >= limit or (at, n) in seen:
                    continue
                seen.add((at, n))
                what = check(items[at], regs)
                if what:
                    found.add((name, what, n, items[at].line))
                todo += [(t, n + items[at].passed) for t in after[at]]

        def of_result(one, regs):
            if one.matrix:
                if one.reads & regs:
                    return "operand of a matrix instruction"
                if (one.c & regs or one.writes & regs) and not one.c == one.writes == regs:
                    return "other accumulator"
            elif one.touches & regs:
                return "result"
            return None

        def of_operand(one, regs):
            return "operand" if one.matrix and (one.reads | one.c) & regs else None

        for i, one in enumerate(items):
            if one.matrix:
                walk(i, 0, one.writes, 8, of_result)
            elif one.writes:
                walk(i, 0, one.writes, 2, of_operand)
    return sorted(found)


def test_the_reader():
    def product(d, a="v[4:7]", b="v[8:11]", c=None):
        return f"v_mfma_scale_f32_16x16x128_f8f6f4 {d}, {a}, {b}, {c or d}, v1, v2 op_sel:[0,0,0] cbsz:4"

    def early(*lines):
        return [f[1:3] for f in faults("\n".join(("_Zk:",) + lines))]

    one = product("a[0:3]")
    assert early(one, one, product("a[4:7]"), "s_nop 7", "v_accvgpr_read_b32 v0, a2") == []
    assert early(one, product("a[2:5]")) == [("other accumulator", 0)]
    assert early(one, product("a[4:7]", c="a[0:3]")) == [("other accumulator", 0)]
    assert early(one, product("a[0:3]", c="a[4:7]")) == [("other accumulator", 0)]
    assert early(one, "s_nop 5", product("a[4:7]", a="a[0:3]")) == [("operand of a matrix instruction", 6)]
    assert early(one, "s_nop 7", product("a[4:7]", a="a[0:3]")) == []
    assert early(one, "v_mov_b32 v0, v9", "v_accvgpr_write_b32 a1, 0") == [("result", 1)]
    assert early("v_lshrrev_b32 v1, s0, v3", "s_nop 0", one) == [("operand", 1)]
    # a loop whose last instruction the next turn reads, and a branch over the wait
    assert early(".LBB0_1:", "v_accvgpr_read_b32 v0, a2", "s_nop 7", one, "s_cbranch_scc1 .LBB0_1", "s_endpgm") == [("result", 1)]
    assert early(".LBB0_1:", "v_accvgpr_read_b32 v0, a2", "s_nop 7", one, "s_nop 15", "s_cbranch_scc1 .LBB0_1", "s_endpgm") == []
    assert early(one, "s_cbranch_scc1 .LBB0_2", "s_nop 15", ".LBB0_2:", "v_accvgpr_read_b32 v0, a2") == [("result", 1)]
    assert early(".LBB0_1:", one, "v_add_u32 v5, v5, v6", "s_cbranch_scc1 .LBB0_1") == [("operand", 1)]


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_accumulators(tmp_path):
    out = tmp_path / "product.s"
    flags = re.search(r"^HIPFLAGS = ((?:.*\\\n)*.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M)[1].replace("\\\n", " ").replace("$(ARCH)", "gfx950").split()
    subprocess.run([HIPCC, *flags, "-w", "--offload-device-only", "-S", "agh_mx_gemm.hip", "-o", str(out)], cwd=CSRC, check=True, capture_output=True)
    text = out.read_text()
    found = functions(text)
    products = [one for items, _ in found.values() for one in items if one.matrix]
    assert len(products) > 500 and all(one.c == one.writes for one in products)
    assert any(t <= i for items, after in found.values() for i, to in enumerate(after) for t in to)  # (loops are seen)
    assert faults(text) == []
    # without the waits behind the last matrix instructions, sums would be written to LDS too early
    assert any(what == "result" and line.startswith("ds_write") for _, what, _, line in faults(text.replace("s_nop 15", "")))
