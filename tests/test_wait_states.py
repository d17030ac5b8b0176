"""The wait states that gfx950 needs between instructions, in the machine code of the library that is built here.

The compiler puts them between its own instructions but does not look into inline assembly (the GEMMs' copies into LDS
and the stores that are counted for their waits). What is looked for, a state being an instruction or one of ``s_nop``'s:

* a copy into LDS reads its LDS address from M0: one state behind the scalar instruction that writes M0;
* a store of more than 8 bytes reads its data late: two states before a vector instruction overwrites them;
* a memory instruction reads a scalar register that a vector instruction wrote: five states between them.

Straight runs are followed; a branch ends one."""

import os
import re
import shutil
import subprocess

import pytest

from sgl_asap_amd import _lib

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm/bin/llvm-objdump")
REGISTERS = re.compile(r"\b([sv])(?:(\d+)|\[(\d+):(\d+)\])(?!\w)|\b(m0|vcc)\b")
MEMORY = ("global_", "buffer_", "flat_", "scratch_")
BRANCHES = ("s_branch", "s_cbranch", "s_endpgm", "s_setpc", "s_swappc")


def registers(operand):
    found = set()
    for kind, one, lo, hi, name in REGISTERS.findall(operand):
        if name:
            found.add(name)
        else:
            found.update(f"{kind}{i}" for i in range(int(lo or one), int(hi or one) + 1))
    return found


def written_by(op, operands):
    """The registers that a vector or scalar instruction writes (its first operand; a second one where it is a carry or a
    swap's other side)."""
    if not operands or op.startswith(("s_cmp", "s_bitcmp", "s_waitcnt", "s_nop", "s_barrier", "s_set", "v_nop")) or op.startswith(MEMORY):
        return set()
    out = registers(operands[0])
    if len(operands) > 1 and ("_co_" in op or "mad_u64" in op or "mad_i64" in op or "div_scale" in op or "swap" in op):
        out |= registers(operands[1])
    if op.startswith("v_cmp") and "vcc" not in operands[0] and not operands[0].startswith("s"):
        out = {"vcc"}
    return out


def missing_waits(lines):
    """(kernel, what, the two instructions) of each place of a disassembly that has too few states."""
    found, kernel, at = [], "", 0
    m0, stores, scalars = None, [], {}  # (state, text) of what the next instructions have to keep away from
    for line in lines:
        if line.endswith(">:"):
            kernel = line.rsplit("<", 1)[1][:-2]
            m0, stores, scalars = None, [], {}
            continue
        text = line.split("//")[0].strip()
        if not text or ":" in text.split()[0]:
            continue
        op, _, rest = text.partition(" ")
        operands = [o.strip() for o in re.split(r",(?![^\[]*\])", rest)] if rest else []
        if op == "s_nop":
            at += int(rest, 0) + 1
            continue
        memory = op.startswith(MEMORY)
        to_lds = memory and ("_lds_" in op or rest.split()[-1:] == ["lds"])
        if to_lds and m0 and at - m0[0] < 1:
            found.append((kernel, "M0", m0[1], text))
        writes = written_by(op, operands)
        if op.startswith("v_"):
            for state, data, store in stores:
                if at - state < 2 and data & writes:
                    found.append((kernel, "data of a store", store, text))
            for r in writes:
                if r[0] == "s" or r == "vcc":
                    scalars[r] = (at + 1, text)
        elif op.startswith("s_"):
            if "m0" in writes:
                m0 = (at + 1, text)
            for r in writes:
                scalars.pop(r, None)
        if memory:
            for r in registers(rest):
                if r in scalars and at - scalars[r][0] < 5:
                    found.append((kernel, "scalar of a vector instruction", scalars[r][1], text))
        at += 1
        stores = [s for s in stores if at - s[0] < 2]
        if memory and "_store_dwordx" in op and op[-1] in "34":
            data = operands[0] if op.startswith("buffer_") else operands[1]
            stores.append((at, registers(data), text))
        if op.startswith(BRANCHES):
            m0, stores, scalars = None, [], {}
    return found


@pytest.mark.parametrize("code,what", [
    ("s_mov_b32 m0, s4\nglobal_load_lds_dwordx4 v2, s[4:5]", "M0"),
    ("s_mov_b32 m0, s4\ns_nop 0\nglobal_load_lds_dwordx4 v2, s[4:5]", None),
    ("s_add_i32 m0, s4, 0x400\nv_add_u32_e32 v1, v2, v3\nglobal_load_lds_dword v2, s[4:5]", None),
    ("global_store_dwordx4 v[4:5], v[0:3], off\nv_mov_b32_e32 v3, 0", "data of a store"),
    ("global_store_dwordx4 v[4:5], v[0:3], off\ns_nop 0\nv_mov_b32_e32 v3, 0", "data of a store"),
    ("global_store_dwordx4 v[4:5], v[0:3], off\ns_nop 1\nv_mov_b32_e32 v3, 0", None),
    ("global_store_dwordx4 v[4:5], v[0:3], off\nv_mov_b32_e32 v9, 0\ns_nop 0\nv_mov_b32_e32 v3, 0", None),
    ("global_store_dwordx4 v[4:5], v[0:3], off\nv_mov_b32_e32 v4, 0", None),
    ("global_store_dwordx2 v[4:5], v[0:1], off\nv_mov_b32_e32 v1, 0", None),
    ("v_readfirstlane_b32 s4, v1\ns_nop 3\nglobal_load_dword v2, v3, s[4:5]", "scalar of a vector instruction"),
    ("v_readfirstlane_b32 s4, v1\ns_nop 4\nglobal_load_dword v2, v3, s[4:5]", None),
    ("v_readfirstlane_b32 s4, v1\ns_mov_b32 s4, 0\nglobal_load_dword v2, v3, s[4:5]", None),
])
def test_what_is_found(code, what):
    assert [w for _, w, _, _ in missing_waits(["0 <kernel>:"] + code.split("\n"))] == ([what] if what else [])


def test_the_library_has_the_wait_states(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    _lib.lib()
    path = shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", path], cwd=tmp_path, check=True, capture_output=True)
    images = sorted(f for f in os.listdir(tmp_path) if f.endswith("gfx950"))
    assert images
    bad, seen = [], 0
    for image in images:
        code = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", image], cwd=tmp_path, check=True, capture_output=True, text=True)
        lines = code.stdout.split("\n")
        seen += sum("_load_lds_" in line for line in lines)
        bad += missing_waits(lines)
    assert seen > 0
    assert not bad, (len(bad), sorted({(w, a.split()[0], b.split()[0]) for _, w, a, b in bad}), bad[:3])
