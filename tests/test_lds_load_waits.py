"""Wait states in front of the direct global->LDS loads of the built library.

The loads are inline assembly, inside which the compiler does not look for hazards, so the distances that gfx950 asks
for have to come from the source: one wait state between a write of M0 and a load that takes its LDS address from it,
five between a vector instruction that writes a scalar register and a load that takes its base from that register.
The library's own device code is disassembled and every way into such a load is followed backwards."""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from conftest import PKG

M0_STATES, BASE_STATES = 1, 5
TARGET = re.compile(r"<.*\+0x([0-9a-f]+)>\s*$")


def objdump():
    for path in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump")):
        if path and os.path.exists(path):
            return path
    pytest.skip("no llvm-objdump")


def registers(op):
    """Names of a scalar operand: s4, s[4:5], m0, vcc."""
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", op)
    if m:
        return {f"s{i}" for i in range(int(m[1]), int(m[2]) + 1)}
    return {op} if re.fullmatch(r"s\d+|m0|vcc", op) else set()


def written(name, ops):
    """Scalar registers that an instruction writes."""
    if name.startswith(("s_cmp", "s_bitcmp", "s_waitcnt", "s_nop", "s_cbranch", "s_branch")) or not ops:
        return set()
    if name.startswith("s_") or name.startswith("v_"):
        out = registers(ops[0])
        if name.startswith("v_") and len(ops) > 1 and ("_co_" in name or "div_scale" in name or "mad_u64" in name or
                                                       "mad_i64" in name):
            out |= registers(ops[1])
        return out
    return set()


def parse(text):
    """Functions of a listing: lists of (address, name, operands, target address or None)."""
    functions, start = [], 0
    for line in text.splitlines():
        head = re.match(r"^([0-9a-f]{8,}) <.*>:$", line)
        if head:
            functions.append([])
            start = int(head[1], 16)
            continue
        if "//" not in line or not functions:
            continue
        code, rest = line.split("//", 1)
        parts = code.split(None, 1)
        if not parts:
            continue
        ops = [o.strip().split()[0] for o in parts[1].split(",") if o.strip()] if len(parts) > 1 else []
        target = None
        if parts[0].startswith(("s_cbranch", "s_branch")):
            t = TARGET.search(rest)
            target = start + (int(t[1], 16) if t else 0)
        functions[-1].append((int(rest.split(":")[0], 16), parts[0], ops, target))
    return functions


def states_of(name, ops):
    return int(ops[0], 0) + 1 if name == "s_nop" else 1


def faults(function):
    """Loads of a function with too few wait states behind a write, as texts."""
    index = {ins[0]: i for i, ins in enumerate(function)}
    into = {}
    for i, ins in enumerate(function):
        if ins[3] in index:
            into.setdefault(index[ins[3]], []).append(i)

    def before(i):
        ways = list(into.get(i, ()))
        if i > 0 and function[i - 1][1] not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            ways.append(i - 1)
        return ways

    found, loads = [], 0
    for i, (at, name, ops, _) in enumerate(function):
        if not name.startswith("global_load_lds"):
            continue
        loads += 1
        base = registers(ops[1]) if len(ops) > 1 else set()
        todo, seen = [(j, 0) for j in before(i)], set()
        while todo:
            j, states = todo.pop()
            if states >= BASE_STATES or (j, states) in seen:
                continue
            seen.add((j, states))
            _, other, other_ops, _ = function[j]
            out = written(other, other_ops)
            if "m0" in out and states < M0_STATES:
                found.append(f"{at:x} {name}: {states} wait states behind {other} m0")
            if base & out and other.startswith("v_"):
                found.append(f"{at:x} {name} {ops}: {states} wait states behind {other} {other_ops}")
            todo += [(k, states + states_of(other, other_ops)) for k in before(j)]
    return found, loads


def test_the_search_itself():
    listing = """
0000000000001000 <f>:
	v_readfirstlane_b32 s4, v1     // 000000001000: 0
	s_nop 2                        // 000000001004: 0
	s_mov_b32 m0, s6               // 000000001008: 0
	global_load_lds_dwordx4 v0, s[4:5] // 00000000100C: 0
	v_readlane_b32 s5, v1, s3      // 000000001014: 0
	s_cbranch_scc1 2               // 000000001018: 0 <f+0x24>
	s_mov_b32 m0, s6               // 00000000101C: 0
	s_nop 4                        // 000000001020: 0
	global_load_lds_dwordx4 v0, s[4:5] nt // 000000001024: 0
	s_mov_b32 m0, s6               // 00000000102C: 0
	s_nop 0                        // 000000001030: 0
	global_load_lds_dwordx4 v[0:1], off // 000000001034: 0
"""
    found, loads = faults(parse(listing)[0])
    assert loads == 3 and len(found) == 3, found
    assert "100c" in found[0] and "m0" in found[0] + found[1] and "4 wait states" in found[0] + found[1]
    assert "1024" in found[2] and "1 wait states behind v_readlane_b32" in found[2]


def test_direct_loads_keep_their_distance(tmp_path):
    tool = objdump()
    lib = tmp_path / "lib.so"
    shutil.copyfile(PKG._lib.lib_path(), lib)
    subprocess.run([tool, "--offloading", lib.name], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    found, loads = [], 0
    for code in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([tool, "-d", "--no-show-raw-insn", code.name], cwd=tmp_path, check=True,
                              capture_output=True, text=True).stdout
        if "global_load_lds" not in text:
            continue
        for function in parse(text):
            f, n = faults(function)
            found += f
            loads += n
    assert loads > 1000, "the library's direct loads"
    assert not found, f"{len(found)} of {loads} loads: " + "; ".join(found[:10])
