"""Scalars that a vector instruction writes (v_readfirstlane, v_readlane, a comparison) and the first memory instruction that
takes its address from one: five wait states lie between them on every path, as the compiler keeps for the instructions
it emits.  It does not look into inline assembly, where loads into LDS are written."""
import os
import re
import shutil
import subprocess

import pytest

from llambda_amd import build
from test_mfma_waits import OBJDUMP, _parse

STATES = 5
MEMORY = ("global_", "buffer_", "flat_", "scratch_")


def _scalars(text):
    out = set()
    for first, last, one, m0 in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(m0)\b", text):
        out |= {"m0"} if m0 else set(range(int(first), int(last) + 1)) if first else {int(one)}
    return out


def _first_operand(operands):
    return operands.split(",")[0]


def _short_waits(code):
    """Sites with too few wait states: (states, writer, memory instruction)."""
    index = {at: i for i, (at, *_) in enumerate(code)}
    found = []
    for i, (_, writer, operands, _) in enumerate(code):
        if not writer.startswith("v_"):
            continue
        written = _scalars(_first_operand(operands))
        if not written:
            continue
        paths, least = [(i + 1, 0, frozenset(written))], {}
        while paths:
            p, states, live = paths.pop()
            while p < len(code) and states < STATES and live and least.get((p, live), STATES) > states:
                least[p, live] = states
                _, opcode, args, target = code[p]
                if opcode.startswith("s_cbranch") or opcode == "s_branch":
                    if target in index:
                        paths.append((index[target], states + 1, live))
                    if opcode == "s_branch":
                        break
                elif opcode == "s_endpgm":
                    break
                elif opcode == "s_nop":
                    states += int(args, 0)
                elif opcode.startswith(MEMORY):
                    reads = _scalars(args) | ({"m0"} if "_lds_" in opcode else set())
                    if reads & live:
                        found.append((states, f"{writer} {operands}", f"{opcode} {args}"))
                        break
                else:  # another value from here on
                    live = live - _scalars(_first_operand(args))
                states += 1
                p += 1
    return found


def _listing(lines, targets):
    return "0000000000000000 <k>:\n" + "".join(
        f"\t{text} // {4 * i:012X}: 00000000{targets.get(i, '')}\n" for i, text in enumerate(lines))


def test_short_waits_are_seen():
    load = "global_load_lds_dwordx4 v1, s[4:5]"
    straight = _parse(_listing(["v_readfirstlane_b32 s5, v0", "s_mov_b32 m0, s9", "s_nop 0", load, "s_endpgm"], {}))["k"]
    assert [s for s, *_ in _short_waits(straight)] == [2]
    for line in ("s_nop 4", "s_nop 2"):
        waits = _parse(_listing(["v_readfirstlane_b32 s5, v0", "s_mov_b32 m0, s9", line, "s_nop 0", load, "s_endpgm"], {}))["k"]
        assert not _short_waits(waits)
    other = _parse(_listing(["v_readfirstlane_b32 s5, v0", "s_add_u32 s5, s5, s8", load, "s_endpgm"], {}))["k"]
    assert not _short_waits(other)
    place = _parse(_listing(["v_readfirstlane_b32 m0, v0", "s_nop 0", load, "s_endpgm"], {}))["k"]
    assert [s for s, *_ in _short_waits(place)] == [1]
    # a branch past the wait
    lines = ["v_cmp_lt_i32_e64 s[4:5], v0, v1", "s_cbranch_scc0 1", "s_nop 4", load, "s_endpgm"]
    assert [s for s, *_ in _short_waits(_parse(_listing(lines, {1: " <k+0xc>"}))["k"])] == [1]


def test_built_kernels(tmp_path):
    if not os.path.exists(build.LIB) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no llvm-objdump here")
    lib = shutil.copy(build.LIB, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    loads, bad = 0, []
    for name in sorted(os.listdir(tmp_path)):
        if build.ARCH not in name:
            continue
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", name], cwd=tmp_path, check=True,
                                 stdout=subprocess.PIPE, text=True).stdout
        for kernel, code in _parse(listing).items():
            loads += sum("_lds_" in c[1] for c in code)
            bad += [(kernel, *site) for site in _short_waits(code)]
    assert loads > 1000
    assert not bad, (len(bad), bad[:8])
