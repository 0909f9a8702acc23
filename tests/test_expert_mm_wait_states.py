"""Distances in front of the loads to LDS that the kernels write themselves, where the
compiler keeps none: one wait state behind a scalar instruction that writes m0, five behind a
vector instruction that writes a scalar register which the load reads. An instruction is one
wait state, s_nop n is n + 1."""

import os
import re

import pytest

from test_code_objects import LLVM, _asm, kernels  # noqa: F401

pytestmark = pytest.mark.skipif(not os.path.exists(LLVM + "/llvm-objdump"),
                                reason="ROCm's LLVM tools are not installed")


def scalars(operands):
    """Numbers of the scalar registers among operands."""
    got = set()
    for first, last, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", operands):
        got |= {int(one)} if one else set(range(int(first), int(last) + 1))
    return got


def short(code):
    """(loads to LDS, what stands too near to one) of a kernel's instructions."""
    lines = [line.split("//")[0].strip() for line in code.splitlines()]
    lines = [line for line in lines if re.match(r"[a-z]\w+( |$)", line)]
    loads, bad = 0, []
    for i, line in enumerate(lines):
        if not re.match(r"(buffer|global)_load_\S+ .*\blds\b|global_load_lds", line):
            continue
        loads += 1
        reads, states, j = scalars(line), 0, i - 1
        while states < 5 and j >= 0:
            before = lines[j]
            name, _, operands = before.partition(" ")
            if states < 1 and name.startswith("s_") and operands.startswith("m0"):
                bad.append((before, line))
            if name.startswith("v_") and scalars(operands.split(",")[0]) & reads:
                bad.append((before, line))
            states += int(operands, 0) + 1 if name == "s_nop" else 1
            j -= 1
    return loads, bad


def test_what_it_finds():
    load = "\n\tbuffer_load_dword v2, s[4:7], 0 offen lds"
    near = "\tv_readlane_b32 s7, v161, 17\n\ts_mov_b32 m0, s3"
    assert short(near + "\n\ts_nop 3" + load) == (1, [])
    assert len(short(near + "\n\ts_nop 2" + load)[1]) == 1
    assert len(short(near + load)[1]) == 2
    assert short("\tv_readlane_b32 s8, v161, 17\n\ts_mov_b32 m0, s3\n\ts_nop 0" + load) == (1, [])


def test_loads_to_lds_keep_their_distance(kernels):  # noqa: F811
    found = {k for k in kernels.values() if re.search(r"\dexpert_mm_(grad_)?kernelI", k[0])}
    assert len(found) >= 38  # by their mangled names: not all of them are taken apart
    for kernel in found:
        loads, bad = short(_asm(kernel))
        assert loads >= 16 and not bad, (kernel[0], loads, bad[:2])
