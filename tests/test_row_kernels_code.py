"""Registers of every instance of the row operators' kernels, found by their mangled
names: the demangler does not know the 16-bit types."""

import os
import re

import pytest

from test_code_objects import LLVM, _run, kernels  # noqa: F401

pytestmark = pytest.mark.skipif(not os.path.exists(LLVM + "/llvm-objdump"),
                                reason="ROCm's LLVM tools are not installed")

FLOAT, DOUBLE, BF16, F16 = "f", "d", "DF16b", "DF16_"
TYPES = (FLOAT, DOUBLE, BF16, F16)
BY_TYPE = ["scan_pass_kernel", "scan_step_kernel", "norm_kernel", "norm_grad_kernel",
           "norm_wide_kernel", "norm_cols_kernel", "route_kernel", "route_grad_kernel",
           "dispatch_kernel", "combine_kernel", "combine_grad_kernel"]
OTHERS = ["norm_sum_kernel", "scan_empty_kernel", "scan_reset_kernel", "segment_marks_kernel",
          "plan_one_kernel", "plan_count_kernel", "plan_scan_kernel", "plan_place_kernel"]


@pytest.fixture(scope="module")
def found(kernels):  # noqa: F811
    """{kernel: {template arguments, mangled: {metadata field: number}}}"""
    got = {}
    for path in sorted({path for _, path in kernels.values()}):
        for entry in _run(LLVM + "/llvm-readelf", "--notes", path).split("- .agpr_count")[1:]:
            name = re.search(r"\.name: +(\S+)", entry).group(1)
            part = re.match(r"_ZN4mdgl(?:12_GLOBAL__N_1)?(\d+)(.*)", name)
            if not part:
                continue
            size = int(part.group(1))
            kernel, rest = part.group(2)[:size], part.group(2)[size:]
            if kernel in BY_TYPE + OTHERS:
                got.setdefault(kernel, {})[rest] = {
                    f: int(v) for f, v in re.findall(r"\.(\w+): +(\d+)\s", entry)}
    return got


@pytest.mark.parametrize("kernel", BY_TYPE + OTHERS)
def test_no_registers_in_memory(found, kernel):
    instances = found[kernel]
    if kernel in BY_TYPE:
        for t in TYPES:
            assert any(rest.startswith("I" + t) for rest in instances), t
    for rest, notes in instances.items():
        assert notes["private_segment_fixed_size"] == 0, rest
        assert notes["vgpr_spill_count"] == 0, rest


def test_instances_of_layer_norm(found):
    """Threads a row and vectors a thread: rows in registers of every type."""
    shapes = {(8, 1), (16, 1), (32, 1), (64, 1), (64, 2), (256, 1), (256, 2), (512, 2), (512, 4)}
    for kernel in ("norm_kernel", "norm_grad_kernel"):
        for t in TYPES:
            have = {(int(a), int(b)) for rest in found[kernel] if rest.startswith("I" + t)
                    for a, b in re.findall(r"Li\d+ELi(\d+)ELi(\d+)E", rest)}
            assert have >= shapes | ({(1024, 4)} if t in (FLOAT, DOUBLE) else set()), (kernel, t)


def test_scans_of_16_bit_rows_keep_two_workgroups(found):
    """128 registers at most: 16 wavefronts, two workgroups, on a compute unit."""
    some = [n for rest, n in found["scan_pass_kernel"].items() if rest.startswith(("I" + BF16,
                                                                                   "I" + F16))]
    assert len(some) == 16 and all(n["vgpr_count"] <= 128 for n in some)
