"""Registers of every instance of the kernels of layers of experts (the
root-mean-square norm, values in 8 bits, the experts' products), found by their mangled
names."""

import os
import re

import pytest

from test_code_objects import LLVM, _run, kernels  # noqa: F401

pytestmark = pytest.mark.skipif(not os.path.exists(LLVM + "/llvm-objdump"),
                                reason="ROCm's LLVM tools are not installed")

FLOAT, DOUBLE, BF16, F16 = "f", "d", "DF16b", "DF16_"
KERNELS = {"rms_kernel": (FLOAT, DOUBLE, BF16, F16), "rms_grad_kernel": (FLOAT, DOUBLE, BF16, F16),
           "rms_wide_kernel": (FLOAT, DOUBLE, BF16, F16),
           "rms_cols_kernel": (FLOAT, DOUBLE, BF16, F16),
           "quant_rows_kernel": (FLOAT, BF16, F16), "quant_blocks_kernel": (FLOAT, BF16, F16),
           "expert_mm_join_kernel": (FLOAT, BF16, F16), "expert_mm_sum_kernel": (BF16, F16),
           # by a configuration, whose first argument is the type
           "expert_mm_kernel": ("NS_6MmConfI" + BF16, "NS_6MmConfI" + F16, "NS_6MmConfINS_4f8_t"),
           "expert_mm_grad_kernel": ("NS_6MmConfI" + BF16, "NS_6MmConfI" + F16)}


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
            if kernel in KERNELS:
                got.setdefault(kernel, {})[rest] = {
                    f: int(v) for f, v in re.findall(r"\.(\w+): +(\d+)\s", entry)}
    return got


@pytest.mark.parametrize("kernel", list(KERNELS))
def test_no_registers_in_memory(found, kernel):
    for t in KERNELS[kernel]:
        assert any(rest.startswith("I" + t) for rest in found[kernel]), t
    for rest, notes in found[kernel].items():
        assert notes["private_segment_fixed_size"] == 0, rest
        assert notes["vgpr_spill_count"] == 0, rest
