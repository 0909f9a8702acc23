"""What the compiler made of the row operators' kernels: registers that their
occupancy rests on, and none spilled to memory."""

import os
import re

import pytest

from test_code_objects import LLVM, _named, _notes, kernels  # noqa: F401

pytestmark = pytest.mark.skipif(not os.path.exists(LLVM + "/llvm-objdump"),
                                reason="ROCm's LLVM tools are not installed")


@pytest.mark.parametrize("pattern", [
    r"scan_pass_kernel<.*", r"scan_step_kernel<.*", r"route_(grad_)?kernel<.*",
    r"norm_kernel<.*", r"norm_grad_kernel<.*, (8|16|32|64|256|512), \d>.*",
    r"(\(anonymous namespace\)::)?combine_(grad_)?kernel<.*",
    r"(\(anonymous namespace\)::)?dispatch_kernel<.*"])
def test_no_registers_in_memory(kernels, pattern):  # noqa: F811
    for name, kernel in _named(kernels, pattern).items():
        assert re.search(r"\.private_segment_fixed_size: 0\b", _notes(kernel)), name


def test_scans_of_16_bit_rows_keep_two_workgroups(kernels):  # noqa: F811
    """128 registers at most: 16 wavefronts, two workgroups, on a compute unit."""
    found = 0
    for name, kernel in kernels.items():
        if re.search(r"scan_pass_kernel", name) and re.search(r"DF16|__bf16|_Float16|half",
                                                              kernel[0] + name):
            notes = _notes(kernel)
            total = sum(int(re.search(p, notes).group(1)) for p in
                        (r"\.vgpr_count: +(\d+)",))
            assert total <= 128, name
            found += 1
    assert found >= 8
