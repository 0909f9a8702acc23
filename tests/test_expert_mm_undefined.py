"""Nothing that was never written goes into the experts' products: a workgroup that has
no tile (the grid is an upper bound) forms its loads' stage and buffers, too. In the
compiler's intermediate code of the kernels such a value is a phi of undef or poison."""

import os
import re
import subprocess

import pytest

from mojodgl import _lib

HIPCC = "/opt/rocm/bin/hipcc"

pytestmark = pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc is not installed")


@pytest.mark.parametrize("source", ["expert_mm_bf16", "expert_mm_f16", "expert_mm_f8",
                                    "expert_mm_grad_bf16", "expert_mm_grad_f16"])
def test_kernels_read_nothing_unwritten(source, tmp_path):
    out = str(tmp_path / "code.ll")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off",
                    "-fno-fast-math", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", "-emit-llvm",
                    os.path.join(_lib.CSRC, source + ".hip"), "-o", out],
                   check=True, capture_output=True, timeout=600)
    code = open(out).read()
    assert len(re.findall(r"^define .*amdgpu_kernel .*expert_mm_", code, re.M)) >= 4
    bad = re.findall(r"^.* = phi .*\[ (?:undef|poison),.*$", code, re.M)
    assert not bad, "{} phis, the first: {}".format(len(bad), bad[0].strip()[:200])
