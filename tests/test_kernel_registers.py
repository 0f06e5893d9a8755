"""The vector registers that the compiler gave the kernels around the expert layer: how many waves a SIMD holds of each.
(512 a lane, handed out by eights: up to 168 three waves fit, up to 128 four.)"""
import os
import re
import subprocess

import pytest

from tests.test_kernel_resources import LIB, READELF, code_objects


@pytest.fixture(scope="module")
def registers(tmp_path_factory):
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    from umdk_amd import _lib
    _lib.lib()  # (its missing-library message first)
    d, found = tmp_path_factory.mktemp("co"), {}
    for i, co in enumerate(code_objects(open(LIB, "rb").read())):
        f = d / f"{i}.co"
        f.write_bytes(co)
        notes = subprocess.run([READELF, "--notes", str(f)], capture_output=True, text=True, check=True).stdout
        for k in re.split(r"\n  - \.a", notes)[1:]:
            found[re.search(r"\n\s+\.name:\s+(\S+)", k).group(1)] = int(re.search(r"\n\s+\.vgpr_count:\s+(\d+)", k).group(1))
    return found


@pytest.mark.parametrize("kernel,count,most", [("route_grouped_kernel", 30, 168), ("add_rms_norm_kernel", 42, 128)])
def test_waves_a_simd(registers, kernel, count, most):
    mine = {k: v for k, v in registers.items() if kernel in k}
    assert len(mine) >= count
    assert {k: v for k, v in mine.items() if v > most} == {}
