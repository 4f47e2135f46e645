"""The layer-boundary kernels as built: none keeps registers in scratch memory.  Their column sums and
accumulators live through whole kernels; a build of the norms' backward pass that spilled some of them
gave wrong sums, and a spilled matrix tile would be slow.  Read from the kernels' metadata in the
library (no GPU needed)."""
import os
import re
import shutil
import subprocess

import pytest

READELF = "/opt/rocm/llvm/bin/llvm-readelf"
KERNELS = ("all_reduce_norm_kernel", "all_reduce_norm_narrow_kernel", "norm_backward_kernel", "norm_backward_narrow_kernel",
           "norm_columns_kernel", "norm_sums_kernel", "mxfp4_quantize_kernel", "mxfp4_quantize_columns_kernel",
           "mxfp4_dequantize_kernel", "mxfp4_matmul_few_kernel", "mxfp4_matmul_rows_kernel", "mxfp4_matmul_ring_kernel",
           "mxfp4_matmul_tile_kernel")


@pytest.fixture(scope="module")
def scratch(lib, tmp_path_factory):
    """{kernel: bytes of scratch memory per lane}"""
    if shutil.which(READELF) is None:
        pytest.skip("llvm-readelf not available")
    from symm_mem_recipes import _lib
    data = open(_lib.LIB_PATH, "rb").read()
    starts = [m.start() for m in re.finditer(b"\x7fELF\x02\x01\x01\x40", data)]      # the device's ABI byte
    assert starts, "no device code found in the library"
    found, work = {}, tmp_path_factory.mktemp("isa")
    for i, at in enumerate(starts):
        f = work / f"{i}.co"
        f.write_bytes(data[at:starts[i + 1] if i + 1 < len(starts) else len(data)])
        notes = subprocess.run([READELF, "--notes", str(f)], capture_output=True, text=True).stdout
        for m in re.finditer(r"\.name:\s+(\S+)\n.*?\.private_segment_fixed_size:\s+(\d+)", notes, re.S):
            found[m.group(1)] = int(m.group(2))
    return found


@pytest.mark.parametrize("kernel", KERNELS)
def test_no_scratch_memory(scratch, kernel):
    sizes = {k: v for k, v in scratch.items() if re.match(r"_ZN3smr\d+" + kernel + r"I", k)}
    assert sizes, "not in the library"
    assert not any(sizes.values()), {k: v for k, v in sizes.items() if v}
