"""Scratch memory of the kernels of the loss head, the norms and the checkpoints, by
the compiler's own listing: none, but for the norms of rows whose chunks and column
sums do not fit the registers (block_norm.hip says which)."""
import concurrent.futures as cf
import os
import re
import shutil
import subprocess

import pytest

from aethelstream_amd import build

SPILL = {
    # Rows of more than 16384 columns, forward and backward, and the backward of a
    # block's rows of more than 12288.
    "block_norm_fwd_kernelILi1024ELi8ELb0",
    "block_norm_bwd_kernelILi1024ELi8ELb1",
    "block_norm_bwd_kernelILi1024ELi8ELb0",
    "block_norm_bwd_kernelILi512ELi8ELb1",
}


def _scratch(source, out):
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "-S", "--offload-device-only",
                    os.path.join(build.CSRC, source), "-o", out], check=True, capture_output=True)
    with open(out) as f:
        listing = f.read()
    return re.findall(r"\.amdhsa_kernel _ZN4nf4s\d+(\w+).*?"
                      r"\.amdhsa_private_segment_fixed_size (\d+)", listing, re.S)


@pytest.mark.skipif(not (os.path.exists(build.HIPCC) or shutil.which(build.HIPCC)),
                    reason="needs hipcc")
def test_no_scratch(tmp_path):
    sources = ("linear_ce.hip", "block_norm.hip", "ckpt8.hip")
    with cf.ThreadPoolExecutor(len(sources)) as ex:
        found = sum(ex.map(lambda s: _scratch(s, str(tmp_path / (s + ".s"))), sources), [])
    assert len(found) > 30
    for name, size in found:
        spills = any(name.startswith(s) for s in SPILL)
        assert (int(size) != 0) == spills, (name, size)
