"""Registers of the kernels that count their waits (``s_waitcnt vmcnt(N)`` over a ring of loads in flight), compiled with the flags
that the library is built with: a spilled register is one more memory operation on that counter, and hipcc waits for it with
``vmcnt(0)``, which drains the ring (no GPU needed: hipcc cross-compiles gfx950)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "biomedkg_amd", "csrc")

KERNELS = {
    "gemm_xw": {"gemm_xw8k_kernel": 6, "gemm_xw8_kernelIDF16bLb1E": 1},
    "kge_bwd_nodes": {"kge_onepass_kernelIDF16bLi16ELi2E": 1},
    "kge_onepass_mx": {"kge_onepass_mx_kernelILb0E": 1, "kge_onepass_mx_kernelILb1E": 1},
    "mx4": {"mx4_tile_kernel": 6, "mx4_stream_kernel": 36},
}


def shipped_flags():
    flags = re.search(r'^FLAGS="\$\{EXTRA_FLAGS\} (.*)"$', open(os.path.join(CSRC, "build.sh")).read(), re.M).group(1).split()
    assert "--offload-arch=gfx950" in flags and "-packed-fp32-ops" in flags
    return flags


@pytest.fixture(scope="module")
def reports(tmp_path_factory):
    """source -> what hipcc says of its kernels (all compiled side by side)"""
    if shutil.which("hipcc") is None:
        pytest.skip("hipcc not on PATH")
    tmp = tmp_path_factory.mktemp("resources")
    runs = {source: subprocess.Popen(["hipcc", *shipped_flags(), "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-c",
                                      source + ".hip", "-o", str(tmp / (source + ".o"))], stderr=subprocess.PIPE, text=True, cwd=CSRC)
            for source in KERNELS}
    return {source: (run.communicate(timeout=900)[1], run.returncode) for source, run in runs.items()}


@pytest.mark.parametrize("source", list(KERNELS))
def test_kernels_that_count_their_waits_do_not_spill(source, reports):
    said, rc = reports[source]
    assert rc == 0, said[-2000:]
    seen = dict.fromkeys(KERNELS[source], 0)
    for block in re.split(r"remark: Function Name: ", said)[1:]:
        name = block.split()[0]
        for key in seen:
            if key in name:
                seen[key] += 1                       # (a spilled scalar register goes to a vector register's lanes, not to memory)
                spill = int(re.search(r"VGPRs Spill: (\d+)", block).group(1))
                scratch = int(re.search(r"ScratchSize \[bytes/lane\]: (\d+)", block).group(1))
                assert spill == 0 and scratch == 0, (name, spill, scratch)
    assert seen == KERNELS[source]
