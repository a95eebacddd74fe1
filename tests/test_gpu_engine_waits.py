"""The tensor-core engine's bounded waits: when its operands never come, every warp gives up as
one, the kernel ends, the status word is set and the GPU goes on working."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from neurocell_b200 import ops

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "neurocell-v2_b200", "csrc")
INCLUDE = os.path.join(os.path.dirname(HERE), "include")


def _build(tmp, limit=64):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    lib = os.path.join(str(tmp), "engine_waits.so")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
                    "-shared", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr", f"-DNC_TC_WAIT_LIMIT={limit}",
                    "-I", CSRC, "-I", INCLUDE, "-o", lib, os.path.join(HERE, "engine_waits.cu")],
                   check=True, capture_output=True, timeout=600)
    return lib


def test_a_whole_warp_leaves_a_wait_together():
    """Where a whole warp waits, an outcome that differed from lane to lane would leave some of
    them behind in elect.sync or __syncwarp: such waits go by a vote."""
    src = open(os.path.join(CSRC, "nc_tc.cuh")).read()
    for role in ("void multiply(", "void collect(", "uint8_t* extra("):
        body = src[src.index(role):]
        body = body[:body.index("\n  }\n")]
        for line in body.splitlines():
            if "_wait(" in line:
                assert "warp_wait(" in line or "__all_sync(" in line, line.strip()


def test_the_starved_engine_builds(tmp_path):
    assert os.path.getsize(_build(tmp_path)) > 0


@pytest.mark.gpu
def test_waits_that_run_out_end_the_kernel(tmp_path):
    lib = ctypes.CDLL(_build(tmp_path))
    # one CTA: 16 epilogue warps and the multiplying one; a pair: twice 8, and the first CTA's
    for pair, threads in ((0, 32 * 17), (1, 32 * 17)):
        for _ in range(2):
            out = (ctypes.c_int * 2)()
            assert lib.starved_engine(pair, out) == 0
            assert out[0] == 1 and out[1] == threads
    x = torch.eye(96, device="cuda:0")
    assert torch.isfinite(ops.orthogonalize(x)).all()
