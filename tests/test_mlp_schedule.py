"""The fused encoder MLP kernel reads the next stage's operands only behind the barrier that publishes them, at every hidden size, with and
without the output projection in front: tests/c/mlp_schedule.cpp walks the stages by the kernel's own rule (moonshine_amd/csrc/mlp_schedule.h)."""
import ctypes as C
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("mlp_schedule") / "mlp_schedule.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(HERE, "..", "moonshine_amd", "csrc"),
                    os.path.join(HERE, "c", "mlp_schedule.cpp"), "-o", out], check=True)
    return C.CDLL(out)


@pytest.mark.parametrize("hidden", [64, 288, 416])
@pytest.mark.parametrize("oproj", [0, 1])
@pytest.mark.parametrize("chunks", [1, 2, 3, 8, 52])
@pytest.mark.parametrize("ahead", [2, 4])
def test_no_stage_is_read_before_it_is_published(lib, hidden, oproj, chunks, ahead):
    assert lib.mlp_schedule_walk(hidden, oproj, chunks, ahead) == 0
