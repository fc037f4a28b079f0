"""Builds and runs tests/cpp/test_moe_api.cpp: the C++ classes of the mixture of experts in libkudnn.so."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LIB = ROOT / "kudnn_amd" / "lib"
ROCM = Path("/opt/rocm")


@pytest.fixture(scope="module")
def binary(tmp_path_factory):
    out = tmp_path_factory.mktemp("cpp") / "test_moe_api"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I", str(ROOT / "include"),
                    "-isystem", str(ROCM / "include"), str(ROOT / "tests" / "cpp" / "test_moe_api.cpp"), "-L", str(LIB), "-lkudnn",
                    "-lkudnn_hip", "-L", str(ROCM / "lib"), "-lamdhip64", f"-Wl,-rpath,{LIB}", f"-Wl,-rpath,{ROCM / 'lib'}", "-o", str(out)],
                   check=True)
    return out


def run(binary, *args):
    r = subprocess.run([str(binary), *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "\n0 failed" in r.stdout, r.stdout + r.stderr


def test_refusals_and_moves(binary):
    run(binary)


@pytest.mark.gpu
def test_integers_through_all_classes(binary):
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    run(binary, "--gpu")
