"""CPU tests of the host rules of the learned projections: a CPU build of vectordb_amd/csrc/project.h."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    """Output of tests/native/projection_rules.cpp."""
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    if shutil.which("g++") is None or not os.path.isdir(os.path.join(rocm, "include", "hip")):
        pytest.skip("no host compiler or no HIP headers")
    exe = str(tmp_path_factory.mktemp("rules") / "projection_rules")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-isystem", os.path.join(rocm, "include"),
                           os.path.join(ROOT, "tests", "native", "projection_rules.cpp"), "-o", exe])
    return subprocess.run([exe], capture_output=True, text=True, timeout=120)


def test_vectors_of_a_factor_lie_inside_it(rules):
    """Whatever the sizes (one input column among them, where a backward pass has ranks one element apart)."""
    assert rules.returncode == 0 and " wrong 0" in rules.stdout, rules.stdout + rules.stderr
