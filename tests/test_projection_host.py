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
    assert rules.returncode == 0 and "factors: cases 172800 wrong 0\n" in rules.stdout, rules.stdout + rules.stderr


def test_launches_of_the_largest_calls_stay_within_the_stated_limit(rules):
    """The sizes that are taken are those that the header states, and none of their launches needs more than 2^23 workgroups."""
    assert rules.returncode == 0 and "limits: cases" in rules.stdout and rules.stdout.endswith(" wrong 0\n"), rules.stdout + rules.stderr
