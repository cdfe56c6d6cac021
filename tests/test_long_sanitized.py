"""The planners of windowed and weighed attention (csrc/plan.cpp, host C++) under
AddressSanitizer and UndefinedBehaviorSanitizer by g++, driven by tests/asan/long_fuzz.cpp."""

import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def fuzz_binary(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ is not available")
    out = str(tmp_path_factory.mktemp("asan") / "long_fuzz")
    subprocess.run(
        [cxx, "-std=c++17", "-O1", "-g", "-fno-omit-frame-pointer",
         "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
         os.path.join(ROOT, "tests", "asan", "long_fuzz.cpp"),
         os.path.join(ROOT, "hayate-exp_amd", "csrc", "plan.cpp"), "-o", out],
        check=True, capture_output=True, text=True)
    return out


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_window_and_weigh_planners_under_sanitizers(fuzz_binary, seed):
    r = subprocess.run([fuzz_binary, str(seed), "100"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-4000:]
    assert r.stdout.strip() == "ok 100"
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr
