"""The planner of shared prefixes and selected pages under AddressSanitizer and
UndefinedBehaviorSanitizer: ``tests/native/segment_plan_fuzz.cpp`` drives
``pg_segment_plan_host`` with random and malformed batches.  Plain C++, built here
with the host compiler; no GPU is involved."""

from __future__ import annotations

import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "pagegauge_amd" / "csrc"


@pytest.fixture(scope="module")
def fuzzer(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ is not available")
    exe = tmp_path_factory.mktemp("segments") / "segment_plan_fuzz"
    cmd = [cxx, "-std=c++17", "-O1", "-g", "-Wall", "-Wextra", "-Werror",
           "-fsanitize=address,undefined", "-fno-sanitize-recover=all", "-fno-omit-frame-pointer",
           f"-I{ROOT / 'include'}", f"-I{CSRC}", str(ROOT / "tests" / "native" / "segment_plan_fuzz.cpp"),
           str(CSRC / "pg_segment_plan.cpp"), str(CSRC / "pg_error.cpp"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True, timeout=240)
    return exe


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_segment_plans_under_sanitizers(fuzzer, seed):
    run = subprocess.run([str(fuzzer), str(seed), "600"], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stdout + run.stderr
    word, plans, rejected = run.stdout.split()
    assert word == "ok" and int(plans) > 300 and int(rejected) > 10
