"""The rows that the operators around the pick give to each launch, up to the largest batch that their arguments hold:
the entry points compiled on the CPU over doubles of the launchers (logits_launches.cpp). No GPU calls."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
HIP = Path("/opt/rocm/include")

pytestmark = pytest.mark.skipif(shutil.which("g++") is None or not (HIP / "hip" / "hip_runtime.h").exists(),
                                reason="g++ or the HIP headers absent")


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    exe = tmp_path_factory.mktemp("launches") / "launches"
    subprocess.run(["g++", "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I", str(HIP), "-I", str(ROOT / "include"),
                    "-I", str(ROOT / "verbo_amd" / "csrc"), str(ROOT / "verbo_amd" / "csrc" / "vsmp_logits_api.cpp"),
                    str(ROOT / "tests" / "logits_launches.cpp"), "-o", str(exe)], check=True)
    return exe


@pytest.mark.parametrize("call", ["adjust", "adjust_left", "logprobs", "head"])
@pytest.mark.parametrize("B", [1, 8192, 65537, (1 << 20) + 1, (1 << 31) - (1 << 20), (1 << 31) - 1])
def test_every_row_is_launched_once(launches, call, B):
    run = subprocess.run([str(launches), call, str(B)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and run.stdout.startswith("ok "), run.stdout
