"""What the host side hands to the kernels, without a GPU:
tests/host_launch/host_launch.cpp is linked with csrc/lt_kv.cpp and stands in
for the CUDA runtime and the launchers."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "langtrain_studio_b200" / "csrc"


@pytest.fixture(scope="module")
def host_launch(tmp_path_factory):
    from langtrain_studio_b200 import build

    cuda = Path(build.nvcc()).resolve().parents[1] / "include"
    exe = tmp_path_factory.mktemp("host_launch") / "host_launch"
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", str(ROOT / "include"), "-I", str(CSRC), "-I", str(cuda),
                    str(ROOT / "tests" / "host_launch" / "host_launch.cpp"), str(CSRC / "lt_kv.cpp"),
                    "-o", str(exe), "-ldl"], check=True)

    def run(scenario):
        r = subprocess.run([str(exe), scenario], capture_output=True, text=True, timeout=120,
                           env={"ASAN_OPTIONS": "detect_leaks=0"})
        assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr

    return run


@pytest.mark.parametrize("fmt", ["f16", "q8_0"])
def test_a_call_keeps_its_staging(host_launch, fmt):
    """Calls of more than 512 tokens with shaped scores: the tokens' descriptors
    stay where the launch reads them while the call stages its intervals."""
    host_launch(f"staging-{fmt}")


@pytest.mark.parametrize("what", ["q4_0", "shaped"])
def test_a_refused_capture_leaves_no_trace(host_launch, what):
    """Attention over a 4-bit cache and with shaped scores is refused inside a
    capture before anything is queued on the stream, whatever the call holds."""
    host_launch(f"capture-{what}")


@pytest.mark.parametrize("fmt", ["f16", "q8_0", "q4_0"])
def test_pointers_are_checked_before_the_launch(host_launch, fmt):
    """Null or misaligned device arrays, of which a kernel's 16-byte accesses would
    fault, are refused by every call that takes them, for every cache format."""
    host_launch(f"pointers-{fmt}")
