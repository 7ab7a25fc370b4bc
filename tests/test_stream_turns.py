"""Whole turns on streams of any origin (tests/stream_turns.cpp), without a device."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "fast-llm_amd", "libfastllm_hip.so")
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")


@pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")
def test_turns(tmp_path):
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    exe = tmp_path / "stream_turns"
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROCM, "include"),
                    os.path.join(ROOT, "tests", "stream_turns.cpp"), "-o", str(exe), LIB, "-Wl,-rpath," + os.path.dirname(LIB),
                    "-Wl,-rpath-link," + os.path.join(ROCM, "lib")], check=True, capture_output=True, text=True)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and p.stdout == "ok\n", p.stdout + p.stderr
