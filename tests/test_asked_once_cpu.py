"""The table of what each kernel has been allowed on each device (csrc/asked_once.h), asked by several threads at once."""
import shutil
import subprocess
from pathlib import Path

from rllm_b200.csrc import build

HERE = Path(__file__).resolve().parent


def test_threads_on_several_devices(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    exe = tmp_path / "asked_once"
    subprocess.run([cxx, "-std=c++17", "-O2", "-pthread", "-I", str(build.CSRC), str(HERE / "asked_once.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, (r.returncode, r.stdout)
