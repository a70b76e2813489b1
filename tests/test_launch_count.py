"""The count of launches under several threads, on the CPU (launch_count_check.cpp over the library's own counter)."""
import os
import subprocess

from conftest import ROOT


def test_no_launch_is_lost(tmp_path):
    exe = str(tmp_path / "launch_count_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-I/usr/local/cuda/include", os.path.join(ROOT, "tests", "launch_count_check.cpp"), "-o", exe, "-lpthread"], check=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
