"""The launches of decode steps over the 4-bit arena under windows up to the largest, without a device: in a
process of its own over a stand-in HIP runtime."""

import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))


def test_largest_windows(tmp_path):
    so = str(tmp_path / "host_hip4.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17",
                    os.path.join(HERE, "host_hip4.cpp"), "-o", so], check=True, timeout=120)
    p = subprocess.run([sys.executable, os.path.join(HERE, "host_windows4.py"), so, "largest_windows"],
                       capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.endswith("ok\n"), p.stdout[-2000:] + p.stderr[-2000:]
