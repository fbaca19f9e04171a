"""Decode steps over the 4-bit arena (windows up to the largest, short rows, fewer rows than a step's, refusals) and
the largest projections, without a device: in processes of their own over a stand-in HIP runtime."""

import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("scenario", ["largest_windows", "short_rows", "fewer_rows", "refused_before_anything",
                                      "largest_weights"])
def test_scenario(tmp_path, scenario):
    so = str(tmp_path / "host_hip4.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17",
                    os.path.join(HERE, "host_hip4.cpp"), "-o", so], check=True, timeout=120)
    p = subprocess.run([sys.executable, os.path.join(HERE, "host_decode4.py"), so, scenario],
                       capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.endswith("ok\n"), p.stdout[-2000:] + p.stderr[-2000:]
