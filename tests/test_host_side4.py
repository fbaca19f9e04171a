"""The host side of the 4-bit calls and of steps built on the device, without a device: each scenario of
host_side4.py in a process of its own over a stand-in HIP runtime."""

import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host_hip4") / "host_hip4.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17",
                    os.path.join(HERE, "host_hip4.cpp"), "-o", so], check=True, timeout=120)
    return so


@pytest.mark.parametrize("scenario", ["host_memory", "device_memory", "refusals", "device_steps",
                                      "capture"])
def test_scenario(stand_in, scenario):
    p = subprocess.run([sys.executable, os.path.join(HERE, "host_side4.py"), stand_in, scenario],
                       capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.endswith("ok\n"), p.stdout[-2000:] + p.stderr[-2000:]
