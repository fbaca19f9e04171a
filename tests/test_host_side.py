"""The library's host side without a device: its own checks, plans and error paths over a stand-in HIP
runtime (host_hip.cpp), each scenario of host_side.py in a process of its own."""

import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def stand_in(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host_hip") / "host_hip.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17",
                    os.path.join(HERE, "host_hip.cpp"), "-o", so], check=True, timeout=120)
    return so


def run(stand_in, scenario):
    p = subprocess.run([sys.executable, os.path.join(HERE, "host_side.py"), stand_in, scenario],
                       capture_output=True, text=True, timeout=120)
    assert p.returncode == 0 and p.stdout.endswith("ok\n"), p.stdout[-2000:] + p.stderr[-2000:]


def test_no_exception_leaves_an_entry_point(stand_in):
    run(stand_in, "host_memory")


def test_a_step_without_device_memory_is_none(stand_in):
    run(stand_in, "device_memory")


def test_shared_plans_that_do_not_fit_the_work_area_are_read_apart(stand_in):
    run(stand_in, "shared_work_area")


def test_planning_spans_costs_no_more_than_rows(stand_in):
    run(stand_in, "plan_time")


def test_key_counts_beyond_the_kernels_are_refused(stand_in):
    run(stand_in, "most_keys")


def test_rows_and_keys_before_the_first_are_refused(stand_in):
    run(stand_in, "rows_before_the_first")
