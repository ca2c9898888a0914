"""The walk down sampled trees, on the CPU: a thread for each lane, against a plain
walk, and no sum that is written while another wave may still read it."""

import subprocess
from pathlib import Path

TESTS = Path(__file__).resolve().parent


def test_lanes_take_the_same_steps_and_share_in_order(tmp_path):
    exe = tmp_path / "walk_lanes"
    subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "-I", str(TESTS.parent / "kernrelay_amd" / "csrc"),
                    str(TESTS / "walk_lanes.cpp"), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.splitlines()[-1] == "ok", r.stdout[-2000:]
