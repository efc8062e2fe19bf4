"""Regions that measure at different levels: tests/cpp/test_placement_levels.cpp."""
import os
import subprocess


def test_regions_at_different_levels(tmp_path):
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "t")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Wextra", "-o", exe, os.path.join(here, "cpp", "test_placement_levels.cpp")],
                   check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "all checks passed" in r.stdout, r.stdout + r.stderr
