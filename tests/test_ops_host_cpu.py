"""The host side of the operators without a GPU: tests/cpp/test_ops_host.cpp, one of its tests to a process."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_ops_host.bin")
NAMES = ["addresses_are_named", "handles_load_the_operators", "loads_the_operators_when_they_are_used", "optimizers_do_without_the_operators"]


def test_all_are_run():
    assert subprocess.run([BIN], capture_output=True, text=True).stdout.split() == sorted(NAMES)


@pytest.mark.parametrize("name", NAMES)
def test_host_side(name):
    r = subprocess.run([BIN, name], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
