"""The host side of the operators without a GPU: tests/cpp/test_ops_host.cpp, one of its tests to a process."""
import os
import subprocess

import pytest

from tests.test_gpu_ops_plans import WAYS

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_ops_host.bin")
NAMES = ["addresses_are_named", "handles_load_the_operators", "loads_the_operators_when_they_are_used", "optimizers_do_without_the_operators"]


def test_all_are_run():
    assert subprocess.run([BIN], capture_output=True, text=True).stdout.split() == sorted(NAMES)


@pytest.mark.parametrize("name", NAMES)
def test_host_side(name):
    r = subprocess.run([BIN, name], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr


# ---- what the GPU tests of the gradient run: a change of a rule must not empty them ------------

TYPES = {"f32": 0, "bf16": 1, "f64": 2, "f16": 3}


def plan(n, rows, cols, dtype, gtype, accumulate):
    """[(kernel, {what: number})] of a gradient."""
    r = subprocess.run([BIN, "plan"] + [str(int(k)) for k in (n, rows, cols, TYPES[dtype], TYPES[gtype], accumulate)],
                       capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    out = []
    for line in r.stdout.splitlines():
        name, _, _, _, *rest = line.split()
        out.append((name, {k: int(v) for k, v in zip(rest[::2], rest[1::2])}))
    return out


@pytest.mark.parametrize("way", list(WAYS))
def test_ways_of_the_gpu_tests(way):
    batch, seq, rows, kernels = WAYS[way]
    names = [name for name, _ in plan(batch * seq, rows, 136, "f32", "f32", True)]
    assert sorted(set(names)) == sorted(kernels)
