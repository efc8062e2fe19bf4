"""The host side of the operators without a GPU: tests/cpp/test_ops_host.cpp, one of its tests to a process."""
import os
import subprocess

import pytest

from tests.test_gpu_ops_plans import PIECES, TILES, WAYS

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


@pytest.mark.parametrize("case,want", PIECES, ids=lambda c: str(c[0]))
def test_pieces_of_the_gpu_tests(case, want):
    n, rows, cols, dtype, gtype, _, _ = case
    for accumulate in (False, True):
        launches = plan(n, rows, cols, dtype, gtype, accumulate)
        a = dict(launches)[[name for name, _ in launches if "_sum_" in name][0]]
        b = dict(launches)[[name for name, _ in launches if "_join_" in name][0]]
        assert (a["piece"], a["lanes"], a["slabs"], b["edges"]) == want


def test_pieces_of_the_gpu_tests_are_of_every_length_in_both_shapes():
    assert {(p[0], p[1] == 64) for _, p in PIECES} >= {(16, True), (32, True), (64, True), (16, False), (32, False), (64, False)}
    assert any(p[1] == 64 and p[3] > 1 and c[1] >= 2000 for c, p in PIECES)


@pytest.mark.parametrize("case,want", TILES, ids=lambda c: str(c[0]))
def test_tiles_of_the_gpu_tests(case, want):
    hist = [a for name, a in plan(*case, 4, "f32", "f32", False) if name == "nbo_order_hist"]
    assert (hist[0]["tiles"], len(hist)) == want and want[0] > 64 and want[0] % 64


@pytest.mark.parametrize("way", list(WAYS))
def test_ways_of_the_gpu_tests(way):
    batch, seq, rows, kernels = WAYS[way]
    names = [name for name, _ in plan(batch * seq, rows, 136, "f32", "f32", True)]
    assert sorted(set(names)) == sorted(kernels)
