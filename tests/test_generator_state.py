"""The dropout generator's state in the Trainer's tail and in checkpoints: what a checkpoint holds is what
the next mask is drawn with, whoever moved the generator."""
import copy
import dataclasses
import pickle

import pytest

from nabla_amd import checkpoint as ck
from nabla_amd import ops
from nabla_amd.trainer import TrainerTail


class FakeRng:
    """A DropoutRng on the host."""

    def __init__(self, seed, step):
        self.at = ops.DropoutRngState(seed, step)

    def state(self):
        return dataclasses.replace(self.at)

    def load_state(self, state):
        self.at = dataclasses.replace(state)

    def advance(self, steps=1):
        self.at.step = (self.at.step + steps) % (1 << 64)


class FakeOptimizer:
    def fused_step(self, *a, **k):
        pass

    def meta_pairs(self):
        return []

    def load_meta_pairs(self, m):
        pass


def tail_of(rng):
    return TrainerTail(FakeOptimizer(), []).with_rng(rng)


def written(tmp_path, state):
    path = str(tmp_path / "meta.txt")
    ck.write_meta(path, FakeOptimizer(), None, None, state)
    return ck.read_meta(path, FakeOptimizer())[1]


def test_checkpoint_has_the_step_of_a_generator_that_others_advance(tmp_path):
    rng = FakeRng(9, 100)
    tail = tail_of(rng)
    tail.after_backward([])
    rng.advance(5)  # a replayed graph that holds the advance, or the program itself
    assert tail.state.rng_state == 106 and written(tmp_path, tail.state).rng_state == 106
    rng.load_state(ops.DropoutRngState(9, 40))
    assert written(tmp_path, tail.state).rng_state == 40
    tail.after_backward([])
    assert written(tmp_path, tail.state).rng_state == 41 == rng.at.step


def test_a_state_that_is_put_in_place_moves_the_generator():
    rng = FakeRng(9, 100)
    tail = tail_of(rng)
    first = tail.state
    state = ck.TrainState(epoch=2, step=3, rng_state=50)
    tail.state = state  # as set_state does
    assert tail.state is state and rng.at.step == 50
    tail.after_backward([])
    assert state.rng_state == 51 and state.step == 4
    assert first.rng_state == 100  # (what is no longer the tail's keeps the number it had)
    rng.advance()
    assert first.rng_state == 100 and state.rng_state == 52
    state.rng_state = 7
    assert rng.at == ops.DropoutRngState(9, 7)
    tail.set_state(ck.TrainState())  # without a step: the generator's own
    assert rng.at.step == 7 == tail.state.rng_state
    other = FakeRng(3, 0)
    tail.with_rng(other)  # a new generator goes on from the state
    assert other.at == ops.DropoutRngState(3, 7)


def test_states_are_values_when_copied():
    rng = FakeRng(9, 100)
    tail = tail_of(rng)
    live = tail.state
    copies = [copy.copy(live), copy.deepcopy(live), pickle.loads(pickle.dumps(live)), dataclasses.replace(live)]
    assert dataclasses.asdict(live)["rng_state"] == 100
    for c in copies:
        assert c == live and type(c) is ck.TrainState
    rng.advance()
    assert live.rng_state == 101 and all(c.rng_state == 100 and c != live for c in copies)
    plain = ck.TrainState(1, 2, 3, 4)
    assert pickle.loads(pickle.dumps(plain)) == plain == ck.TrainState(epoch=1, step=2, grad_accum=3, rng_state=4)
    assert ck.TrainState().rng_state is None


@pytest.mark.gpu
def test_checkpoint_after_replays_of_a_graph_that_advances_the_generator(gpu, tmp_path):
    """Forward, backward and the advance captured, replayed three times: a resumed run draws the mask that the
    fourth replay would."""
    import torch

    from nabla_amd import _lib

    lib, s = _lib.load(), torch.cuda.Stream()
    x, y = torch.ones(64, 257, device="cuda:0"), torch.empty(64, 257, device="cuda:0")
    rng = ops.DropoutRng(77, 5)
    tail = tail_of(rng)
    torch.cuda.synchronize()
    _lib.check(lib.nbo_set_stream(s.cuda_stream))
    try:
        with torch.cuda.stream(s):
            ops.dropout(x, 0.5, rng, 1, y)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                ops.dropout(x, 0.5, rng, 1, y)
                rng.advance()
            for _ in range(3):
                g.replay()
            state = written(tmp_path, tail.state)
            assert state.rng_state == 8
            fresh = ops.DropoutRng(77, 0)
            tail_of(fresh).set_state(state)
            z = torch.empty_like(y)
            last = y.clone()
            ops.dropout(x, 0.5, fresh, 1, z)
            g.replay()
            s.synchronize()
            assert torch.equal(y, z) and not torch.equal(last, y)
    finally:
        _lib.check(lib.nbo_set_stream(None))


# ---- the seed ------------------------------------------------------------------------------


def test_checkpoint_carries_the_seed(tmp_path):
    """A run that is resumed with a generator of another seed draws the first one's masks."""
    tail = tail_of(FakeRng((1 << 64) - 9, 100))
    tail.after_backward([])
    state = written(tmp_path, tail.state)
    assert (state.rng_state, state.rng_seed) == (101, (1 << 64) - 9)
    assert "rng.state=101\nrng.seed=18446744073709551607\n" in (tmp_path / "meta.txt").read_text()
    for attach_first in (True, False):
        rng = FakeRng(5, 0)
        resumed = tail_of(rng) if attach_first else TrainerTail(FakeOptimizer(), [])
        resumed.set_state(copy.copy(state))
        resumed.with_rng(rng)
        assert rng.at == ops.DropoutRngState((1 << 64) - 9, 101)
        resumed.with_rng(FakeRng(6, 0))  # another generator on purpose: its own seed
        assert resumed.state.rng_seed == 6 and resumed.state.rng_state == 101


def test_checkpoints_without_a_seed_are_read_and_written_as_before(tmp_path):
    state = written(tmp_path, ck.TrainState(1, 2, 3, 4))
    assert state == ck.TrainState(1, 2, 3, 4) and state.rng_seed is None
    assert "rng.seed" not in (tmp_path / "meta.txt").read_text()
    rng = FakeRng(5, 0)
    tail_of(rng).set_state(state)
    assert rng.at == ops.DropoutRngState(5, 4)


def test_cpp_side_reads_and_writes_the_seed(tmp_path):
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "t.cpp"
    src.write_text(r"""
#include "nabla_checkpoint.hpp"
using namespace nabla::optim;
namespace nabla { namespace optim {
struct Opt {}; // found by its namespace
Pairs meta_pairs_of(const Opt &) { return {}; }
void load_meta_pairs_into(Opt &, const MetaMap &) {}
} }
int main(int, char **argv)
{
    Opt o;
    const MetaContents in = read_meta(argv[1], o);
    write_meta(argv[2], o, nullptr, nullptr, in.state);
    return 0;
}
""")
    libdir = os.path.join(root, "nabla_amd")
    r = subprocess.run(["g++", "-O0", "-std=c++17", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                        "-I", os.path.join(root, "include"), "-o", str(tmp_path / "t"), str(src), "-L", libdir,
                        "-l:libnabla_optim.so", f"-Wl,-rpath,{libdir}", "-Wl,-rpath,/opt/rocm/lib"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    for k, state in enumerate([ck.TrainState(1, 2, 3, 4, (1 << 64) - 9), ck.TrainState(1, 2, 3, 4), ck.TrainState(1, 2, 3)]):
        written(tmp_path, state)
        out = tmp_path / f"out{k}.txt"
        assert subprocess.run([str(tmp_path / "t"), str(tmp_path / "meta.txt"), str(out)]).returncode == 0
        assert out.read_text() == (tmp_path / "meta.txt").read_text()
