"""The operators on the GPU where their plan decides what runs: captures, long pieces, many tiles."""
import os
import subprocess
import sys

import pytest
import torch

from nabla_amd import _lib, ops
from nabla_amd import optim as nb
from tests.test_gpu_ops import DEV, assert_within, check_grad, kept, rand_ids, randn, rounding

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_first_operator_of_a_process_inside_a_capture(gpu):
    """Its code object is loaded then; the graph holds the lookup alone."""
    code = r"""
import torch
from nabla_amd import _lib, ops
table = torch.randn(50, 33, device="cuda:0")
ids = torch.randint(0, 50, (70,), device="cuda:0")
out = torch.zeros(70, 33, device="cuda:0")
_lib.init()
s = torch.cuda.Stream()
torch.cuda.synchronize()
_lib.check(_lib.load().nbo_set_stream(s.cuda_stream))
with torch.cuda.stream(s):
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        ops.embedding(table, ids, out)
    for k in range(3):
        table.add_(1.0)
        out.zero_()
        g.replay()
        s.synchronize()
        assert torch.equal(out, table[ids]), k
_lib.check(_lib.load().nbo_set_stream(None))
print("captured ok")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100, cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=ROOT))
    assert r.returncode == 0 and "captured ok" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]


# ---- a training step, by each of the gradient's ways ------------------------------------------

# (sequences, their length, rows of the token table): what runs between the ids and the gradient
WAYS = {
    "direct": (3, 130, 700, ["nbo_embed_direct_f32"]),
    "range": (3, 500, 700, ["nbo_order_range", "nbo_embed_sum_f32", "nbo_embed_join_f32"]),
    "split": (3, 3000, 700, ["nbo_order_split", "nbo_order_merge", "nbo_embed_sum_f32", "nbo_embed_join_f32"]),
    "radix": (3, 3000, 530_000, ["nbo_order_hist", "nbo_order_scan", "nbo_order_scatter", "nbo_embed_sum_f32",
                                 "nbo_embed_join_f32"]),
}


class Block:
    """dropout(2 wte[tokens] + wpe[positions]) and its gradients, next to an AdamW over both tables."""

    def __init__(self, seed, way):
        self.batch, self.seq, self.rows, self.kernels = WAYS[way]
        self.cols, self.n = 136, self.batch * self.seq
        self.params = [randn(self.rows, self.cols, "f32", seed), randn(self.seq, self.cols, "f32", seed + 1)]
        self.grads = [torch.zeros_like(p) for p in self.params]
        self.tokens = rand_ids(self.n, self.rows, seed + 2, 0.1, True).reshape(self.batch, self.seq)
        self.positions = torch.arange(self.seq, device=DEV, dtype=torch.int32).repeat(self.batch)
        self.target = randn(self.n, self.cols, "f32", seed + 3)
        self.x, self.dx = torch.empty_like(self.target), torch.empty_like(self.target)
        self.ws = ops.EmbeddingWorkspace(self.n, self.cols)
        self.rng = ops.DropoutRng(seed, 17)
        self.opt = nb.AdamW.new(1e-2, [tuple(p.shape) for p in self.params])
        self.plist, self.glist = nb.TensorList(self.params), nb.TensorList(self.grads)
        self.tokens_grad = nb.TensorList(self.grads[:1])

    def gradients(self):
        ops.embedding(self.params[1], self.positions, self.x)
        ops.embedding(self.params[0], self.tokens, self.x, scale=2.0, add=self.x)
        ops.dropout(self.x, 0.2, self.rng, 4, self.x)
        torch.sub(self.x, self.target, out=self.dx)  # d/dx of half the squared distance
        ops.dropout_grad(self.dx, 0.2, self.rng, 4, self.dx)
        ops.embedding_grad(self.dx, self.positions, self.grads[1], self.ws)  # fresh: the positions' table is cleared
        ops.embedding_grad(self.dx, self.tokens, self.grads[0], self.ws, scale=2.0, accumulate=True)
        self.rng.advance()

    def step(self):
        self.gradients()
        self.opt.step(self.plist, self.glist)  # (no norm pass: its scratch is one for the whole library)
        nb.zero_grad(self.tokens_grad)

    def state(self):
        return [self.x, self.dx] + self.grads + self.params + [self.opt.read_state(k) for k in ("m0", "v0", "m1", "v1")]


def launched(kernels, call):
    """How often each kernel runs in call()."""
    import ctypes as C

    lib, counts = _lib.load(), {}
    _lib.check(lib.nbo_profile_enable(1))
    try:
        call()
        for k in kernels:
            n, ms = C.c_uint64(0), C.c_double(0)
            _lib.check(lib.nbo_profile_read(k.encode(), C.byref(n), C.byref(ms)))
            counts[k] = n.value
    finally:
        _lib.check(lib.nbo_profile_enable(0))
    return counts


@pytest.mark.parametrize("way", list(WAYS))
def test_gradients_of_the_input_block_against_autograd(gpu, way):
    """One step's gradients against torch's autograd in f64 on the CPU."""
    b = Block(5, way)
    wte, wpe = (p.double().cpu().requires_grad_() for p in b.params)
    keep, thr = kept(b.n * b.cols, 5, 17, 4, 0.2)
    factor = keep.reshape(b.n, b.cols).cpu().double() * (65536.0 / (65536 - thr))
    ids = b.tokens.reshape(-1).cpu()
    ok = (ids >= 0) & (ids < b.rows)
    rows, at = ids.clamp(0, b.rows - 1), b.positions.long().cpu()
    twice, target = 2.0 * ok.double()[:, None], b.target.cpu().double()
    y = (wpe[at] + twice * wte[rows]) * factor
    (0.5 * (y - target) ** 2).sum().backward()
    counts = launched(b.kernels, b.gradients)
    assert all(counts.values()), counts
    assert b.rng.state().step == 18
    with torch.no_grad():  # what a term's roundings, some ten, are relative to
        size = factor * (factor * (wpe[at].abs() + twice * wte[rows].abs()) + target.abs())
    for got, want, where, scale in ((b.grads[0], wte.grad, rows, twice), (b.grads[1], wpe.grad, at, torch.ones_like(twice))):
        terms = torch.zeros(len(want), 1, dtype=torch.float64).index_add_(0, where, scale.clamp(max=1.0))
        bound = (terms + 10) * 2.0 ** -24 * (1 + 2 ** -10) * torch.zeros_like(want).index_add_(0, where, scale * size)
        assert ((got.double().cpu() - want).abs() <= bound).all()
        assert ((got.cpu() != 0) == (want != 0)).all()


@pytest.mark.parametrize("ways", [("direct", "direct"), ("range", "range"), ("split", "split"), ("range", "split"),
                                  ("radix", "split")], ids="-".join)
def test_training_steps_replay_from_two_graphs_on_two_streams(gpu, ways):
    """Forward, backward, optimizer step and the generator's advance, captured once: every replay is an eager
    step of a twin, bit for bit.  Two graphs, each with its own workspace, are replayed at the same time."""
    lib = _lib.load()
    twins = [Block(5, ways[0]), Block(6, ways[1])]
    blocks = [Block(5, ways[0]), Block(6, ways[1])]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    torch.cuda.synchronize()
    try:
        for b, s in zip(blocks, streams):
            _lib.check(lib.nbo_set_stream(s.cuda_stream))
            with torch.cuda.stream(s):
                b.step()
                s.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    b.step()
                s.synchronize()
                graphs.append(g)
    finally:
        _lib.check(lib.nbo_set_stream(None))
    torch.cuda.synchronize()
    for t in twins:
        counts = launched(t.kernels, t.step)
        assert all(counts.values()), counts
    for replay in range(4):
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                if replay % 2:
                    s.synchronize()
        for t in twins:  # eager work between and beside the replays
            t.step()
        torch.cuda.synchronize()
        for b, t in zip(blocks, twins):
            assert b.rng.state() == t.rng.state() and b.rng.state().step == 19 + replay
            for k, (got, want) in enumerate(zip(b.state(), t.state())):
                assert torch.equal(got, want), (replay, k)


@pytest.mark.parametrize("way", list(WAYS))
def test_training_goes_on_from_a_checkpoint(gpu, tmp_path, way):
    """Three micro-batches through TrainerTail, saved after the first and resumed with fresh objects (the
    generator with another seed): the same masks, gradients and parameters."""
    from nabla_amd import checkpoint as ck
    from nabla_amd.trainer import TrainerTail

    def micro_batch(b, tail):
        ops.embedding(b.params[0], b.tokens, b.x)
        ops.dropout(b.x, 0.3, b.rng, 2, b.x)
        torch.sub(b.x, b.target, out=b.dx)
        ops.dropout_grad(b.dx, 0.3, b.rng, 2, b.dx)
        ops.embedding_grad(b.dx, b.tokens, b.grads[0], b.ws)
        tail.after_backward(b.grads)

    a = Block(5, way)
    ta = TrainerTail(a.opt, a.params).with_rng(a.rng).with_grad_clip(1.0)
    micro_batch(a, ta)
    names = ["wte", "wpe"]
    ck.save_checkpoint(str(tmp_path), list(zip(names, a.params)), a.opt, None, None, ta.state, native=True)
    b = Block(5, way)
    _, state, _ = ck.load_checkpoint(str(tmp_path), b.opt, into=list(zip(names, b.params)))
    b.rng = ops.DropoutRng(99, 0)
    tb = TrainerTail(b.opt, b.params).with_rng(b.rng).with_grad_clip(1.0)
    tb.set_state(state)
    for _ in range(2):
        micro_batch(a, ta)
        micro_batch(b, tb)
        assert torch.equal(a.x, b.x) and a.rng.state() == b.rng.state()
        assert torch.equal(a.params[0], b.params[0]) and torch.equal(a.grads[0], b.grads[0])


# ---- pieces of every length, many boundaries, many tiles ---------------------------------------

# (ids, rows, columns, types, hot ids, padding) and what the plan makes of them: (ids per piece, lanes that work on
# one, waves side by side, boundaries to a workgroup of the join)
PIECES = [
    ((65537, 300, 2056, "f16", "f16", False, 0.0), (64, 64, 5, 2)),
    ((65537, 3000, 2056, "bf16", "f32", True, 0.1), (64, 64, 5, 2)),
    ((65537, 2000, 1030, "f64", "f64", True, 0.0), (64, 64, 9, 3)),
    ((131073, 20000, 4104, "bf16", "bf16", True, 0.0), (64, 64, 9, 5)),
    ((40001, 300, 2056, "bf16", "bf16", False, 0.0), (32, 64, 5, 2)),
    ((40001, 9000, 2056, "f16", "f32", True, 0.2), (32, 64, 5, 2)),
    ((20011, 900, 2056, "f32", "f32", True, 0.0), (32, 64, 9, 2)),
    ((20011, 900, 2050, "bf16", "bf16", True, 0.1), (16, 64, 5, 2)),
    ((600001, 3000, 200, "bf16", "bf16", True, 0.0), (64, 32, 1, 3)),
    ((600001, 70000, 200, "f16", "f32", False, 0.1), (64, 32, 1, 3)),
    ((300001, 3000, 200, "bf16", "bf16", True, 0.0), (32, 32, 1, 3)),
    ((300001, 9000, 61, "f32", "f32", True, 0.3), (16, 16, 1, 5)),
    ((1200001, 50000, 24, "bf16", "bf16", True, 0.0), (16, 4, 1, 19)),
    ((17000001, 40000, 3, "f16", "f16", True, 0.0), (64, 1, 1, 64)),
]


def check_long_grad(dy, ids, grad, ws, scale, accumulate, what):
    """check_grad with the sums of the definition on the CPU: on the GPU, torch's additions of a million f64 rows to
    a few hot ones take seconds."""
    rows, before = grad.shape[0], grad.clone()
    at = torch.nonzero((ids >= 0) & (ids < rows))[:, 0]
    i, x = ids[at].long().cpu(), dy[at].double().cpu()
    total = torch.zeros(rows, grad.shape[1], dtype=torch.float64).index_add_(0, i, x).to(DEV)
    size = torch.zeros(rows, grad.shape[1], dtype=torch.float64).index_add_(0, i, x.abs()).to(DEV)
    m = torch.bincount(i, minlength=rows).double().to(DEV)[:, None]
    want = scale * total + (before.double() if accumulate else 0.0)
    ops.embedding_grad(dy, ids, grad, ws, scale=scale, accumulate=accumulate)
    u, h, tiny = rounding(grad.dtype)
    # m - 1 additions in some order, the factor and the product, the sum with what was there; the f64 sums' own
    slack = ((m * u / (1 - m * u) + 3 * u + m * 2.0 ** -52) * abs(scale) * size + u * want.abs()) * (1 + 2 ** -20)
    assert_within(grad, want, slack + h * (want.abs() + slack) + tiny, what)
    rest = m[:, 0] == 0
    assert torch.equal(grad[rest], before[rest] if accumulate else torch.zeros_like(before[rest])), what
    first = grad.clone()
    grad.copy_(before)
    ops.embedding_grad(dy, ids, grad, ws, scale=scale, accumulate=accumulate)
    assert torch.equal(first, grad), what + ": another run gives other bits"


@pytest.mark.parametrize("case", [c for c, _ in PIECES], ids=lambda c: f"{c[0]}-{c[1]}x{c[2]}-{c[3]}-{c[4]}")
def test_embedding_grad_over_whole_pieces(gpu, case):
    """Tokens in every place of a piece: rows that fill it, begin and end in it, span many."""
    n, rows, cols, dtype, gtype, hot, pad = case
    ws = ops.EmbeddingWorkspace(n, cols)
    ids = rand_ids(n, rows, 3, pad, hot)
    dy = randn(n, cols, dtype, 1)
    check = check_long_grad if n > 1 << 19 else check_grad
    check(dy, ids, randn(rows, cols, gtype, 2), ws, 1.5, True, "accumulated")
    ids[n // 3:n // 3 + 200] = rows - 1  # a row of some pieces beside the others
    check(dy, ids, randn(rows, cols, gtype, 2), ws, 1.0, False, "fresh")


# (ids, rows): radix passes over more tiles than a wave has lanes; tiles and passes
TILES = [((300001, 600011), (74, 2)), ((530000, (1 << 21) + 5), (130, 3)), ((262145, 1 << 20), (65, 3))]


@pytest.mark.parametrize("case", [c for c, _ in TILES], ids=lambda c: f"{c[0]}-{c[1]}")
def test_embedding_grad_by_radix_passes_over_many_tiles(gpu, case):
    n, rows = case
    ws = ops.EmbeddingWorkspace(n, 4)
    ids = rand_ids(n, rows, 3, 0.05)
    ids[::7] = rows - 1
    ids[3::11] = 0
    check_long_grad(randn(n, 4, "f32", 1), ids, randn(rows, 4, "f32", 2), ws, 1.0, False, "fresh")
    check_long_grad(randn(n, 3, "f16", 1), rand_ids(n, rows, 4, 0.1, True, torch.int32), randn(rows, 3, "f16", 2), ws, 1.0,
                    True, "accumulated")


# ---- the generator ----------------------------------------------------------------------------

# counter, key and result of Philox4x32-10, as its authors publish them with their library (known answers)
KNOWN = [((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
         ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
          (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]


@pytest.mark.parametrize("known", KNOWN, ids=["zeros", "pi"])
def test_known_answers_of_the_generator(gpu, known):
    """Each 16 bits of the result from the masks: an element is kept at the rate that they are and dropped at the
    next."""
    (block, site, low, high), key, words = known
    cols = 8 if block == 0 else 1 << 27
    rows = block * 8 // cols + 1
    if torch.cuda.mem_get_info(DEV)[0] < rows * cols * 4 + (1 << 30):
        pytest.skip("needs 20 GB of free device memory")
    x = torch.ones(rows, cols, device=DEV, dtype=torch.bfloat16)
    out = torch.empty_like(x)
    rng = ops.DropoutRng(key[0] | key[1] << 32, low | high << 32)
    halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
    for j, h in enumerate(halves):
        for thr in (h, h + 1):
            ops.dropout(x, thr / 65536, rng, site, out)
            assert bool(out.reshape(-1)[block * 8 + j] != 0) == (h >= thr), (j, h, thr)
