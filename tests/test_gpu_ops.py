"""The operators of include/nabla_ops.h on the GPU, against their definitions in 64 bits.

Tolerances are arithmetic, not measurements: u = 2^-24 is the rounding of an f32 operation (2^-53 of an
f64 one), h = eps / 2 the rounding to the stored type, 2^-25 half of f16's smallest step.
"""
import gc

import numpy as np
import pytest
import torch

from nabla_amd import _lib, ops
from nabla_amd import optim as nb

pytestmark = pytest.mark.gpu

T = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "f64": torch.float64}
DEV = "cuda:0"


def rounding(dtype):
    """(unit of the arithmetic, half step of the stored type relative to a value, half of its smallest step)"""
    u = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}.get(dtype, 0.0)
    return u, torch.finfo(dtype).eps / 2, tiny


def rand_ids(n, rows, seed, pad=0.0, hot=False, dtype=torch.int64):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if hot:  # log-uniform: a few rows hold most tokens
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        ids = (((rows + 1.0) ** u) - 1).long().clamp_(0, rows - 1)
    else:
        ids = torch.randint(0, rows, (n,), generator=g, device=DEV)
    bad = torch.tensor([-1, rows, -2 ** 31, 2 ** 31 - 1], device=DEV)
    which = torch.randint(0, 4, (n,), generator=g, device=DEV)
    ids = torch.where(torch.rand(n, generator=g, device=DEV) < pad, bad[which], ids)
    return ids.to(dtype)


def randn(rows, cols, dtype, seed, stride=None):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    x = torch.empty(rows, stride or cols, device=DEV, dtype=torch.float32).normal_(generator=g)
    return x.to(T[dtype])[:, :cols]


def assert_within(got, want, bound, what=""):
    err = (got.double() - want).abs()
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert not torch.isnan(err).any(), what
    assert worst <= 0.0, f"{what}: {int((err > bound).sum())} of {err.numel()} beyond the bound, worst by {worst}"


# ---- embedding -----------------------------------------------------------------------------

PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f64", "f64"), ("f32", "bf16"), ("f32", "f16")]
SIZES = [(1, 1, 1), (5, 3, 7), (50, 8, 1), (64, 1, 513), (300, 64, 1025), (1000, 771, 300), (40, 4100, 33), (7, 9001, 3)]


def check_embedding(table, ids, out, scale, add):
    rows = table.shape[0]
    i = ids.reshape(-1).long()
    ok = ((i >= 0) & (i < rows))[:, None]
    w = torch.where(ok, table[torch.where(ok[:, 0], i, 0)].double(), 0.0)
    before = add.double().clone() if add is not None else torch.zeros_like(w)
    ops.embedding(table, ids, out, scale=scale, add=add)
    term = scale * w
    want = before + term
    u, h, tiny = rounding(out.dtype)
    if add is None and scale == 1.0 and out.dtype == table.dtype:
        assert torch.equal(out.double(), want)  # nothing is rounded
    else:
        # the factor's and the product's rounding, the sum's, the stored value's
        slack = (2 * u * term.abs() + u * want.abs()) * (1 + 2 ** -20)
        assert_within(out, want, slack + h * (want.abs() + slack) + tiny, f"{table.dtype} -> {out.dtype}")


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("pair", PAIRS, ids=lambda p: "-".join(p))
def test_embedding(gpu, pair, size):
    rows, cols, n = size
    table = randn(rows, cols, pair[0], 1)
    for k, (scale, with_add, wide) in enumerate([(1.0, False, True), (45.25, False, False), (0.3, True, True)]):
        ids = rand_ids(n, rows, 10 + k, 0.2, dtype=torch.int64 if wide else torch.int32)
        out = torch.full((n, cols), 7.0, device=DEV, dtype=T[pair[1]])
        add = randn(n, cols, pair[1], 20 + k) if with_add else None
        check_embedding(table, ids, out, scale, add)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("offset,cols", [(0, 40), (1, 40), (3, 37), (5, 600)])
def test_embedding_of_views_writes_nothing_else(gpu, dtype, offset, cols):
    """Strided rows at odd element offsets, in place on the summand, column slices side by side."""
    stride = 2 * cols + 11
    table = randn(90, cols, dtype, 1, stride=cols + 3)
    big = randn(50, stride, dtype, 2)
    before = big.clone()
    ids = rand_ids(50, 90, 3, 0.1)
    left, right = big[:, offset:offset + cols], big[:, offset + cols:offset + 2 * cols]
    check_embedding(table, ids, left, 1.5, right)
    check_embedding(table, ids, right, 0.5, right)  # in place
    rest = torch.ones(stride, dtype=torch.bool, device=DEV)
    rest[offset:offset + 2 * cols] = False
    assert torch.equal(big[:, rest], before[:, rest])


def test_embedding_padding_is_zero_whatever_the_scale(gpu):
    table = torch.full((4, 16), float("inf"), device=DEV)
    ids = torch.tensor([-1, 4, 2 ** 40, -2 ** 63, 2], device=DEV)
    out = torch.full((5, 16), 3.0, device=DEV)
    ops.embedding(table, ids, out, scale=float("nan"))
    assert torch.equal(out[:4], torch.zeros(4, 16, device=DEV)) and torch.isnan(out[4]).all()
    ops.embedding(table[:0], ids, out)  # a table without rows: all padding
    assert torch.equal(out, torch.zeros(5, 16, device=DEV))
    out.fill_(3.0)
    ops.embedding(table, ids[:0], out[:0])  # no tokens
    assert torch.equal(out, torch.full((5, 16), 3.0, device=DEV))


# ---- the gradient --------------------------------------------------------------------------

def check_grad(dy, ids, grad, ws, scale=1.0, accumulate=False, what=""):
    """One call against f64, and again for the same bits."""
    rows = grad.shape[0]
    i = ids.reshape(-1).long()
    at = torch.nonzero((i >= 0) & (i < rows))[:, 0]
    total = torch.zeros(rows, grad.shape[1], device=DEV, dtype=torch.float64)
    size = torch.zeros_like(total)
    total.index_add_(0, i[at], dy[at].double())
    size.index_add_(0, i[at], dy[at].double().abs())
    count = torch.zeros(rows, device=DEV, dtype=torch.float64).index_add_(0, i[at], torch.ones(len(at), device=DEV,
                                                                                               dtype=torch.float64))
    before = grad.clone()
    want = scale * total + (before.double() if accumulate else 0.0)
    ops.embedding_grad(dy, ids, grad, ws, scale=scale, accumulate=accumulate)
    u, h, tiny = rounding(grad.dtype)
    # count - 1 additions in some order, the factor and the product, the sum with what was there
    m = count[:, None]
    gamma = m * u / (1 - m * u)
    slack = ((gamma + 3 * u) * abs(scale) * size + u * want.abs()) * (1 + 2 ** -20)
    # (the f64 sums that stand for the definition are rounded too)
    slack = slack + m * 2.0 ** -52 * abs(scale) * size
    assert_within(grad, want, slack + h * (want.abs() + slack) + tiny, what)
    named = count > 0
    if accumulate:
        assert torch.equal(grad[~named], before[~named]), what + ": rows no id names"
    else:
        assert not grad[~named].any(), what + ": rows no id names"
    first = grad.clone()
    grad.copy_(before)
    ops.embedding_grad(dy, ids, grad, ws, scale=scale, accumulate=accumulate)
    assert torch.equal(first, grad), what + ": another run gives other bits"


GRAD_PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f64", "f64"), ("bf16", "f32"), ("f16", "f32")]


@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 257, 512, 513, 1000, 4097, 8192, 8193, 40000])
@pytest.mark.parametrize("pair", GRAD_PAIRS, ids=lambda p: "-".join(p))
def test_embedding_grad(gpu, pair, n):
    rows, cols = 1201, 72 if n % 2 else 77
    ws = ops.EmbeddingWorkspace(n, cols)
    dy = randn(n, cols, pair[0], n + 1)
    for k, (scale, accumulate, hot, pad, wide) in enumerate([(1.0, False, True, 0.0, True), (0.75, True, True, 0.3, False),
                                                             (3.0, False, False, 0.1, False)]):
        ids = rand_ids(n, rows, 30 + k, pad, hot, torch.int64 if wide else torch.int32)
        grad = randn(rows, cols, pair[1], 40 + k)
        check_grad(dy, ids, grad, ws, scale, accumulate, f"case {k}")


@pytest.mark.parametrize("cols", [1, 2, 3, 5, 7, 8, 9, 31, 64, 100, 255, 256, 257, 511, 512, 513, 1100, 4099])
@pytest.mark.parametrize("pair", [("f32", "f32"), ("f16", "f16"), ("f64", "f64"), ("bf16", "f32")], ids=lambda p: "-".join(p))
def test_embedding_grad_widths(gpu, pair, cols):
    ws = ops.EmbeddingWorkspace(3000, cols)
    for n, accumulate in ((100, True), (3000, False)):
        dy = randn(n, cols, pair[0], n)
        grad = randn(333, cols, pair[1], 5)
        check_grad(dy, rand_ids(n, 333, 6, 0.1, True), grad, ws, 1.0, accumulate, f"{n}")


@pytest.mark.parametrize("n", [512, 1500, 20000])
def test_embedding_grad_of_one_row_and_of_padding_alone(gpu, n):
    """Every token the same (its row spans all pieces), and none at all."""
    cols = 520
    ws = ops.EmbeddingWorkspace(n, cols)
    dy = randn(n, cols, "bf16", 1)
    for accumulate in (False, True):
        for fill in (0, 17, 99, -1, 100):
            ids = torch.full((n,), fill, device=DEV)
            check_grad(dy, ids, randn(100, cols, "f32", 2), ws, 1.0, accumulate, f"all {fill}")
        ids = torch.full((n,), 5, device=DEV)  # two long rows and one token between
        ids[n // 2] = 6
        ids[n // 2 + 1:] = 7
        check_grad(dy, ids, randn(100, cols, "bf16", 2), ws, 1.0, accumulate, "three rows")


@pytest.mark.parametrize("rows,n", [(1, 300), (2, 20000), (255, 20000), (256, 20000), (1023, 20000), (1024, 20000),
                                    ((1 << 20) - 1, 20000), (1 << 20, 20000), ((1 << 21) + 5, 30000), (3_000_017, 5000), (1 << 21, 8192),
                                    ((1 << 21) + 1, 8192), ((1 << 19) - 1, 8193), (1 << 19, 8193),
                                    (1, 140000), (2, 140000), (255, 140001), (256, 140000), (1023, 139999),
                                    (1024, 140000), (50257, 300000)])
def test_embedding_grad_table_sizes(gpu, rows, n):
    """Around the ways to order the ids (key ranges; radix passes for many ids or rows) and the digit widths
    of the passes; the last rows of the table among the ids."""
    ws = ops.EmbeddingWorkspace(n, 4)
    ids = rand_ids(n, rows, 3, 0.05)
    ids[::7] = rows - 1
    ids[3::11] = 0
    check_grad(randn(n, 4, "f32", 1), ids, randn(rows, 4, "f32", 2), ws, 1.0, False, "fresh")
    check_grad(randn(n, 3, "f16", 1), ids.int(), randn(rows, 3, "f16", 2), ws, 1.0, True, "accumulated")


@pytest.mark.parametrize("rows,step,n", [(60000, 256, 700), (60000, 256, 8192), (131072, 256, 8193), (131072, 256, 70000),
                                         (400000, 1024, 30000), (131072, 128, 70000), (1900000, 2048, 5000)])
def test_embedding_grad_of_ids_that_fall_into_one_range(gpu, rows, step, n):
    """Ids a power of two apart: one workgroup of the order has all of them, the others none."""
    ids = rand_ids(n, (rows - 1) // step + 1, 5, hot=True) * step + step // 2
    ids = torch.where(torch.arange(n, device=DEV) % 13 == 0, -1, ids)
    check_grad(randn(n, 20, "bf16", 1), ids, randn(rows, 20, "bf16", 2), ops.EmbeddingWorkspace(n, 20))


def test_embedding_grad_does_not_read_padded_rows(gpu):
    for n in (200, 2000, 20000):
        ws = ops.EmbeddingWorkspace(n, 24)
        ids = rand_ids(n, 50, 1, 0.4)
        dy = randn(n, 24, "f32", 2)
        padded = (ids < 0) | (ids >= 50)
        clean = dy.clone()
        dy[padded] = float("nan")
        a, b = torch.empty(50, 24, device=DEV), torch.empty(50, 24, device=DEV)
        ops.embedding_grad(dy, ids, a, ws)
        ops.embedding_grad(clean, ids, b, ws)
        assert torch.equal(a, b)
        # inf and NaN in rows that count reach their own row of the table and no other
        clean[(~padded).nonzero()[0, 0]] = float("inf")
        ops.embedding_grad(clean, ids, a, ws)
        hit = ids[(~padded).nonzero()[0, 0]].item()
        assert torch.isinf(a[hit]).all() and torch.equal(a[torch.arange(50, device=DEV) != hit],
                                                         b[torch.arange(50, device=DEV) != hit])


@pytest.mark.parametrize("n", [90, 3000])
@pytest.mark.parametrize("pair", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")], ids=lambda p: "-".join(p))
def test_embedding_grad_of_views_writes_nothing_else(gpu, pair, n):
    cols, stride = 75, 190
    ws = ops.EmbeddingWorkspace(5000, 100)
    dy = randn(n, cols, pair[0], 1, stride=cols + 6)
    ids = rand_ids(n, 400, 2, 0.1, True)
    for accumulate in (False, True):
        big = randn(400, stride, pair[1], 3)
        before = big.clone()
        check_grad(dy, ids, big[:, 7:7 + cols], ws, 1.0, accumulate)
        assert torch.equal(big[:, :7], before[:, :7]) and torch.equal(big[:, 7 + cols:], before[:, 7 + cols:])


@pytest.mark.parametrize("rows,cols,stride,dtype", [(65536, 7, 7, "f32"), (65537, 7, 7, "f32"), (70001, 1, 1, "f16"),
                                                    (70001, 3, 5, "f16"), (70001, 1, 2, "f64"), (70000, 1000, 1031, "bf16"),
                                                    (70003, 1031, 1031, "bf16"), (70000, 16, 16, "bf16"), (2000003, 2, 3, "f32"),
                                                    (1966080, 1, 1, "f32"), (1966081, 9, 9, "f16")])
@pytest.mark.parametrize("n", [0, 5, 512, 600])
def test_embedding_grad_clears_large_matrices(gpu, rows, cols, stride, dtype, n):
    """Fresh gradients of matrices that are cleared ahead of the sums, with gaps between the rows and without."""
    big = torch.full((rows, stride), 3.0, device=DEV, dtype=T[dtype])
    ids = rand_ids(n, rows, 2, 0.1)
    if n:
        ids[0], ids[-1] = rows - 1, 0
    check_grad(randn(n, cols, dtype, 1), ids, big[:, :cols], ops.EmbeddingWorkspace(n, cols))
    assert torch.equal(big[:, cols:], torch.full_like(big[:, cols:], 3.0))


def test_embedding_grad_against_differences(gpu):
    """d(sum of c * embedding) / d(table) by central differences in f64: the operator is linear in the
    table, so they are exact up to rounding."""
    rows, cols, n = 6, 5, 40
    table, c = randn(rows, cols, "f64", 1), randn(n, cols, "f64", 2)
    ids = rand_ids(n, rows, 3, 0.2)
    grad, out = torch.empty_like(table), torch.empty(n, cols, device=DEV, dtype=torch.float64)
    ops.embedding_grad(c, ids, grad, ops.EmbeddingWorkspace(n, cols), scale=1.75)

    def loss(t):
        ops.embedding(t, ids, out, scale=1.75)
        return (c * out).sum().item()

    for r in range(rows):
        for k in range(cols):
            e = torch.zeros_like(table)
            e[r, k] = 0.5
            d = loss(table + e) - loss(table - e)
            # 200 terms of at most 1.75 * 4.5 * 4.5 each, all rounded a few times
            assert abs(d - grad[r, k].item()) <= 200 * 36 * 8 * 2.0 ** -53


def test_workspace_limits_are_refused(gpu):
    ws = ops.EmbeddingWorkspace(100, 16)
    grad = torch.zeros(9, 16, device=DEV)
    with pytest.raises(_lib.NablaOptimError, match="the workspace is for 100 of 16"):
        ops.embedding_grad(torch.zeros(101, 16, device=DEV), torch.zeros(101, device=DEV, dtype=torch.int64), grad, ws)
    with pytest.raises(_lib.NablaOptimError, match="the workspace is for 100 of 16"):
        ops.embedding_grad(torch.zeros(4, 17, device=DEV), torch.zeros(4, device=DEV, dtype=torch.int64),
                           torch.zeros(9, 17, device=DEV), ws)
    with pytest.raises(nb.NablaPanic, match="shapes must match"):
        ops.embedding_grad(torch.zeros(4, 15, device=DEV), torch.zeros(4, device=DEV, dtype=torch.int64), grad, ws)
    with pytest.raises(_lib.NablaOptimError, match="overlaps"):
        ops.embedding_grad(grad[:4], torch.zeros(4, device=DEV, dtype=torch.int64), grad, ws)
    with pytest.raises(_lib.NablaOptimError, match="not memory the HIP runtime knows"):
        ops.embedding_grad(torch.zeros(4, 16), torch.zeros(4, device=DEV, dtype=torch.int64), grad, ws)
    with pytest.raises(_lib.NablaOptimError, match="not memory the HIP runtime knows"):
        ops.embedding(grad, torch.zeros(4, dtype=torch.int64), torch.zeros(4, 16, device=DEV))


# ---- dropout -------------------------------------------------------------------------------

def kept(n, seed, step, site, p, first=0):
    """Which of elements first .. first + n - 1 (first a multiple of eight) are kept: numpy, from the
    definition."""
    thr, u = int(65536 * p + 0.5), np.uint64
    blocks = np.arange(first // 8, (first + n + 7) // 8, dtype=u)
    c = [blocks] + [np.full_like(blocks, x) for x in (site, step % 2 ** 32, step // 2 ** 32)]
    k = [seed % 2 ** 32, seed // 2 ** 32]
    low = u(0xFFFFFFFF)
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack(c, axis=1).astype("<u4").view("<u2").reshape(-1)
    return torch.from_numpy(bits[:n] >= thr).to(DEV), thr


def test_known_answer_of_the_generator(gpu):
    """Philox4x32-10 of counter 0 under key 0, as its authors publish it."""
    words = [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    halves = [h for w in words for h in (w & 0xFFFF, w >> 16)]
    u = np.uint64
    for j, h in enumerate(halves):
        for thr in (h, h + 1):
            keep = kept_cpu(thr / 65536)
            assert bool(keep[j]) == (h >= thr), (j, u(h))


def kept_cpu(p):
    return kept(8, 0, 0, 0, p)[0].cpu()


def check_dropout(x, p, rng, site, out, residual, state):
    want_kept, thr = kept(x.numel(), state[0], state[1], site, p)
    want_kept = want_kept.reshape(x.shape)
    before = residual.double().clone() if residual is not None else torch.zeros(x.shape, device=DEV, dtype=torch.float64)
    factor = 65536.0 / (65536 - thr) if thr < 65536 else 0.0
    term = torch.where(want_kept, x.double() * factor, 0.0)
    ops.dropout(x, p, rng, site, out, residual=residual)
    want = before + term
    u, h, tiny = rounding(out.dtype)
    slack = (2 * u * term.abs() + u * want.abs()) * (1 + 2 ** -20)
    assert_within(out, want, slack + h * (want.abs() + slack) + tiny, f"{x.dtype} {tuple(x.shape)} p {p}")
    if residual is None:
        assert not out[~want_kept].any()


@pytest.mark.parametrize("dtype", list(T))
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (1, 8), (3, 3), (1, 255), (5, 257), (64, 768), (33, 1001)],
                         ids=lambda s: "x".join(map(str, s)))
def test_dropout(gpu, dtype, shape):
    seed, step = 0xFEDCBA9876543210, (5 << 32) - 1
    rng = ops.DropoutRng(seed, step)
    for k, (p, with_residual) in enumerate([(0.0, False), (0.1, True), (0.5, False), (1.0, True), (2.0 ** -17, False)]):
        x = randn(*shape, dtype, k)
        residual = randn(*shape, dtype, 50 + k) if with_residual else None
        check_dropout(x, p, rng, 3 + k, torch.full_like(x, 9.0), residual, (seed, step))
    rng.advance()  # the step's low half wraps
    check_dropout(x, 0.3, rng, 0xFFFFFFFF, torch.full_like(x, 9.0), None, (seed, step + 1))


@pytest.mark.parametrize("dtype", list(T))
@pytest.mark.parametrize("cols", [1, 5, 8, 12, 13, 40, 300, 2055, 9000])
def test_dropout_of_views_writes_nothing_else(gpu, dtype, cols):
    """The mask goes by the element's place in the matrix, whatever the strides are."""
    rng = ops.DropoutRng(7, 9)
    stride = 2 * cols + 9
    big = randn(11, stride, dtype, 1)
    before = big.clone()
    x, out = big[:, 1:1 + cols], big[:, 1 + cols:1 + 2 * cols]
    check_dropout(x, 0.4, rng, 2, out, None, (7, 9))
    check_dropout(x, 0.4, rng, 2, out, out, (7, 9))  # onto the residual
    flat = x.contiguous()
    check_dropout(flat, 0.4, rng, 2, flat, None, (7, 9))  # in place
    assert torch.equal(big[:, :1 + cols], before[:, :1 + cols]) and torch.equal(big[:, 1 + 2 * cols:],
                                                                                before[:, 1 + 2 * cols:])


def test_dropped_elements_are_zero_whatever_they_hold(gpu):
    rng = ops.DropoutRng(3)
    x = torch.full((64, 64), float("nan"), device=DEV)
    x[::2] = float("inf")
    out = torch.empty_like(x)
    ops.dropout(x, 0.5, rng, 0, out)
    keep = kept(4096, 3, 0, 0, 0.5)[0].reshape(64, 64)
    assert not out[~keep].any() and not torch.isfinite(out[keep]).any()
    ops.dropout(x, 1.0, rng, 0, out)
    assert not out.any()


def test_dropout_gradient_uses_the_same_mask_and_its_mean_is_kept(gpu):
    rng = ops.DropoutRng(11, 4)
    ones = torch.ones(2000, 512, device=DEV)
    y, dx, other = torch.empty_like(ones), torch.empty_like(ones), torch.empty_like(ones)
    ops.dropout(ones, 0.25, rng, 5, y)
    ops.dropout_grad(ones, 0.25, rng, 5, dx)
    assert torch.equal(y, dx)  # dy = x = 1: the operator is linear, the derivative is the mask times the factor
    # 1.024e6 draws: the mean of kept / (1 - p) is 1 with a deviation of sqrt(p / (1 - p) / n) = 5.7e-4
    assert abs(y.double().mean().item() - 1.0) < 5 * 5.8e-4
    for site, advance in ((6, 0), (5, 1)):
        if advance:
            rng.advance(advance)
        ops.dropout(ones, 0.25, rng, site, other)
        # two independent masks agree in 0.25^2 + 0.75^2 = 0.625 of the places, deviation 4.8e-4
        assert abs((other == y).double().mean().item() - 0.625) < 5 * 4.8e-4


def test_generator_state(gpu):
    rng = ops.DropoutRng((1 << 64) - 1, (1 << 64) - 2)
    assert rng.state() == ops.DropoutRngState((1 << 64) - 1, (1 << 64) - 2)
    rng.advance(3)  # modulo 2^64
    assert rng.state().step == 1
    rng.load_state(ops.DropoutRngState(5, 6))
    assert rng.state() == ops.DropoutRngState(5, 6)
    with pytest.raises(_lib.NablaOptimError, match=r"not in \[0, 1\]"):
        ops.dropout(torch.zeros(4, device=DEV), -0.1, rng, 0, torch.zeros(4, device=DEV))
    with pytest.raises(_lib.NablaOptimError, match=r"not in \[0, 1\]"):
        ops.dropout(torch.zeros(4, device=DEV), float("nan"), rng, 0, torch.zeros(4, device=DEV))
    with pytest.raises(_lib.NablaOptimError, match="overlaps x in part"):
        x = torch.zeros(20, device=DEV)
        ops.dropout(x[:16], 0.1, rng, 0, x[4:])
    with pytest.raises(_lib.NablaOptimError, match="element type"):
        ops.dropout(x, 0.1, rng, 0, torch.zeros(20, device=DEV, dtype=torch.bfloat16))


# ---- beyond 32 bits ------------------------------------------------------------------------

@pytest.mark.parametrize("n", [40, 3000, 20000])
def test_ids_beyond_32_bits_are_padding(gpu, n):
    """Ids whose low halves are rows of the table."""
    rows, cols = 50, 40
    ids = rand_ids(n, rows, 1)
    far = torch.tensor([1 << 32, -(1 << 32), 1 << 62, -(1 << 63)], device=DEV)[torch.arange(n, device=DEV) % 4]
    ids = torch.where(torch.arange(n, device=DEV) % 3 == 0, ids + far, ids)
    table = randn(rows, cols, "f32", 2)
    check_embedding(table, ids, torch.empty(n, cols, device=DEV), 1.0, None)
    check_grad(randn(n, cols, "f32", 3), ids, table, ops.EmbeddingWorkspace(n, cols))


def test_offsets_beyond_32_bits(gpu):
    """Tables, batches and matrices of more than 2^32 elements: their last rows."""
    rows, cols = (1 << 22) + 3, 1032  # 4.3e9 elements, 8.7 GB
    table = torch.zeros(rows, cols, device=DEV, dtype=torch.bfloat16)
    table[-5:] = randn(5, cols, "bf16", 1)
    ids = torch.arange(rows - 5, rows, device=DEV)
    out = torch.empty(5, cols, device=DEV, dtype=torch.bfloat16)
    ops.embedding(table, ids, out)
    assert torch.equal(out, table[-5:])
    # the gradient of those rows, from the last rows of a batch as large
    few = torch.zeros(9, cols, device=DEV, dtype=torch.bfloat16)
    where = torch.full((rows,), -1, device=DEV, dtype=torch.int32)
    where[-5:] = torch.tensor([1, 8, 1, 0, 8], device=DEV, dtype=torch.int32)
    ops.embedding_grad(table, where, few, ops.EmbeddingWorkspace(rows, cols))
    want = torch.zeros(9, cols, device=DEV).index_add_(0, where[-5:], table[-5:].float())
    assert torch.equal(few, want.bfloat16())
    ops.embedding_grad(out, ids, table, ops.EmbeddingWorkspace(5, cols), accumulate=True)
    assert torch.equal(table[-5:].float(), out.float() * 2) and not table[:-5].any()
    # a lookup with as many rows
    ops.embedding(few, where, table)
    assert torch.equal(table[-5:], few[where[-5:].long()]) and not table[:-5].any()
    # dropout of the same matrix, in place: the last elements' mask
    table.fill_(1.0)
    ops.dropout(table, 0.5, ops.DropoutRng(21, 2), 1, table)
    first = (table.numel() - 4096) // 8 * 8
    keep = kept(table.numel() - first, 21, 2, 1, 0.5, first)[0]
    assert torch.equal(table.reshape(-1)[first:].float(), keep.float() * 2)


def test_dropout_of_more_units_than_32_bits(gpu):
    """2^32 units and a few: f64 elements two to a unit, 64 GiB in one run, in place."""
    rows, cols = (1 << 23) + 1, 1024
    n = rows * cols
    gc.collect()
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(DEV)[0] < n * 8 + (1 << 30):
        pytest.skip("needs 65 GiB of free device memory")
    x = torch.ones(rows, cols, device=DEV, dtype=torch.float64)
    ops.dropout(x, 0.5, ops.DropoutRng(21, 2), 1, x)
    x = x.reshape(-1)
    first = n - 4096
    assert torch.equal(x[first:], kept(n - first, 21, 2, 1, 0.5, first)[0].double() * 2)
    assert torch.equal(x[:4096], kept(4096, 21, 2, 1, 0.5)[0].double() * 2)
    del x
    torch.cuda.empty_cache()


# ---- together, as a training step uses them ---------------------------------------------------

class _InputBlock:
    """dropout(wte[tokens] + wpe[positions]) and its gradients, next to an AdamW over both tables."""

    def __init__(self, seed):
        self.rows, self.cols, self.batch, self.seq = 700, 136, 3, 130
        self.n = self.batch * self.seq
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

    def step(self, fused=False):
        ops.embedding(self.params[1], self.positions, self.x)
        ops.embedding(self.params[0], self.tokens, self.x, scale=2.0, add=self.x)
        ops.dropout(self.x, 0.2, self.rng, 4, self.x)
        torch.sub(self.x, self.target, out=self.dx)  # d/dx of half the squared distance
        ops.dropout_grad(self.dx, 0.2, self.rng, 4, self.dx)
        ops.embedding_grad(self.dx, self.tokens, self.grads[0], self.ws, scale=2.0, accumulate=True)
        ops.embedding_grad(self.dx, self.positions, self.grads[1], self.ws, accumulate=True)
        self.rng.advance()
        if fused:
            self.opt.fused_step(self.plist, self.glist, max_norm=1.0, zero_grads=True)
        else:  # (no norm pass: its scratch is one for the whole library)
            self.opt.step(self.plist, self.glist)
            nb.zero_grad(self.glist)

    def state(self):
        return [self.x, self.dx] + self.params + [self.opt.read_state(k) for k in ("m0", "v0", "m1", "v1")]


def test_gradients_of_the_input_block_against_autograd(gpu):
    """One step's gradients against torch's autograd in f64 on the CPU."""
    b = _InputBlock(5)
    wte, wpe = (p.double().cpu().requires_grad_() for p in b.params)
    keep, thr = kept(b.n * b.cols, 5, 17, 4, 0.2)
    factor = keep.reshape(b.n, b.cols).cpu().double() * (65536.0 / (65536 - thr))
    ids = b.tokens.reshape(-1).cpu()
    ok = ((ids >= 0) & (ids < b.rows)).double()[:, None]
    y = (wpe[b.positions.long().cpu()] + 2.0 * ok * wte[ids.clamp(0, b.rows - 1)]) * factor
    (0.5 * (y - b.target.cpu().double()) ** 2).sum().backward()
    grads = []
    b.opt.fused_step = lambda *a, **k: grads.extend(g.double().cpu() for g in b.grads)  # before they are cleared
    b.step(fused=True)
    assert b.rng.state().step == 18
    for got, want in zip(grads, (wte.grad, wpe.grad)):
        # at most 130 terms of magnitude below 60, some ten roundings each: 130 * 60 * (130 + 10) u
        assert (got - want).abs().max().item() <= 130 * 60 * 140 * 2.0 ** -24
        assert ((got != 0) == (want != 0)).all()


def test_training_step_replays_from_a_hip_graph(gpu):
    """Forward, backward, optimizer step and the generator's advance, captured once: every replay is an
    eager step of a twin, bit for bit -- with new masks each time.  Two graphs, each with its own
    workspace, are replayed at the same time on two streams."""
    lib = _lib.load()
    twins = [_InputBlock(5), _InputBlock(6)]
    blocks = [_InputBlock(5), _InputBlock(6)]
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
        t.step()
    for replay in range(4):
        last = [b.x.clone() for b in blocks]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                if replay % 2:
                    s.synchronize()
        for t in twins:  # eager work between and beside the replays
            t.step()
        torch.cuda.synchronize()
        for b, t, before in zip(blocks, twins, last):
            assert b.rng.state() == t.rng.state() and b.rng.state().step == 19 + replay
            for k, (got, want) in enumerate(zip(b.state(), t.state())):
                assert torch.equal(got, want), (replay, k)
            assert not torch.equal((b.x == 0), (before == 0))  # another mask


def test_training_step_with_the_fused_optimizer_replays_from_a_hip_graph(gpu):
    lib = _lib.load()
    b, twin, s = _InputBlock(8), _InputBlock(8), torch.cuda.Stream()
    torch.cuda.synchronize()
    _lib.check(lib.nbo_set_stream(s.cuda_stream))
    try:
        with torch.cuda.stream(s):
            b.step(True)
            twin.step(True)
            s.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                b.step(True)
            for replay in range(3):
                g.replay()
                twin.step(True)
                s.synchronize()
                for k, (got, want) in enumerate(zip(b.state(), twin.state())):
                    assert torch.equal(got, want), (replay, k)
                assert not any(x.any() for x in b.grads)
    finally:
        _lib.check(lib.nbo_set_stream(None))


def test_inputs_on_another_stream(gpu):
    """The library's stream set to the caller's: the operators wait for what that stream has produced."""
    lib = _lib.load()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    _lib.check(lib.nbo_set_stream(s.cuda_stream))
    try:
        with torch.cuda.stream(s):
            table = randn(50000, 512, "f32", 1)
            for _ in range(20):
                table = table * 1.0 + 1.0
            ids = rand_ids(5000, 50000, 2)
            out = torch.empty(5000, 512, device=DEV)
            ops.embedding(table, ids, out)
            want = table[ids]
            s.synchronize()
            assert torch.equal(out, want)
    finally:
        _lib.check(lib.nbo_set_stream(None))


def test_training_goes_on_from_a_checkpoint_with_the_same_masks(gpu, tmp_path):
    """Three micro-batches through TrainerTail, saved after the first and resumed with fresh objects: the
    masks, gradients and parameters of the others are the same bits."""
    from nabla_amd import checkpoint as ck
    from nabla_amd.trainer import TrainerTail

    def micro_batch(b, tail):
        ops.embedding(b.params[0], b.tokens, b.x)
        ops.dropout(b.x, 0.3, b.rng, 2, b.x)
        torch.sub(b.x, b.target, out=b.dx)
        ops.dropout_grad(b.dx, 0.3, b.rng, 2, b.dx)
        ops.embedding_grad(b.dx, b.tokens, b.grads[0], b.ws)
        tail.after_backward(b.grads)

    a = _InputBlock(5)
    ta = TrainerTail(a.opt, a.params).with_rng(a.rng).with_grad_clip(1.0)
    micro_batch(a, ta)
    assert a.rng.state().step == 18 == ta.state.rng_state
    names = ["wte", "wpe"]
    ck.save_checkpoint(str(tmp_path), list(zip(names, a.params)), a.opt, None, None, ta.state)
    b = _InputBlock(5)  # another process: initial values again
    params, state, _ = ck.load_checkpoint(str(tmp_path), b.opt)
    for (name, value), p in zip(params, b.params):
        p.copy_(torch.as_tensor(value).to(p))
    b.rng.load_state(ops.DropoutRngState(5, 0))
    tb = TrainerTail(b.opt, b.params).with_rng(b.rng).with_grad_clip(1.0)
    tb.set_state(state)
    for _ in range(2):
        micro_batch(a, ta)
        micro_batch(b, tb)
        assert torch.equal(a.x, b.x) and a.rng.state() == b.rng.state()
        assert torch.equal(a.params[0], b.params[0]) and torch.equal(a.grads[0], b.grads[0])


def test_cpp_program(gpu):
    import os
    import subprocess

    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_ops.bin")
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "0 failure(s)" in r.stdout, r.stdout + r.stderr


def test_grids_folded_into_two_dimensions(gpu):
    """Launches of more than 2^24 - 1 workgroups are folded; NBO_GRID_X_MAX=7 in the environment (a test
    hook of the runtime) folds every one here, the last grid row partly unused."""
    import os
    import subprocess
    import sys

    code = r"""
import torch
from nabla_amd import ops
from tests import test_gpu_ops as t
for pair, rows, cols, n in (("bf16", 3000, 513, 100), ("f32", 3000, 77, 2000), ("f16", 2000, 24, 9000),
                            ("f32", (1 << 21) + 9, 3, 700)):
    table, add = t.randn(rows, cols, pair, 1), t.randn(n, cols, pair, 2)
    ids = t.rand_ids(n, rows, 3, 0.1, True)
    t.check_embedding(table, ids, torch.empty_like(add), 1.5, add)
    ws = ops.EmbeddingWorkspace(n, cols)
    for accumulate in (False, True):
        t.check_grad(add, ids, table, ws, 1.0, accumulate, pair)
    t.check_dropout(add, 0.3, ops.DropoutRng(4, 5), 6, torch.empty_like(add), add, (4, 5))
    t.check_dropout(add[:, :-1], 0.3, ops.DropoutRng(4, 5), 6, torch.empty_like(add)[:, 1:], None, (4, 5))
print("folded ok")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, NBO_GRID_X_MAX="7", PYTHONPATH=root)
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=root, env=env)
    assert r.returncode == 0 and "folded ok" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]
