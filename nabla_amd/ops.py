"""Operators beside the optimizer step: embedding lookup, its gradient, and dropout.

They produce and consume the tensors the step works on: the embedding matrix is the largest
parameter of a language model, its gradient is the one that is not a matrix product, and
dropout is an element-wise pass like the Backend primitives (``nabla_amd.backend``).  Each call
is one entry point of ``include/nabla_ops.h``: hand-written gfx950 kernels on the library's
stream, nothing allocated, nothing read back, so that a call may be captured into a HIP graph.

    rng = ops.DropoutRng(seed)
    ws = ops.EmbeddingWorkspace(max_ids=8192, max_cols=768)
    ops.embedding(wpe, positions, x)                       # x = wpe[positions]
    ops.embedding(wte, tokens, x, add=x)                   # x = x + wte[tokens]
    ops.dropout(x, 0.1, rng, site=0, out=x)
    ...                                                    # the model, forward and backward
    ops.dropout_grad(dx, 0.1, rng, site=0, out=dx)         # the same mask again, from the counter
    ops.embedding_grad(dx, tokens, wte_grad, ws, accumulate=True)
    ops.embedding_grad(dx, positions, wpe_grad, ws, accumulate=True)
    optimizer.fused_step(params, grads, zero_grads=True)
    rng.advance()

Tensors are torch tensors on cuda:0, or anything else with ``data_ptr()``, ``shape`` and
``dtype``.  A tensor of more than two dimensions stands for the matrix of its last one; rows may be
strided, the elements of a row are adjacent.

The calls are outside torch's autograd, as the optimizers' are: what they write has no graph behind it, and the
backward pass calls ``dropout_grad`` and ``embedding_grad`` itself.  So a tensor that requires a gradient is
refused where gradients are recorded (``detach()`` it, or call under ``torch.no_grad()``, as inside a
``torch.autograd.Function``), and autograd is told that the tensor a call has written holds other values.
A graph that has captured a call needs its tensors, workspace and generator for as long as it is replayed.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Optional

from . import _lib
from .optim import _call, _dtype_code, _shape2

try:
    from torch import Tensor as _Tensor, is_grad_enabled as _recording
    from torch.autograd.graph import increment_version as _increment_version
except ImportError:  # other tensors have no autograd
    _Tensor = _recording = _increment_version = None


_dtype_codes = {}  # by dtype object: spares the smallest calls the name's parsing


def _matrix(t) -> _lib.Matrix:
    if getattr(t, "requires_grad", False) and _recording is not None and _recording():
        raise RuntimeError("this call is not recorded by autograd, and a tensor given to it requires a gradient: pass "
                           "tensor.detach() or call under torch.no_grad()")
    try:
        rows, cols = t.shape
        stride, unit = t.stride()
    except (AttributeError, ValueError):  # no strides, or not two dimensions
        if hasattr(t, "is_contiguous") and not t.is_contiguous():
            raise ValueError("a strided tensor must have two dimensions") from None
        rows, cols = _shape2(t)
        stride, unit = cols, 1
    if unit != 1 and cols > 1:
        raise ValueError("the elements of a row must be adjacent")
    code = _dtype_codes.get(t.dtype)
    if code is None:
        code = _dtype_codes[t.dtype] = _dtype_code(t)
    return _lib.Matrix(t.data_ptr(), rows, cols, stride, code)


def _done(status: int, written) -> None:
    """The end of a call that has written a tensor: what autograd has saved of it for a backward pass is gone."""
    if status:
        _call(status)
    if _Tensor is not None and isinstance(written, _Tensor):
        _increment_version(written)


_id_codes = {}


def _ids(t) -> _lib.Ids:
    code = _id_codes.get(t.dtype)
    if code is None:
        name = str(t.dtype).rsplit(".", 1)[-1]
        if name not in ("int32", "int64"):
            raise TypeError(f"ids are int32 or int64, not {name}")
        code = _id_codes[t.dtype] = _lib.ID_I64 if name == "int64" else _lib.ID_I32
    if hasattr(t, "is_contiguous") and not t.is_contiguous():
        raise ValueError("ids must be contiguous")
    n = 1
    for k in t.shape:
        n *= int(k)
    return _lib.Ids(t.data_ptr(), n, code)


def embedding(table, ids, out, scale: float = 1.0, add=None) -> None:
    """out[t] = add[t] + scale * table[ids[t]]; without `add`, scale * table[ids[t]].

    An id outside the table (negative, or not below its rows: padding) stands for a row of zeros.
    `out` has the table's type, or bf16 / f16 over an f32 table; `add` has out's type and may be
    `out` itself.  Computed in f32 (f64 tables: f64), rounded once."""
    a = _matrix(add) if add is not None else None
    _done(_lib.load().nbo_embedding(_matrix(table), _ids(ids), a, scale, _matrix(out)), out)


class EmbeddingWorkspace:
    """Scratch of `embedding_grad` for up to `max_ids` ids and `max_cols` columns.  Nothing in it
    outlives a call; two calls that run at the same time (two captured graphs on two streams)
    need one each."""

    def __init__(self, max_ids: int, max_cols: int):
        self._h = None
        h = C.c_void_p()
        _call(_lib.load().nbo_embedding_ws_create(int(max_ids), int(max_cols), C.byref(h)))
        self._h = h

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            try:
                _lib.load().nbo_embedding_ws_destroy(h)
            except Exception:
                pass


def embedding_grad(grad_out, ids, grad, workspace: EmbeddingWorkspace, scale: float = 1.0,
                   accumulate: bool = False) -> None:
    """The gradient of `embedding` with respect to the table:
    grad[v] = (grad[v] if accumulate else 0) + scale * sum of grad_out[t] over ids[t] == v.

    Without `accumulate` every row of `grad` is written, zeros where no id names it; with it the
    rows no id names are not touched.  What rows of `grad_out` hold whose id is outside the table does
    not matter.  `grad` has grad_out's type, or f32 under bf16 / f16.  Sums are f32 (f64: f64) in a fixed
    order, the same bits on every run, rounded once."""
    _done(_lib.load().nbo_embedding_grad(_matrix(grad_out), _ids(ids), scale, 1 if accumulate else 0, _matrix(grad),
                                         workspace._h), grad)


@dataclass
class DropoutRngState:
    seed: int = 0
    step: int = 0


class DropoutRng:
    """The counter-based generator's state, on the device: masks are a function of (seed, step,
    site, element), nothing is stored.  `advance()` once a micro-batch, after its backward pass;
    inside a captured graph too, whose replays then draw new masks."""

    def __init__(self, seed: int = 0, step: int = 0):
        self._h = None
        h = C.c_void_p()
        _call(_lib.load().nbo_rng_create(_u64(seed), _u64(step), C.byref(h)))
        self._h = h

    def __del__(self):
        h, self._h = getattr(self, "_h", None), None
        if h:
            try:
                _lib.load().nbo_rng_destroy(h)
            except Exception:
                pass

    def advance(self, steps: int = 1) -> None:
        _call(_lib.load().nbo_rng_advance(self._h, _u64(steps)))

    def state(self) -> DropoutRngState:
        seed, step = C.c_uint64(0), C.c_uint64(0)
        _call(_lib.load().nbo_rng_state_get(self._h, C.byref(seed), C.byref(step)))
        return DropoutRngState(seed.value, step.value)

    def load_state(self, state: DropoutRngState) -> None:
        _call(_lib.load().nbo_rng_load_state(self._h, _u64(state.seed), _u64(state.step)))


def _u64(x: int) -> int:
    x = int(x)
    if not 0 <= x < 1 << 64:
        raise ValueError(f"{x} is not an unsigned 64-bit number")
    return x


def dropout(x, p: float, rng: DropoutRng, site: int, out, residual=None) -> None:
    """out = residual + (kept ? x / (1 - p) : 0); without `residual`, the second term alone.

    p is taken to the nearest 2^-16, in the mask and in the factor.  `site` tells the dropouts of one
    step apart: one number per place in the model.  A dropped element is zero whatever x holds
    there.  `out` may be `x` or `residual`."""
    if not 0 <= site < 1 << 32:
        raise ValueError(f"site {site} is not an unsigned 32-bit number")
    r = _matrix(residual) if residual is not None else None
    _done(_lib.load().nbo_dropout(_matrix(x), r, p, rng._h, site, _matrix(out)), out)


def dropout_grad(grad_out, p: float, rng: DropoutRng, site: int, out) -> None:
    """The gradient of `dropout` with respect to x, at the same step and site of `rng`: grad_out
    through the same mask and factor.  (With respect to `residual` it is grad_out itself; to add what
    reaches x by other ways, call `dropout` with that as `residual`.)"""
    dropout(grad_out, p, rng, site, out)
