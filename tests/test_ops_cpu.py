"""The operators of include/nabla_ops.h without a GPU: symbols, struct layouts, and what their entry
points refuse before they touch the device."""
import ctypes as C
import os
import re

import pytest

from nabla_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nabla_ops.h")
BASE = 0x7F0000000000  # an address nothing is ever read from: every call here ends before the device


def _decls():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_library_exports_every_declared_symbol():
    lib = _lib.load()
    declared = sorted(set(re.findall(r"\b(nbo_[a-z0-9_]+)\s*\(", _decls())))
    assert declared == sorted(_lib.OPS_SYMBOLS)
    for name in declared:
        assert hasattr(lib, name), name
        args = re.search(r"\bint %s\s*\(([^)]*)\)" % name, _decls()).group(1)
        assert len(args.split(",")) == len(_lib.OPS_SYMBOLS[name][1]), name


def test_struct_layouts_match_the_header():
    assert C.sizeof(_lib.Matrix) == 4 * 8 + 2 * 4 and C.sizeof(_lib.Ids) == 2 * 8 + 2 * 4
    for name, ty in (("nbo_matrix", _lib.Matrix), ("nbo_ids", _lib.Ids)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _decls(), flags=re.S).group(1)
        fields = [n.strip(" *\n") for d in body.split(";") if d.strip() for n in
                  re.sub(r"^\s*(const\s+)?\w+", "", d.strip()).split(",")]
        assert fields == [f for f, _ in ty._fields_]


def test_header_is_plain_c99(tmp_path):
    import subprocess

    src = tmp_path / "t.c"
    src.write_text('#include "nabla_ops.h"\nint main(void) { nbo_matrix m = {0}; nbo_ids i = {0}; '
                   "return nbo_embedding(&m, &i, 0, 1.0, 0) == NBO_ERR_ARG ? 0 : 1; }\n")
    libdir = os.path.join(ROOT, "nabla_amd")
    r = subprocess.run(["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-Wno-missing-field-initializers",
                        "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "t"), str(src), "-L", libdir,
                        "-l:libnabla_optim.so", f"-Wl,-rpath,{libdir}", "-Wl,-rpath,/opt/rocm/lib"],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert subprocess.run([str(tmp_path / "t")]).returncode == 0


def mat(rows, cols, at=BASE, stride=None, dtype=_lib.DT_F32):
    return _lib.Matrix(at, rows, cols, cols if stride is None else stride, dtype, 0)


def ids(n, at=BASE + (1 << 40), kind=_lib.ID_I64):
    return _lib.Ids(at, n, kind, 0)


TABLE, OUT, ADD = BASE, BASE + (1 << 36), BASE + (1 << 37)
F32, BF16, F64, F16 = _lib.DT_F32, _lib.DT_BF16, _lib.DT_F64, _lib.DT_F16


def _embedding(table, i, add, out):
    return _lib.load().nbo_embedding(table, i, add, 1.0, out)


REFUSED_EMBEDDING = [
    ("null table", None, ids(3), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("null ids", mat(9, 4), None, None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("null out", mat(9, 4), ids(3), None, None, _lib.ERR_ARG),
    ("dtype", mat(9, 4, dtype=7), ids(3), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("id type", mat(9, 4), ids(3, kind=2), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("rows of out", mat(9, 4), ids(3), None, mat(2, 4, OUT), _lib.ERR_SHAPE),
    ("cols of out", mat(9, 4), ids(3), None, mat(3, 5, OUT), _lib.ERR_SHAPE),
    ("shape of add", mat(9, 4), ids(3), mat(1, 4, ADD), mat(3, 4, OUT), _lib.ERR_SHAPE),
    ("type of out", mat(9, 4, dtype=BF16), ids(3), None, mat(3, 4, OUT), _lib.ERR_DTYPE),
    ("type of out", mat(9, 4, dtype=BF16), ids(3), None, mat(3, 4, OUT, dtype=F16), _lib.ERR_DTYPE),
    ("type of out", mat(9, 4, dtype=F64), ids(3), None, mat(3, 4, OUT, dtype=BF16), _lib.ERR_DTYPE),
    ("type of add", mat(9, 4), ids(3), mat(3, 4, ADD), mat(3, 4, OUT, dtype=BF16), _lib.ERR_DTYPE),
    ("stride", mat(9, 4, stride=3), ids(3), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("alignment of the table", mat(9, 4, TABLE + 2), ids(3), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("alignment of ids", mat(9, 4), ids(3, BASE + (1 << 40) + 4), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("null address", mat(9, 4, None), ids(3), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("null address of ids", mat(9, 4), ids(3, None), None, mat(3, 4, OUT), _lib.ERR_ARG),
    ("out in the table", mat(9, 4), ids(3), None, mat(3, 4, TABLE + 16), _lib.ERR_ARG),
    ("out over the ids", mat(9, 4), ids(3), None, mat(3, 4, BASE + (1 << 40) + 16), _lib.ERR_ARG),
    ("out overlaps add in part", mat(9, 4), ids(3), mat(3, 4, OUT + 16), mat(3, 4, OUT), _lib.ERR_ARG),
    ("interleaved columns that overlap", mat(9, 4), ids(3), mat(3, 4, OUT + 12, stride=8), mat(3, 4, OUT, stride=8),
     _lib.ERR_ARG),
    ("too many rows", mat(1 << 31, 4), ids(3), None, mat(3, 4, OUT), _lib.ERR_TOO_LARGE),
    ("too many columns", mat(2, (1 << 27) + 1), ids(3), None, mat(3, (1 << 27) + 1, OUT), _lib.ERR_TOO_LARGE),
    ("too many ids", mat(9, 4), ids(1 << 31), None, mat(1 << 31, 4, OUT), _lib.ERR_TOO_LARGE),
    ("stride beyond 64 bits", mat(9, 4, stride=1 << 60), ids(3), None, mat(3, 4, OUT), _lib.ERR_TOO_LARGE),
]


@pytest.mark.parametrize("case", REFUSED_EMBEDDING, ids=[f"{k}-{c[0]}" for k, c in enumerate(REFUSED_EMBEDDING)])
def test_embedding_refuses(case):
    _, table, i, add, out, status = case
    assert _embedding(table, i, add, out) == status
    assert _lib.load().nbo_last_error()


def _passes_the_argument_checks(rc):
    """What a well-formed call ends with where there is no memory behind its addresses: no device, or
    (with one) the address check."""
    text = _lib.load().nbo_last_error()
    return rc == _lib.ERR_NO_DEVICE or (rc == _lib.ERR_ARG and b"not memory the HIP runtime knows" in text)


def test_column_slices_of_one_allocation_do_not_overlap():
    add, out = mat(3, 4, OUT, stride=8), mat(3, 4, OUT + 16, stride=8)
    assert _passes_the_argument_checks(_embedding(mat(9, 4), ids(3), add, out))
    assert _passes_the_argument_checks(_embedding(mat(9, 4), ids(3), out, add))
    assert _passes_the_argument_checks(_embedding(mat(9, 4), ids(3), mat(3, 4, OUT), mat(3, 4, OUT)))  # in place
    # one row: its stride says nothing
    assert _passes_the_argument_checks(_embedding(mat(9, 4), ids(1), mat(1, 4, OUT, 0), mat(1, 4, OUT, 99)))


def test_embedding_grad_refuses(monkeypatch):
    lib = _lib.load()

    def call(dy, i, grad, ws=None):
        return lib.nbo_embedding_grad(dy, i, 1.0, 0, grad, ws)

    good = (mat(3, 4, OUT), ids(3), mat(9, 4))
    assert call(None, good[1], good[2]) == _lib.ERR_ARG
    assert call(good[0], None, good[2]) == _lib.ERR_ARG
    assert call(good[0], good[1], None) == _lib.ERR_ARG
    assert call(*good) == _lib.ERR_ARG and b"workspace" in lib.nbo_last_error()
    assert lib.nbo_embedding_ws_create(8, 8, None) == _lib.ERR_ARG
    h = C.c_void_p(1)
    assert lib.nbo_embedding_ws_create(1 << 31, 8, C.byref(h)) == _lib.ERR_TOO_LARGE and not h.value


DROPOUT = [
    ("null x", None, None, 0.1, mat(3, 4, OUT), _lib.ERR_ARG),
    ("null out", mat(3, 4), None, 0.1, None, _lib.ERR_ARG),
    ("null generator", mat(3, 4), None, 0.1, mat(3, 4, OUT), _lib.ERR_ARG),
]


@pytest.mark.parametrize("case", DROPOUT, ids=[c[0] for c in DROPOUT])
def test_dropout_refuses_nulls(case):
    _, x, residual, p, out, status = case
    assert _lib.load().nbo_dropout(x, residual, p, None, 0, out) == status


def test_generator_refuses_nulls():
    lib = _lib.load()
    seed = C.c_uint64()
    assert lib.nbo_rng_create(1, 0, None) == _lib.ERR_ARG
    assert lib.nbo_rng_state_get(None, C.byref(seed), C.byref(seed)) == _lib.ERR_ARG
    assert lib.nbo_rng_load_state(None, 1, 2) == _lib.ERR_ARG
    assert lib.nbo_rng_advance(None, 1) == _lib.ERR_ARG
    assert lib.nbo_rng_destroy(None) in (_lib.OK, _lib.ERR_NO_DEVICE)
    assert lib.nbo_embedding_ws_destroy(None) in (_lib.OK, _lib.ERR_NO_DEVICE)


def test_python_arguments_are_checked():
    import torch

    with pytest.raises(TypeError, match="int32 or int64"):
        ops._ids(torch.zeros(3))
    with pytest.raises(TypeError, match="int32 or int64"):
        ops._ids(torch.zeros(3, dtype=torch.uint8))
    with pytest.raises(ValueError, match="contiguous"):
        ops._ids(torch.zeros(6, dtype=torch.int64)[::2])
    with pytest.raises(ValueError, match="adjacent"):
        ops._matrix(torch.zeros(4, 3).t())
    with pytest.raises(ValueError, match="two dimensions"):
        ops._matrix(torch.zeros(2, 3, 8)[:, :, :4])
    with pytest.raises(TypeError, match="unsupported tensor dtype"):
        ops._matrix(torch.zeros(2, 3, dtype=torch.int32))
    with pytest.raises(ValueError, match="64-bit"):
        ops._u64(1 << 64)
    with pytest.raises(ValueError, match="32-bit"):
        ops.dropout(None, 0.1, None, 1 << 32, None)
    m = ops._matrix(torch.zeros(2, 3, 8, dtype=torch.bfloat16))
    assert (m.rows, m.cols, m.stride, m.dtype) == (6, 8, 8, BF16)
    m = ops._matrix(torch.zeros(5, 8)[:, 2:7])
    assert (m.rows, m.cols, m.stride, m.dtype) == (5, 5, 8, F32)
    m = ops._matrix(torch.zeros(7, dtype=torch.float16))
    assert (m.rows, m.cols, m.dtype) == (1, 7, F16)
    assert ops._ids(torch.zeros(2, 3, dtype=torch.int32)).n == 6


def test_rust_declarations_agree_with_the_header():
    """integration/rust/ops.rs cannot be compiled here: the same symbols, and for every argument the
    same kind and width."""
    c_kind = {"double": "f64", "uint64_t": "u64", "uint32_t": "u32", "int": "int", "int32_t": "i32"}
    r_kind = {"f64": "f64", "u64": "u64", "u32": "u32", "c_int": "int", "i32": "i32"}
    c, rust = {}, {}
    for name, args in re.findall(r"\bint (nbo_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", _decls()):
        c[name] = ["ptr" if "*" in a else c_kind[a.replace("const", "").split()[0]] for a in args.split(",")]
    text = re.sub(r"//.*", "", open(os.path.join(ROOT, "integration", "rust", "ops.rs")).read())
    for name, args in re.findall(r"pub fn (nbo_[a-z0-9_]+)\s*\(([^)]*)\)\s*->\s*c_int;", text):
        kinds = [a.split(":", 1)[1].strip() for a in args.split(",")]
        rust[name] = ["ptr" if k.startswith("*") else r_kind[k] for k in kinds]
    assert c == rust and len(c) == 10
    for c_name, r_name in (("nbo_matrix", "NboMatrix"), ("nbo_ids", "NboIds")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (c_name, c_name), _decls(), flags=re.S).group(1)
        want = []
        for d in body.split(";"):
            if d.strip():
                ty, names = re.match(r"\s*((?:const )?\w+)\s+(.*)", d.strip(), flags=re.S).groups()
                want += [(n.strip(" *"), "ptr" if "*" in n else c_kind[ty]) for n in names.split(",")]
        rbody = re.search(r"pub struct %s \{(.*?)\}" % r_name, text, flags=re.S).group(1)
        got = [(n.rstrip("_"), "ptr" if t.strip().startswith("*") else r_kind[t.strip()])
               for n, t in re.findall(r"pub (\w+): ([^,]+)", rbody)]
        assert got == want, (got, want)
    for name in ("NBO_ID_I32", "NBO_ID_I64"):
        assert int(re.search(r"\b%s = (\d+)" % name, _decls()).group(1)) == int(
            re.search(r"pub const %s: i32 = (\d+);" % name, text).group(1))


def test_cpp_program_is_built():
    assert os.path.exists(os.path.join(ROOT, "tests", "cpp", "test_ops.bin")), "build it with `make -C tests/cpp`"


class _Rng:
    """What TrainerTail needs of a DropoutRng."""

    def __init__(self, step):
        self.at = ops.DropoutRngState(9, step)

    def state(self):
        return ops.DropoutRngState(self.at.seed, self.at.step)

    def load_state(self, state):
        self.at = ops.DropoutRngState(state.seed, state.step)

    def advance(self, steps=1):
        self.at.step = (self.at.step + steps) % (1 << 64)


def test_trainer_tail_advances_the_generator_once_per_micro_batch():
    from nabla_amd.checkpoint import TrainState
    from nabla_amd.trainer import TrainerTail

    class Opt:
        def fused_step(self, *a, **k):
            if self.fail:
                raise RuntimeError("no")

    opt = Opt()
    opt.fail = False
    rng = _Rng((1 << 64) - 2)
    tail = TrainerTail(opt, []).with_rng(rng)
    assert tail.state.rng_state == (1 << 64) - 2
    assert tail.after_backward([]) and tail.after_backward([])
    assert rng.at.step == 0 == tail.state.rng_state and tail.state.step == 2
    opt.fail = True
    with pytest.raises(RuntimeError):
        tail.after_backward([])
    assert rng.at.step == 1 == tail.state.rng_state and tail.state.step == 2
    # a restored state moves the generator, before or after it is attached
    tail.set_state(TrainState(epoch=1, step=7, grad_accum=1, rng_state=40))
    assert rng.at == ops.DropoutRngState(9, 40)
    other = TrainerTail(opt, [])
    other.set_state(TrainState(rng_state=50))
    other.with_rng(rng)
    assert rng.at.step == 50
    other.set_state(TrainState(rng_state=None))  # a checkpoint without one: the generator's own
    assert rng.at.step == 50 == other.state.rng_state
