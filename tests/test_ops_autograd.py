"""The operators beside torch's autograd: a gradient is never lost without a word."""
import pytest
import torch

from nabla_amd import ops


@pytest.mark.parametrize("place", ["table", "add", "out", "grad_out", "grad", "x", "residual", "dropped", "dx"])
def test_tensors_that_require_a_gradient_are_refused_while_gradients_are_recorded(place):
    plain, w = torch.zeros(3, 8), torch.zeros(3, 8, requires_grad=True)
    t = lambda name: w * 1.0 if name == place and place in ("add", "x") else w if name == place else plain
    ids = torch.zeros(3, dtype=torch.int64)

    class Rng:
        _h = None

    calls = {
        ("table", "add", "out"): lambda: ops.embedding(t("table"), ids, t("out"), add=t("add")),
        ("grad_out", "grad"): lambda: ops.embedding_grad(t("grad_out"), ids, t("grad"), Rng()),
        ("x", "residual", "dropped"): lambda: ops.dropout(t("x"), 0.1, Rng(), 0, t("dropped"), residual=t("residual")),
        ("dx",): lambda: ops.dropout_grad(t("dx"), 0.1, Rng(), 0, plain),
    }
    call = next(c for names, c in calls.items() if place in names)
    with pytest.raises(RuntimeError, match="not recorded by autograd"):
        call()


def test_without_recording_they_are_taken():
    w = torch.zeros(3, 8, requires_grad=True)
    with torch.no_grad():
        assert ops._matrix(w).rows == 3
    with torch.inference_mode():
        assert ops._matrix(w).rows == 3
        ops._done(0, torch.zeros(2))  # (has no version: nothing to tell)
    assert ops._matrix(w.detach()).cols == 8

    class Inside(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            assert ops._matrix(x).rows == 3
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            return g

    Inside.apply(w).sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("call", ["embedding", "embedding_grad", "dropout", "dropout_grad"])
def test_autograd_notices_that_a_saved_tensor_has_been_written(gpu, call):
    x = torch.randn(6, 8, device="cuda:0")
    w = torch.randn(6, 8, device="cuda:0", requires_grad=True)
    ids = torch.arange(6, device="cuda:0")
    y = (x * w).sum()  # saves x
    if call == "embedding":
        ops.embedding(torch.ones(6, 8, device="cuda:0"), ids, x, add=x)
    elif call == "embedding_grad":
        ops.embedding_grad(torch.ones(6, 8, device="cuda:0"), ids, x, ops.EmbeddingWorkspace(6, 8), accumulate=True)
    elif call == "dropout":
        ops.dropout(x, 0.5, ops.DropoutRng(1), 0, x)
    else:
        ops.dropout_grad(x, 0.5, ops.DropoutRng(1), 0, x[:])  # a view of it
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
