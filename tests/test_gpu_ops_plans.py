"""The operators on the GPU where their plan decides what runs: captures, long pieces, many tiles."""
import os
import subprocess
import sys

import pytest

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
