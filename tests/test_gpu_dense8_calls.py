"""Ways of calling the dense operators on 8-bit blocks: captured before any other call, and on streams of any kind."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

import tcc_spmm_b200 as T
from tests import dense8_util as D

pytestmark = pytest.mark.gpu

FIRST_CAPTURED = """
import torch
from tests.test_gpu_dense8 import layer, layer_inputs
args = layer_inputs(3, m=200, n=500 // 4 * 4, k=4096)  # few tiles of a long k: CTAs share it
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    out = layer(*args)
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, layer(*args)))
print("same")
"""


def test_first_calls_of_a_process_may_be_captured():
    """What a call asks the device for once (attributes, occupancy, the driver's entry point) may fall into a capture."""
    run = subprocess.run([sys.executable, "-c", FIRST_CAPTURED], cwd=Path(__file__).resolve().parent.parent, timeout=300,
                         capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.strip() == "same", run.stdout + run.stderr


@pytest.mark.parametrize("rows", [300, 20000])  # without and with a workspace of the call's own
def test_streams_of_any_kind(rows):
    """A torch stream, its handle, and an object that holds one, as every call of the library takes them."""
    n, k = 64, 128
    q64, scales = D.quantize(D.make(rows, k, torch.float32, 1), "int8")
    q, dy = q64.to(torch.int8), D.make(rows, n, torch.bfloat16, 2)
    assert (T.weight_grad_int8_workspace_size(rows, n, k) > 0) == (rows == 20000)
    want = torch.empty(n, k, device="cuda")
    T.weight_grad_int8(dy, q, scales, want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream, SimpleNamespace(cuda_stream=side.cuda_stream)):
        dw, dx = torch.empty(n, k, device="cuda"), torch.empty(rows, n, device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        T.weight_grad_int8(dy, q, scales, dw, stream=stream)
        T.activation_backward_int8(dy, q[:, :n], scales, dx, activation="relu", stream=stream)
        side.synchronize()
        assert torch.equal(dw, want)
        assert torch.equal(dx, torch.where(q[:, :n] > 0, dy, torch.zeros_like(dy)))
