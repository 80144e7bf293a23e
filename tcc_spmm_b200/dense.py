"""Dense operators on 8-bit blocks: the quantizer to 8-bit floating point, the product of two such
matrices, and INT8 activation checkpoints with the gradients computed from them.

A matrix is cut into blocks of 128 columns of a row, or of 128 x 128 elements; every block has one
power-of-two scale, kept as its biased exponent byte (torch.uint8, or torch.float8_e8m0fnu; value
2^(byte - 127)). include/tcc_spmm_b200.h states the rule.

Every operand is a 2-D CUDA tensor of one device whose last dimension has stride 1; rows may be
any distance apart. The calls enqueue work on `stream` (default: torch's current stream of that
device), never synchronise, and raise InvalidArgument for tensors that do not fit together. They
write into tensors that the caller gives. The reference has no counterpart.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _native as N
from .api import InvalidArgument, _check, _stream_handle

BLOCK = 128
ACTIVATIONS = {"relu": 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "identity": 4}
LAYOUTS = {"nk": 0, "kn": 1}


def _types():
    import torch

    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise InvalidArgument(message)


def _matrix(name: str, t, device=None, shape=None) -> int:
    """Checks a 2-D operand and returns its row stride in elements."""
    _need(hasattr(t, "data_ptr") and t.dim() == 2, f"{name} must be a 2-D tensor")
    _need(t.is_cuda, f"{name} must be a CUDA tensor")
    _need(device is None or t.device == device, f"{name} is on {t.device}, expected {device}")
    _need(shape is None or tuple(t.shape) == tuple(shape), f"{name} has shape {tuple(t.shape)}, expected {shape}")
    rows, cols = t.shape
    _need(rows < 2 ** 32 and cols < 2 ** 32, f"{name} is too large")
    _need(cols <= 1 or t.stride(1) == 1, f"{name} must have stride 1 along its last dimension")
    if rows <= 1:
        return max(cols, t.stride(0) if rows == 1 else cols)
    _need(t.stride(0) >= cols, f"the rows of {name} overlap")
    return t.stride(0)


def _scales(name: str, t, device, rows: int, cols: int, block_rows=(1, BLOCK)) -> int:
    """Checks the scale bytes of a [rows, cols] matrix and returns the rows per block."""
    import torch

    _need(hasattr(t, "data_ptr") and t.dtype in (torch.uint8, torch.float8_e8m0fnu),
          f"{name} must hold scale bytes (uint8 or float8_e8m0fnu)")
    _need(t.device == device, f"{name} is on {t.device}, expected {device}")
    shapes = {b: (-(-rows // b), -(-cols // BLOCK)) for b in block_rows}
    for b, shape in shapes.items():
        if tuple(t.shape) == shape:
            _need(t.is_contiguous(), f"{name} must be contiguous")
            return b
    raise InvalidArgument(f"{name} has shape {tuple(t.shape)}, expected {' or '.join(map(str, shapes.values()))}")


def _type(name: str, t, allowed) -> int:
    code = _types().get(t.dtype)
    _need(code in allowed, f"{name} has unsupported type {t.dtype}")
    return code


def _launch(device, call, *args) -> None:
    import torch

    if device.index is None or device.index == torch.cuda.current_device():
        _check(call(*args))
    else:
        with torch.cuda.device(device):
            _check(call(*args))


def quantize_blocks_fp8(x, q, scales, block_rows: int = 1, stream=None) -> None:
    """q, scales = the blocks of x [rows, cols] (fp32, bf16 or fp16) in 8-bit floating point.

    q: [rows, cols] of float8_e4m3fn or float8_e5m2; scales: [ceil(rows / block_rows),
    ceil(cols / 128)] bytes; block_rows 1 (activations) or 128 (weights). matmul_fp8_blocks runs
    fastest on a q whose rows start on 16 bytes."""
    xs = _matrix("x", x)
    qs = _matrix("q", q, x.device, x.shape)
    xt, qt = _type("x", x, (0, 1, 2)), _type("q", q, (3, 4))
    _need(block_rows in (1, BLOCK), "block_rows must be 1 or 128")
    rows, cols = x.shape
    _scales("scales", scales, x.device, rows, cols, (block_rows,))
    _launch(x.device, N.lib().tcc_quantize_blocks_fp8, x.data_ptr(), xt, xs, q.data_ptr(), qt, qs, scales.data_ptr(),
            rows, cols, block_rows, _stream_handle(stream, x))


def matmul_fp8_blocks(a, a_scales, b, b_scales, output, bias=None, b_layout: str = "nk", stream=None) -> None:
    """output [m, n] = a [m, k] times the transpose of b [n, k] (b_layout "nk", a layer's forward
    product) or times b [k, n] ("kn": the gradient of a layer's input, from the same weights), plus
    bias [n] (fp32).

    a and b: float8_e4m3fn or float8_e5m2 blocks; the shapes of the scales tell blocks of a row from
    blocks of 128 x 128 (b [k, n] needs the latter). The sum is accumulated in fp32 and rounded once
    to output's type (fp32, bf16 or fp16)."""
    _need(b_layout in LAYOUTS, f"b_layout must be one of {sorted(LAYOUTS)}")
    as_ = _matrix("a", a)
    device, (m, k) = a.device, a.shape
    bs = _matrix("b", b, device)
    n = b.shape[0] if b_layout == "nk" else b.shape[1]
    _need(tuple(b.shape) == ((n, k) if b_layout == "nk" else (k, n)), f"b has shape {tuple(b.shape)}, k is {k}")
    os_ = _matrix("output", output, device, (m, n))
    at, bt, ot = _type("a", a, (3, 4)), _type("b", b, (3, 4)), _type("output", output, (0, 1, 2))
    a_rows = _scales("a_scales", a_scales, device, m, k)
    b_rows = _scales("b_scales", b_scales, device, *b.shape, (1, BLOCK) if b_layout == "nk" else (BLOCK,))
    if bias is not None:
        import torch

        _need(bias.dtype == torch.float32 and tuple(bias.shape) == (n,) and bias.is_contiguous() and
              bias.device == device, f"bias must be {n} contiguous fp32 values on {device}")
    _launch(device, N.lib().tcc_matmul_fp8_blocks, a.data_ptr(), at, as_, a_scales.data_ptr(), a_rows, b.data_ptr(), bt,
            bs, b_scales.data_ptr(), b_rows, LAYOUTS[b_layout], bias.data_ptr() if bias is not None else None,
            output.data_ptr(), ot, os_, m, n, k, _stream_handle(stream, a))


def activation_checkpoint_int8(x, y, q, scales, activation: str = "gelu", stream=None) -> None:
    """y = f(x), and x kept for the backward pass as INT8 blocks of 128 columns of a row.

    x, y: [rows, cols] of one type (fp32, bf16 or fp16), y may be x itself; q: int8 [rows, cols];
    scales: [rows, ceil(cols / 128)] bytes. activation: relu, gelu, gelu_tanh, silu, or identity,
    which keeps x alone (y None)."""
    import torch

    _need(activation in ACTIVATIONS, f"activation must be one of {sorted(ACTIVATIONS)}")
    xs = _matrix("x", x)
    xt = _type("x", x, (0, 1, 2))
    if activation == "identity":
        _need(y is None, "the identity writes no y: pass None")
        ys = 0
    else:
        ys = _matrix("y", y, x.device, x.shape)
        _need(y.dtype == x.dtype, "y must have x's type")
        _need(y.data_ptr() != x.data_ptr() or ys == xs, "y may be x itself, not another view of it")
    qs = _matrix("q", q, x.device, x.shape)
    _need(q.dtype == torch.int8, "q must be int8")
    rows, cols = x.shape
    _scales("scales", scales, x.device, rows, cols, (1,))
    _launch(x.device, N.lib().tcc_activation_checkpoint_int8, x.data_ptr(), xs, y.data_ptr() if y is not None else None,
            ys, xt, q.data_ptr(), qs, scales.data_ptr(), rows, cols, ACTIVATIONS[activation], _stream_handle(stream, x))


def activation_backward_int8(grad_y, q, scales, grad_x, activation: str = "gelu", stream=None) -> None:
    """grad_x = grad_y * f'(x^), x^ the values that the checkpoint (q, scales) of
    activation_checkpoint_int8 stands for.

    grad_y, grad_x: [rows, cols] of one type (fp32, bf16 or fp16); grad_x may be grad_y itself.
    ReLU passes the gradient where x^ > 0."""
    import torch

    _need(activation in ACTIVATIONS and activation != "identity",
          f"activation must be one of {sorted(set(ACTIVATIONS) - {'identity'})}")
    gs = _matrix("grad_y", grad_y)
    gt = _type("grad_y", grad_y, (0, 1, 2))
    xs = _matrix("grad_x", grad_x, grad_y.device, grad_y.shape)
    _need(grad_x.dtype == grad_y.dtype, "grad_x must have grad_y's type")
    _need(grad_x.data_ptr() != grad_y.data_ptr() or xs == gs, "grad_x may be grad_y itself, not another view of it")
    qs = _matrix("q", q, grad_y.device, grad_y.shape)
    _need(q.dtype == torch.int8, "q must be int8")
    rows, cols = grad_y.shape
    _scales("scales", scales, grad_y.device, rows, cols, (1,))
    _launch(grad_y.device, N.lib().tcc_activation_backward_int8, grad_y.data_ptr(), gs, gt, q.data_ptr(), qs,
            scales.data_ptr(), grad_x.data_ptr(), xs, rows, cols, ACTIVATIONS[activation],
            _stream_handle(stream, grad_y))


def weight_grad_int8_workspace_size(rows: int, n: int, k: int) -> int:
    """Bytes of workspace that weight_grad_int8 needs for grad_y [rows, n] and a checkpoint [rows, k]."""
    size = C.c_uint64()
    _check(N.lib().tcc_weight_grad_int8_workspace_size(rows, n, k, C.byref(size)))
    return size.value


def weight_grad_int8(grad_y, q, scales, grad_w, accumulate: bool = False, workspace: Optional[object] = None,
                     stream=None) -> None:
    """grad_w [n, k] = the transpose of grad_y [rows, n] times x^ [rows, k], added to grad_w with
    accumulate=True: the weight gradient of a layer whose input was kept as a checkpoint (q, scales)
    of activation_checkpoint_int8.

    grad_y: fp32, bf16 or fp16; grad_w: fp32. workspace: a contiguous CUDA tensor of
    weight_grad_int8_workspace_size bytes or more, not shared with a call that may run at the same
    time; None takes it from torch's allocator, on the stream of the call."""
    import torch

    gs = _matrix("grad_y", grad_y)
    device, (rows, n) = grad_y.device, grad_y.shape
    gt = _type("grad_y", grad_y, (0, 1, 2))
    _need(hasattr(q, "dim") and q.dim() == 2 and q.shape[0] == rows, f"q must be a 2-D tensor of {rows} rows")
    k = q.shape[1]
    qs = _matrix("q", q, device)
    _need(q.dtype == torch.int8, "q must be int8")
    ws = _matrix("grad_w", grad_w, device, (n, k))
    _need(grad_w.dtype == torch.float32, "grad_w must be fp32")
    _scales("scales", scales, device, rows, k, (1,))
    need = weight_grad_int8_workspace_size(rows, n, k)
    if workspace is None and need:
        if isinstance(stream, int):
            stream = torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device)
        with torch.cuda.stream(stream):  # nothing for None: the current stream
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
    if workspace is not None:
        _need(workspace.device == device and workspace.is_contiguous(), f"the workspace must be contiguous on {device}")
    have = workspace.numel() * workspace.element_size() if workspace is not None else 0
    _launch(device, N.lib().tcc_weight_grad_int8, grad_y.data_ptr(), gt, gs, q.data_ptr(), qs, scales.data_ptr(),
            grad_w.data_ptr(), ws, rows, n, k, int(bool(accumulate)),
            workspace.data_ptr() if workspace is not None else None, have, _stream_handle(stream, grad_y))
