"""Dense operators on 8-bit blocks: the quantizer to 8-bit floating point, the product of two such
matrices, and INT8 activation checkpoints with the gradients computed from them.

A matrix is cut into blocks of 128 columns of a row, or of 128 x 128 elements; every block has one
power-of-two scale, kept as its biased exponent byte (torch.uint8, or torch.float8_e8m0fnu; value
2^(byte - 127)). include/tcc_spmm_b200.h states the rule.

Every operand is a 2-D CUDA tensor of one device whose last dimension has stride 1; rows may be
any distance apart. The calls enqueue work on `stream` (default: torch's current stream of that
device), never synchronise, and raise InvalidArgument for tensors that do not fit together. They
write into tensors that the caller gives. The reference has no counterpart.

The checks run on every call, and a small operator takes a few microseconds, so they are written
for speed: plain comparisons, with messages formed only when one fails.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

from . import _native as N
from .api import InvalidArgument, _check, _stream_handle

BLOCK = 128
ACTIVATIONS = {"relu": 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "identity": 4}
LAYOUTS = {"nk": 0, "kn": 1}

_torch = None     # torch, its raw-stream and device queries, and the type codes, once used
_TYPES: dict = {}
_FLOATS, _FP8 = frozenset((0, 1, 2)), frozenset((3, 4))


def _load():
    global _torch
    import torch

    _TYPES.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3,
                   torch.float8_e5m2: 4})
    _torch = torch
    return torch


def _refuse(message: str):
    raise InvalidArgument(message)


def _matrix(name: str, t, device=None, shape=None) -> int:
    """Checks a 2-D operand and returns its row stride in elements."""
    torch = _torch or _load()
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        _refuse(f"{name} must be a 2-D tensor")
    if not t.is_cuda:
        _refuse(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        _refuse(f"{name} is on {t.device}, expected {device}")
    rows, cols = t.shape
    if shape is not None and (rows != shape[0] or cols != shape[1]):
        _refuse(f"{name} has shape {(rows, cols)}, expected {tuple(shape)}")
    if rows >= 2 ** 32 or cols >= 2 ** 32:
        _refuse(f"{name} is too large")
    row_stride, col_stride = t.stride()
    if cols > 1 and col_stride != 1:
        _refuse(f"{name} must have stride 1 along its last dimension")
    if rows <= 1:  # no second row: the distance to it says nothing
        return -(-cols // 16) * 16
    if row_stride < cols:
        _refuse(f"the rows of {name} overlap")
    return row_stride


def _scales(name: str, t, device, rows: int, cols: int, row_blocks: bool = True, square_blocks: bool = True) -> int:
    """Checks the scale bytes of a [rows, cols] matrix and returns the rows per block."""
    torch = _torch
    if not isinstance(t, torch.Tensor) or (t.dtype != torch.uint8 and t.dtype != torch.float8_e8m0fnu):
        _refuse(f"{name} must hold scale bytes (uint8 or float8_e8m0fnu)")
    if t.device != device:
        _refuse(f"{name} is on {t.device}, expected {device}")
    if t.dim() == 2 and t.is_contiguous():
        r, c = t.shape
        if c == -(-cols // BLOCK):
            if row_blocks and r == rows:
                return 1
            if square_blocks and r == -(-rows // BLOCK):
                return BLOCK
    want = [(rows, -(-cols // BLOCK))] * row_blocks + [(-(-rows // BLOCK), -(-cols // BLOCK))] * square_blocks
    _refuse(f"{name} has shape {tuple(t.shape)}, expected contiguous {' or '.join(map(str, want))}")


def _type(name: str, t, allowed) -> int:
    code = _TYPES.get(t.dtype)
    if code not in allowed:
        _refuse(f"{name} has unsupported type {t.dtype}")
    return code


def _launch(device, stream, call, *args) -> None:
    """call(*args, stream) with `device` current."""
    torch = _torch
    index = device.index
    raw = torch._C._cuda_getCurrentRawStream(index) if stream is None else _stream_handle(stream)
    if index == torch._C._cuda_getDevice():
        status = call(*args, raw)
    else:
        with torch.cuda.device(device):
            status = call(*args, raw)
    if status:
        _check(status)


def quantize_blocks_fp8(x, q, scales, block_rows: int = 1, stream=None) -> None:
    """q, scales = the blocks of x [rows, cols] (fp32, bf16 or fp16) in 8-bit floating point.

    q: [rows, cols] of float8_e4m3fn or float8_e5m2; scales: [ceil(rows / block_rows),
    ceil(cols / 128)] bytes; block_rows 1 (activations) or 128 (weights). matmul_fp8_blocks runs
    fastest on a q whose rows start on 16 bytes."""
    xs = _matrix("x", x)
    device, shape = x.device, x.shape
    qs = _matrix("q", q, device, shape)
    xt, qt = _type("x", x, _FLOATS), _type("q", q, _FP8)
    if block_rows != 1 and block_rows != BLOCK:
        _refuse("block_rows must be 1 or 128")
    rows, cols = shape
    _scales("scales", scales, device, rows, cols, block_rows == 1, block_rows == BLOCK)
    _launch(device, stream, N.lib().tcc_quantize_blocks_fp8, x.data_ptr(), xt, xs, q.data_ptr(), qt, qs,
            scales.data_ptr(), rows, cols, block_rows)


def matmul_fp8_blocks(a, a_scales, b, b_scales, output, bias=None, b_layout: str = "nk", stream=None) -> None:
    """output [m, n] = a [m, k] times the transpose of b [n, k] (b_layout "nk", a layer's forward
    product) or times b [k, n] ("kn": the gradient of a layer's input, from the same weights), plus
    bias [n] (fp32).

    a and b: float8_e4m3fn or float8_e5m2 blocks; the shapes of the scales tell blocks of a row from
    blocks of 128 x 128 (b [k, n] needs the latter). The sum is accumulated in fp32 and rounded once
    to output's type (fp32, bf16 or fp16)."""
    layout = LAYOUTS.get(b_layout)
    if layout is None:
        _refuse(f"b_layout must be one of {sorted(LAYOUTS)}")
    as_ = _matrix("a", a)
    device, (m, k) = a.device, a.shape
    bs = _matrix("b", b, device)
    b_rows, b_cols = b.shape
    n, b_k = (b_cols, b_rows) if layout else (b_rows, b_cols)
    if b_k != k:
        _refuse(f"b has shape {(b_rows, b_cols)} in layout {b_layout}, but k is {k}")
    os_ = _matrix("output", output, device, (m, n))
    at, bt, ot = _type("a", a, _FP8), _type("b", b, _FP8), _type("output", output, _FLOATS)
    a_block = _scales("a_scales", a_scales, device, m, k)
    b_block = _scales("b_scales", b_scales, device, b_rows, b_cols, not layout)
    if bias is not None and not (bias.dtype == _torch.float32 and bias.dim() == 1 and bias.numel() == n and
                                 bias.is_contiguous() and bias.device == device):
        _refuse(f"bias must be {n} contiguous fp32 values on {device}")
    _launch(device, stream, N.lib().tcc_matmul_fp8_blocks, a.data_ptr(), at, as_, a_scales.data_ptr(), a_block,
            b.data_ptr(), bt, bs, b_scales.data_ptr(), b_block, layout, None if bias is None else bias.data_ptr(),
            output.data_ptr(), ot, os_, m, n, k)


def _int8(name: str, q) -> None:
    if q.dtype != _torch.int8:
        _refuse(f"{name} must be int8")


def _pair(name: str, t, other, stride: int, other_stride: int) -> None:
    """An output of the input's type that is the input itself or no view of it from the same start."""
    if t.dtype != other.dtype:
        _refuse(f"{name} must have its input's type")
    if t.data_ptr() == other.data_ptr() and stride != other_stride:
        _refuse(f"{name} may be its input itself, not another view of it")


def activation_checkpoint_int8(x, y, q, scales, activation: str = "gelu", stream=None) -> None:
    """y = f(x), and x kept for the backward pass as INT8 blocks of 128 columns of a row.

    x, y: [rows, cols] of one type (fp32, bf16 or fp16), y may be x itself; q: int8 [rows, cols];
    scales: [rows, ceil(cols / 128)] bytes. activation: relu, gelu, gelu_tanh, silu, or identity,
    which keeps x alone (y None)."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        _refuse(f"activation must be one of {sorted(ACTIVATIONS)}")
    xs = _matrix("x", x)
    device, shape = x.device, x.shape
    xt = _type("x", x, _FLOATS)
    if activation == "identity":
        if y is not None:
            _refuse("the identity writes no y: pass None")
        ys, y_ptr = 0, None
    else:
        ys, y_ptr = _matrix("y", y, device, shape), y.data_ptr()
        _pair("y", y, x, ys, xs)
    qs = _matrix("q", q, device, shape)
    _int8("q", q)
    rows, cols = shape
    _scales("scales", scales, device, rows, cols, True, False)
    _launch(device, stream, N.lib().tcc_activation_checkpoint_int8, x.data_ptr(), xs, y_ptr, ys, xt, q.data_ptr(), qs,
            scales.data_ptr(), rows, cols, code)


def activation_backward_int8(grad_y, q, scales, grad_x, activation: str = "gelu", stream=None) -> None:
    """grad_x = grad_y * f'(x^), x^ the values that the checkpoint (q, scales) of
    activation_checkpoint_int8 stands for.

    grad_y, grad_x: [rows, cols] of one type (fp32, bf16 or fp16); grad_x may be grad_y itself.
    ReLU passes the gradient where x^ > 0."""
    code = ACTIVATIONS.get(activation)
    if code is None or activation == "identity":
        _refuse(f"activation must be one of {sorted(set(ACTIVATIONS) - {'identity'})}")
    gs = _matrix("grad_y", grad_y)
    device, shape = grad_y.device, grad_y.shape
    gt = _type("grad_y", grad_y, _FLOATS)
    xs = _matrix("grad_x", grad_x, device, shape)
    _pair("grad_x", grad_x, grad_y, xs, gs)
    qs = _matrix("q", q, device, shape)
    _int8("q", q)
    rows, cols = shape
    _scales("scales", scales, device, rows, cols, True, False)
    _launch(device, stream, N.lib().tcc_activation_backward_int8, grad_y.data_ptr(), gs, gt, q.data_ptr(), qs,
            scales.data_ptr(), grad_x.data_ptr(), xs, rows, cols, code)


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
    gs = _matrix("grad_y", grad_y)
    torch = _torch
    device, (rows, n) = grad_y.device, grad_y.shape
    gt = _type("grad_y", grad_y, _FLOATS)
    qs = _matrix("q", q, device)
    q_rows, k = q.shape
    if q_rows != rows:
        _refuse(f"q has {q_rows} rows, grad_y {rows}")
    _int8("q", q)
    ws = _matrix("grad_w", grad_w, device, (n, k))
    if grad_w.dtype != torch.float32:
        _refuse("grad_w must be fp32")
    _scales("scales", scales, device, rows, k, True, False)
    if workspace is None:
        need = weight_grad_int8_workspace_size(rows, n, k)
        if need:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream, device) if stream else torch.cuda.default_stream(device)
            with torch.cuda.stream(stream):  # nothing for None: the current stream
                workspace = torch.empty(need, dtype=torch.uint8, device=device)
    elif workspace.device != device or not workspace.is_contiguous():
        _refuse(f"the workspace must be contiguous on {device}")
    have = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _launch(device, stream, N.lib().tcc_weight_grad_int8, grad_y.data_ptr(), gt, gs, q.data_ptr(), qs,
            scales.data_ptr(), grad_w.data_ptr(), ws, rows, n, k, 1 if accumulate else 0,
            None if workspace is None else workspace.data_ptr(), have)
