"""Dense operators on 8-bit blocks: the quantizer to 8-bit floating point, the product of two such
matrices, and INT8 activation checkpoints with the gradients computed from them.

A matrix is cut into blocks of 128 columns of a row, or of 128 x 128 elements; every block has one
power-of-two scale, kept as its biased exponent byte (torch.uint8, or torch.float8_e8m0fnu; value
2^(byte - 127)). include/tcc_spmm_b200.h states the rule.

Every operand is a 2-D CUDA tensor of one device whose last dimension has stride 1; rows may be
any distance apart, and the tensors of a call share no memory but where it says so. The calls enqueue work on `stream` (default: torch's current stream of that
device), never synchronise, and raise InvalidArgument for tensors that do not fit together. They
write into tensors that the caller gives. The reference has no counterpart.

The checks run on every call, and a small operator takes a few microseconds, so they are written
for speed: plain comparisons, with messages formed only when one fails, and one packed argument
for the library.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional

from . import _native as N
from .api import InvalidArgument, _check, _stream_handle

BLOCK = 128
ACTIVATIONS = {"relu": 0, "gelu": 1, "gelu_tanh": 2, "silu": 3, "identity": 4}
LAYOUTS = {"nk": 0, "kn": 1}
_LARGEST = 0xFFFFFF00  # rows or columns: the kernels round them up to whole tiles in 32 bits

# torch, its raw-stream and current-device queries, and the type codes, once an operator is used
_torch = _raw_stream = _current_device = _call = None
_FLOATS: dict = {}
_FP8: dict = {}
_SCALES: set = set()


def _load():
    global _torch, _raw_stream, _current_device, _call
    import torch

    _FLOATS.update({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2})
    _FP8.update({torch.float8_e4m3fn: 3, torch.float8_e5m2: 4})
    _SCALES.update((torch.uint8, torch.float8_e8m0fnu))
    _raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
    _call = N.lib().tcc_dense8_call
    _torch = torch


def _refuse(message: str):
    raise InvalidArgument(message)


def _matrix(name: str, t, device: int = -1) -> tuple:
    """(rows, columns, row stride in elements, device) of a 2-D CUDA operand, on `device` if that is given."""
    try:
        rows, cols = t.shape
        row_stride, col_stride = t.stride()
        on = t.get_device()
    except (AttributeError, TypeError, ValueError, RuntimeError):
        _refuse(f"{name} must be a 2-D CUDA tensor")
    if on < 0:
        _refuse(f"{name} must be a CUDA tensor")
    if on != device and device >= 0:
        _refuse(f"{name} is on cuda:{on}, expected cuda:{device}")
    if rows > _LARGEST or cols > _LARGEST:
        _refuse(f"{name} is too large")
    if col_stride != 1 and cols > 1:
        _refuse(f"{name} must have stride 1 along its last dimension")
    if rows <= 1:  # no second row: the distance to it says nothing
        return rows, cols, (cols + 15) & -16, on
    if row_stride < cols:
        _refuse(f"the rows of {name} overlap")
    return rows, cols, row_stride, on


def _shaped(name: str, t, rows: int, cols: int, device: int) -> int:
    """The row stride of a 2-D CUDA operand that must have this shape."""
    try:
        row_stride, col_stride = t.stride()
        if col_stride == 1 and row_stride >= cols and rows > 1 and t.shape == (rows, cols) and t.get_device() == device:
            return row_stride
    except (AttributeError, TypeError, ValueError, RuntimeError):
        pass
    r, c, stride, _ = _matrix(name, t, device)  # the special cases, and the messages
    if r != rows or c != cols:
        _refuse(f"{name} has shape {(r, c)}, expected {(rows, cols)}")
    return stride


def _scales(name: str, t, device: int, rows: int, cols: int, row_blocks: bool = True, square_blocks: bool = True) -> int:
    """Checks the scale bytes of a [rows, cols] matrix and returns the rows per block."""
    wide = (cols + 127) >> 7
    try:
        if t.dtype in _SCALES and t.get_device() == device and t.is_contiguous():
            shape = t.shape
            if row_blocks and shape == (rows, wide):
                return 1
            if square_blocks and shape == ((rows + 127) >> 7, wide):
                return BLOCK
    except (AttributeError, TypeError):
        _refuse(f"{name} must be a CUDA tensor")
    if t.dtype not in _SCALES:
        _refuse(f"{name} must hold scale bytes (uint8 or float8_e8m0fnu)")
    if t.get_device() != device:
        _refuse(f"{name} is on {t.device}, expected cuda:{device}")
    want = [(rows, wide)] * row_blocks + [((rows + 127) >> 7, wide)] * square_blocks
    _refuse(f"{name} has shape {tuple(t.shape)}, expected contiguous {' or '.join(map(str, want))}")


def _type(name: str, t, types: dict) -> int:
    code = types.get(t.dtype)
    if code is None:
        _refuse(f"{name} has unsupported type {t.dtype}")
    return code


_QUANTIZE, _PRODUCT, _CHECKPOINT, _BACKWARD, _WEIGHT_GRAD = range(5)  # tcc_dense8_call's operators
_words = [struct.Struct(f"{n}Q").pack for n in (11, 19, 12, 12, 15)]


def _launch(device: int, stream, op: int, *args) -> None:
    """Operator `op` with these arguments and the stream, with `device` current."""
    raw = _raw_stream(device) if stream is None else _stream_handle(stream)
    words = _words[op](*args, raw)
    if device == _current_device():
        status = _call(op, words)
    else:
        with _torch.cuda.device(device):
            status = _call(op, words)
    if status:
        _check(status)


def quantize_blocks_fp8(x, q, scales, block_rows: int = 1, stream=None) -> None:
    """q, scales = the blocks of x [rows, cols] (fp32, bf16 or fp16) in 8-bit floating point.

    q: [rows, cols] of float8_e4m3fn or float8_e5m2; scales: [ceil(rows / block_rows),
    ceil(cols / 128)] bytes; block_rows 1 (activations) or 128 (weights). matmul_fp8_blocks runs
    fastest on a q whose rows start on 16 bytes."""
    if _torch is None:
        _load()
    rows, cols, xs, device = _matrix("x", x)
    qs = _shaped("q", q, rows, cols, device)
    xt, qt = _type("x", x, _FLOATS), _type("q", q, _FP8)
    if block_rows != 1 and block_rows != BLOCK:
        _refuse("block_rows must be 1 or 128")
    _scales("scales", scales, device, rows, cols, block_rows == 1, block_rows == BLOCK)
    _launch(device, stream, _QUANTIZE, x.data_ptr(), xt, xs, q.data_ptr(), qt, qs,
            scales.data_ptr(), rows, cols, block_rows)


def matmul_fp8_blocks(a, a_scales, b, b_scales, output, bias=None, b_layout: str = "nk", stream=None) -> None:
    """output [m, n] = a [m, k] times the transpose of b [n, k] (b_layout "nk", a layer's forward
    product) or times b [k, n] ("kn": the gradient of a layer's input, from the same weights), plus
    bias [n] (fp32).

    a and b: float8_e4m3fn or float8_e5m2 blocks; the shapes of the scales tell blocks of a row from
    blocks of 128 x 128 (b [k, n] needs the latter). The sum is accumulated in fp32 and rounded once
    to output's type (fp32, bf16 or fp16). Rows of a or b that do not start on 16 bytes run on a
    kernel without tensor cores, a hundred times slower for large matrices: give 8-bit operands a row
    stride that is a multiple of 16."""
    if _torch is None:
        _load()
    layout = LAYOUTS.get(b_layout)
    if layout is None:
        _refuse(f"b_layout must be one of {sorted(LAYOUTS)}")
    m, k, as_, device = _matrix("a", a)
    b_rows, b_cols, bs, _ = _matrix("b", b, device)
    n, b_k = (b_cols, b_rows) if layout else (b_rows, b_cols)
    if b_k != k:
        _refuse(f"b has shape {(b_rows, b_cols)} in layout {b_layout}, but k is {k}")
    os_ = _shaped("output", output, m, n, device)
    at, bt, ot = _type("a", a, _FP8), _type("b", b, _FP8), _type("output", output, _FLOATS)
    a_block = _scales("a_scales", a_scales, device, m, k)
    b_block = _scales("b_scales", b_scales, device, b_rows, b_cols, not layout)
    if bias is not None and not (isinstance(bias, _torch.Tensor) and bias.dtype == _torch.float32 and tuple(bias.shape) == (n,) and
                                 bias.is_contiguous() and bias.get_device() == device):
        _refuse(f"bias must be {n} contiguous fp32 values on cuda:{device}")
    _launch(device, stream, _PRODUCT, a.data_ptr(), at, as_, a_scales.data_ptr(), a_block,
            b.data_ptr(), bt, bs, b_scales.data_ptr(), b_block, layout, 0 if bias is None else bias.data_ptr(),
            output.data_ptr(), ot, os_, m, n, k)


def _pair(name: str, t, other, stride: int, other_stride: int) -> None:
    """An output of the input's type that is the input itself or no view of it from the same start."""
    if t.dtype != other.dtype:
        _refuse(f"{name} must have its input's type")
    if stride != other_stride and t.data_ptr() == other.data_ptr():
        _refuse(f"{name} may be its input itself, not another view of it")


def activation_checkpoint_int8(x, y, q, scales, activation: str = "gelu", stream=None) -> None:
    """y = f(x), and x kept for the backward pass as INT8 blocks of 128 columns of a row.

    x, y: [rows, cols] of one type (fp32, bf16 or fp16), y may be x itself; q: int8 [rows, cols];
    scales: [rows, ceil(cols / 128)] bytes. activation: relu, gelu, gelu_tanh, silu, or identity,
    which keeps x alone (y None)."""
    if _torch is None:
        _load()
    code = ACTIVATIONS.get(activation)
    if code is None:
        _refuse(f"activation must be one of {sorted(ACTIVATIONS)}")
    rows, cols, xs, device = _matrix("x", x)
    xt = _type("x", x, _FLOATS)
    if activation == "identity":
        if y is not None:
            _refuse("the identity writes no y: pass None")
        ys = y_ptr = 0
    else:
        ys, y_ptr = _shaped("y", y, rows, cols, device), y.data_ptr()
        _pair("y", y, x, ys, xs)
    qs = _shaped("q", q, rows, cols, device)
    if q.dtype != _torch.int8:
        _refuse("q must be int8")
    _scales("scales", scales, device, rows, cols, True, False)
    _launch(device, stream, _CHECKPOINT, x.data_ptr(), xs, y_ptr, ys, xt, q.data_ptr(), qs,
            scales.data_ptr(), rows, cols, code)


def activation_backward_int8(grad_y, q, scales, grad_x, activation: str = "gelu", stream=None) -> None:
    """grad_x = grad_y * f'(x^), x^ the values that the checkpoint (q, scales) of
    activation_checkpoint_int8 stands for.

    grad_y, grad_x: [rows, cols] of one type (fp32, bf16 or fp16); grad_x may be grad_y itself.
    ReLU passes the gradient where x^ > 0."""
    if _torch is None:
        _load()
    code = ACTIVATIONS.get(activation)
    if code is None or activation == "identity":
        _refuse(f"activation must be one of {sorted(set(ACTIVATIONS) - {'identity'})}")
    rows, cols, gs, device = _matrix("grad_y", grad_y)
    gt = _type("grad_y", grad_y, _FLOATS)
    xs = _shaped("grad_x", grad_x, rows, cols, device)
    _pair("grad_x", grad_x, grad_y, xs, gs)
    qs = _shaped("q", q, rows, cols, device)
    if q.dtype != _torch.int8:
        _refuse("q must be int8")
    _scales("scales", scales, device, rows, cols, True, False)
    _launch(device, stream, _BACKWARD, grad_y.data_ptr(), gs, gt, q.data_ptr(), qs,
            scales.data_ptr(), grad_x.data_ptr(), xs, rows, cols, code)


def weight_grad_int8_workspace_size(rows: int, n: int, k: int) -> int:
    """Bytes of workspace that weight_grad_int8 needs for grad_y [rows, n] and a checkpoint [rows, k]."""
    if not all(0 <= size <= _LARGEST for size in (rows, n, k)):
        _refuse(f"rows, n and k must be between 0 and {_LARGEST}")
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
    if _torch is None:
        _load()
    rows, n, gs, device = _matrix("grad_y", grad_y)
    gt = _type("grad_y", grad_y, _FLOATS)
    q_rows, k, qs, _ = _matrix("q", q, device)
    if q_rows != rows:
        _refuse(f"q has {q_rows} rows, grad_y {rows}")
    if q.dtype != _torch.int8:
        _refuse("q must be int8")
    ws = _shaped("grad_w", grad_w, n, k, device)
    if grad_w.dtype != _torch.float32:
        _refuse("grad_w must be fp32")
    _scales("scales", scales, device, rows, k, True, False)
    if workspace is None:
        need = weight_grad_int8_workspace_size(rows, n, k)
        if need:
            cuda = _torch.cuda
            if stream is not None and not isinstance(stream, cuda.Stream):  # a handle, or what holds one
                handle = _stream_handle(stream)
                stream = cuda.ExternalStream(handle, device) if handle else cuda.default_stream(device)
            with cuda.stream(stream):  # nothing for None: the current stream
                workspace = _torch.empty(need, dtype=_torch.uint8, device=grad_y.device)
    elif (not isinstance(workspace, _torch.Tensor) or workspace.get_device() != device or
          not workspace.is_contiguous()):
        _refuse(f"the workspace must be contiguous on cuda:{device}")
    have = 0 if workspace is None else workspace.numel() * workspace.element_size()
    _launch(device, stream, _WEIGHT_GRAD, grad_y.data_ptr(), gt, gs, q.data_ptr(), qs,
            scales.data_ptr(), grad_w.data_ptr(), ws, rows, n, k, 1 if accumulate else 0,
            0 if workspace is None else workspace.data_ptr(), have)
