"""The dense operators' argument checks and the 64-bit definitions their GPU tests compare with."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import tcc_spmm_b200 as T
from tests import dense8_util as D


def test_c_abi_refuses_before_any_device_work(native):
    size = C.c_uint64()
    quantize, product = native.tcc_quantize_blocks_fp8, native.tcc_matmul_fp8_blocks
    keep, back, grad = (native.tcc_activation_checkpoint_int8, native.tcc_activation_backward_int8,
                        native.tcc_weight_grad_int8)
    bad = [
        (quantize, (16, 3, 128, 16, 3, 128, 16, 4, 128, 1, None), b"reads fp32"),
        (quantize, (16, 0, 128, 16, 0, 128, 16, 4, 128, 1, None), b"writes e4m3"),
        (quantize, (16, 0, 128, 16, 3, 128, 16, 4, 128, 2, None), b"block_rows"),
        (quantize, (None, 0, 128, 16, 3, 128, 16, 4, 128, 1, None), b"requires x"),
        (quantize, (16, 0, 127, 16, 3, 128, 16, 4, 128, 1, None), b"x: stride"),
        (quantize, (16, 0, 128, 16, 3, 127, 16, 4, 128, 1, None), b"q: stride"),
        (quantize, (17, 0, 128, 16, 3, 128, 16, 4, 128, 1, None), b"aligned"),
        (quantize, (16, 0, 1 << 62, 16, 3, 128, 16, 4, 128, 1, None), b"x: stride"),
        (quantize, (16, 0, 128, 16, 3, 128, None, 4, 128, 1, None), b"requires scales"),
        (product, (16, 0, 128, 16, 1, 16, 3, 128, 16, 128, 0, None, 16, 0, 128, 4, 128, 128, None), b"multiplies"),
        (product, (16, 3, 128, 16, 1, 16, 3, 128, 16, 128, 0, None, 16, 3, 128, 4, 128, 128, None), b"writes fp32"),
        (product, (16, 3, 128, 16, 3, 16, 3, 128, 16, 128, 0, None, 16, 0, 128, 4, 128, 128, None), b"block rows"),
        (product, (16, 3, 128, 16, 1, 16, 3, 128, 16, 1, 1, None, 16, 0, 128, 4, 128, 128, None), b"128 x 128"),
        (product, (16, 3, 128, 16, 1, 16, 3, 128, 16, 1, 2, None, 16, 0, 128, 4, 128, 128, None), b"layout"),
        (product, (16, 3, 127, 16, 1, 16, 3, 128, 16, 128, 0, None, 16, 0, 128, 4, 128, 128, None), b"a: stride"),
        (product, (16, 3, 128, 16, 1, 16, 3, 127, 16, 128, 0, None, 16, 0, 128, 4, 128, 128, None), b"b: stride"),
        (product, (16, 3, 128, 16, 1, 16, 3, 128, 16, 128, 0, None, 16, 0, 127, 4, 128, 128, None), b"output: stride"),
        (product, (16, 3, 128, 16, 1, 16, 3, 128, 16, 128, 0, 18, 16, 0, 128, 4, 128, 128, None), b"aligned"),
        (product, (16, 3, 128, None, 1, 16, 3, 128, 16, 128, 0, None, 16, 0, 128, 4, 128, 128, None), b"scales"),
        (product, (16, 3, 128, 16, 1, 16, 3, 128, 16, 128, 0, None, None, 0, 128, 4, 128, 128, None), b"output"),
        (keep, (16, 128, 16, 128, 3, 16, 128, 16, 4, 128, 1, None), b"takes fp32"),
        (keep, (16, 128, 16, 128, 0, 16, 128, 16, 4, 128, 5, None), b"unknown activation"),
        (keep, (16, 128, 16, 128, 0, 16, 128, 16, 4, 128, 4, None), b"null y"),
        (keep, (16, 128, None, 128, 0, 16, 128, 16, 4, 128, 1, None), b"requires y"),
        (back, (16, 128, 0, 16, 128, 16, 16, 128, 4, 128, 4, None), b"unknown activation"),
        (back, (16, 128, 0, 16, 127, 16, 16, 128, 4, 128, 1, None), b"q: stride"),
        (back, (16, 128, 0, 16, 128, None, 16, 128, 4, 128, 1, None), b"requires scales"),
        (grad, (16, 3, 128, 16, 128, 16, 16, 128, 4, 128, 128, 0, None, 0, None), b"in fp32"),
        (grad, (16, 0, 127, 16, 128, 16, 16, 128, 4, 128, 128, 0, None, 0, None), b"grad_y: stride"),
        (grad, (16, 0, 128, 16, 128, 16, 18, 128, 4, 128, 128, 0, None, 0, None), b"aligned grad_w"),
        (grad, (16, 0, 128, 16, 128, 16, 16, 128, 1 << 20, 128, 128, 0, None, 0, None), b"workspace"),
        (grad, (16, 0, 128, 16, 128, 16, 16, 128, 1 << 20, 128, 128, 0, 24, 1 << 40, None), b"workspace"),
        (native.tcc_weight_grad_int8_workspace_size, (4, 128, 128, None), b"output"),
    ]
    for call, args, message in bad:
        assert call(*args) == 1, (call.__name__, args)
        assert message in native.tcc_last_error(), (call.__name__, args, native.tcc_last_error())
    # sizes of zero need no memory
    assert quantize(None, 0, 0, None, 3, 0, None, 0, 128, 1, None) == 0
    assert product(None, 3, 0, None, 1, None, 3, 0, None, 128, 0, None, None, 0, 0, 0, 128, 128, None) == 0
    assert keep(None, 0, None, 0, 0, None, 0, None, 4, 0, 1, None) == 0
    assert back(None, 0, 0, None, 0, None, None, 0, 0, 4, 1, None) == 0
    assert grad(None, 0, 0, None, 0, None, None, 0, 4, 0, 128, 0, None, 0, None) == 0
    assert native.tcc_weight_grad_int8_workspace_size(4, 0, 128, C.byref(size)) == 0 and size.value == 0


def test_c_abi_refuses_sizes_that_no_tile_count_holds(native):
    """Sizes are rounded up to whole blocks and tiles of up to 256 in 32 bits."""
    size, big, wide = C.c_uint64(), 0xFFFFFF01, 1 << 32
    quantize, product, grad = native.tcc_quantize_blocks_fp8, native.tcc_matmul_fp8_blocks, native.tcc_weight_grad_int8
    keep, back = native.tcc_activation_checkpoint_int8, native.tcc_activation_backward_int8
    bad = [
        (quantize, (16, 0, wide, 16, 3, wide, 16, 1, big, 1, None)),
        (quantize, (16, 0, 1, 16, 3, 1, 16, big, 1, 128, None)),
        (keep, (16, wide, 16, wide, 0, 16, wide, 16, 1, 0xFFFFFFFF, 1, None)),
        (back, (16, wide, 0, 16, wide, 16, 16, wide, 1, 0xFFFFFFFF, 1, None)),
        (product, (16, 3, 1, 16, 1, 16, 3, 1, 16, 128, 0, None, 16, 0, 1, big, 1, 1, None)),
        (product, (16, 3, 1, 16, 1, 16, 3, 1, 16, 128, 0, None, 16, 0, wide, 1, big, 1, None)),
        (product, (16, 3, wide, 16, 1, 16, 3, wide, 16, 128, 0, None, 16, 0, 1, 1, 1, big, None)),
        (grad, (16, 0, 1, 16, 1, 16, 16, 1, 0xFFFFFFFF, 1, 1, 0, 16, 1 << 40, None)),
        (grad, (16, 0, 1, 16, wide, 16, 16, wide, 1, 1, big, 0, 16, 1 << 40, None)),
        (native.tcc_weight_grad_int8_workspace_size, (big, 128, 128, C.byref(size))),
        (native.tcc_weight_grad_int8_workspace_size, (128, 128, big, C.byref(size))),
    ]
    for call, args in bad:
        assert call(*args) == 1, (call.__name__, args)
        assert b"too large" in native.tcc_last_error(), (call.__name__, args, native.tcc_last_error())
    assert native.tcc_weight_grad_int8_workspace_size(0xFFFFFF00, 128, 128, C.byref(size)) == 0
    for sizes in ((-1, 128, 128), (1 << 32, 128, 128), (128, 128, big)):
        with pytest.raises(T.InvalidArgument):
            T.weight_grad_int8_workspace_size(*sizes)


def test_packed_call_refuses_unknown_operators(native):
    for op in (-1, 5):
        assert native.tcc_dense8_call(op, bytes(8 * 19)) == 1


def test_python_refuses_cpu_tensors():
    x = torch.zeros(4, 128)
    q = torch.zeros(4, 128, dtype=torch.int8)
    s = torch.zeros(4, 1, dtype=torch.uint8)
    for call in (lambda: T.quantize_blocks_fp8(x, q.view(torch.float8_e4m3fn), s),
                 lambda: T.matmul_fp8_blocks(q.view(torch.float8_e4m3fn), s, q.view(torch.float8_e4m3fn), s, x),
                 lambda: T.activation_checkpoint_int8(x, x.clone(), q, s),
                 lambda: T.activation_backward_int8(x, q, s, x.clone()),
                 lambda: T.weight_grad_int8(x, q, s, torch.zeros(128, 128))):
        with pytest.raises(T.InvalidArgument):
            call()


@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
def test_definition_rounds_as_the_type_does(kind):
    """The 64-bit definition of an element's rounding is torch's conversion, on every tie and border."""
    x = torch.cat([torch.arange(-4096, 4097) * 2.0 ** -4, torch.arange(-600, 601) * 2.0 ** -12, torch.tensor([448.0])])
    x = x.clamp(-D.LARGEST[kind], D.LARGEST[kind])
    x = torch.nn.functional.pad(x, (0, -len(x) % 127)).reshape(-1, 127)
    x = torch.cat([x, torch.full((x.shape[0], 1), D.LARGEST[kind])], 1)  # scale 1 in every block
    q, scales = D.quantize(x, kind)
    assert (scales == 127).all()
    assert torch.equal(q, x.to(D.FP8[kind]).double())


def test_definition_of_the_scale():
    x = torch.tensor([[127.0], [127.0001], [63.5], [0.0], [1e-45], [3e38], [float("inf")], [float("nan")]])
    _, scales = D.quantize(x, "int8")
    assert scales.flatten().tolist() == [127, 128, 126, 127, 1, 248, 255, 255]
