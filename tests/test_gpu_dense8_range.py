"""The dense operators on 8-bit blocks at the ends of the number range, against their definitions in 64 bits."""
from __future__ import annotations

import pytest
import torch

import tcc_spmm_b200 as T
from tests import dense8_util as D

pytestmark = pytest.mark.gpu

KINDS = ["relu", "silu", "gelu", "gelu_tanh"]


def checkpoint(x, kind):
    y = None if kind == "identity" else torch.empty_like(x)
    q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
    scales = torch.empty(x.shape[0], -(-x.shape[1] // 128), dtype=torch.uint8, device="cuda")
    T.activation_checkpoint_int8(x, y, q, scales, activation=kind)
    return y, q, scales


def large_rows(dtype):
    """Blocks whose largest element runs up to the type's ends: rows of one value, of its negative, and a row that
    is masked with the lowest value in places."""
    top = torch.finfo(dtype).max
    sizes = [v for v in (1e4, 1e10, 2.0 ** 66, 1e25, 3e38, top) if v <= top]
    x = torch.zeros(3 * len(sizes), 200, device="cuda")
    for i, v in enumerate(sizes):
        x[3 * i] = v
        x[3 * i + 1] = -v
        x[3 * i + 2] = torch.linspace(-2, 2, 200, device="cuda")
        x[3 * i + 2, ::7] = -v
    return x.to(dtype)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_functions_of_large_values(dtype, kind):
    """From 1e4 on every function is x or 0, and its slope 1 or 0; a value that is kept as zero has the slope of
    zero. An element may stand for 2^128, which no float holds: its slope is still the definition's."""
    x = large_rows(D.TYPES[dtype])
    y, q, scales = checkpoint(x, kind)
    want_q, want_scales = D.quantize(x, "int8")
    assert torch.equal(scales, want_scales) and torch.equal(q.double(), want_q)
    far = x.abs() >= 1e4
    assert torch.equal(y[far], x[far].clamp(min=0))
    want = D.activation(x.double(), kind)
    # |x| <= 2 elsewhere: a dozen fp32 roundings and the type's own
    assert ((y.double() - want).abs()[~far] <= (D.half_step(x.dtype) + 32 * D.U) * want.abs()[~far] + 2.0 ** -24).all()
    xh = D.values(q, scales)
    assert (xh[far].abs() >= 9e3).all()  # kept within half a step, a 2^-7th of the block's largest at most
    for grad in (torch.float32, torch.bfloat16, torch.float16):
        dy = D.make(*x.shape, grad, 3)
        dx = torch.empty_like(dy)
        T.activation_backward_int8(dy, q, scales, dx, activation=kind)
        assert torch.equal(dx[far], torch.where(xh > 0, dy, torch.zeros_like(dy))[far])
        zero = xh == 0
        want = dy.double()[zero] * (0.0 if kind == "relu" else 0.5)
        least = 2.0 ** -25 if grad == torch.float16 else 2.0 ** -130
        assert ((dx.double()[zero] - want).abs() <= (D.half_step(grad) + 32 * D.U) * want.abs() + least).all()
        assert not dx.isnan().any()


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("n", [8, 200])  # one CTA a tile of dW, or two
@pytest.mark.parametrize("grad", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_weight_grad_of_large_values(dtype, grad, n, aligned):
    """Large elements meet zeros of dy (sums that leave them out) and, one to a sum, small values of dy, with which
    even 2^128 gives a finite product. A sum of one product is exact in fp32 (8 bits of x^ by up to 11 of dy)."""
    x = large_rows(D.TYPES[dtype])
    _, q, scales = checkpoint(x, "identity")
    rows, k = x.shape
    dy = torch.zeros(rows, n)
    for j in range(n):
        if j < rows:
            dy[j, j] = 0.75 * 2.0 ** -8 * (-1) ** j
    off = 0 if aligned else 1
    held = D.strided(rows, n, D.TYPES[grad], D.up16(n) + off, off)
    held.copy_(dy)
    kept = D.strided(rows, k, torch.int8, D.up16(k) + off, off)
    kept.copy_(q)
    dw = torch.full((n, k), float("nan"), device="cuda")
    T.weight_grad_int8(held, kept, scales, dw)
    xh = D.values(q, scales)
    want = dy.cuda().double().t() @ xh
    assert xh.abs().max() == 2.0 ** 128 and torch.equal(dw.double(), want)
    T.weight_grad_int8(held, kept, scales, dw, accumulate=True)
    assert torch.equal(dw.double(), 2 * want)


@pytest.mark.parametrize("grad", ["fp32", "bf16"])
@pytest.mark.parametrize("byte", [0, 1, 2, 3])
def test_weight_grad_of_the_smallest_scales(byte, grad):
    """The scales at the lower end (0 is the format's, the quantizers write no less than 1) with a dy that brings
    the sums back into range: every product is exact."""
    rows, n, k = 70, 20, 255
    q = (torch.arange(rows * k).reshape(rows, k) % 255 - 127).to(torch.int8).cuda()
    scales = torch.full((rows, 2), byte, dtype=torch.uint8, device="cuda")
    dy = torch.zeros(rows, n, device="cuda")
    dy[:, 0], dy[3, 1], dy[69, 19] = 2.0 ** 60, -2.0 ** 100, 2.0 ** 126
    dw = torch.empty(n, k, device="cuda")
    T.weight_grad_int8(dy.to(D.TYPES[grad]), q, scales, dw)
    want = dy.double().t() @ D.values(q, scales)
    assert torch.equal(dw.double(), want)


# ---- product --------------------------------------------------------------------------------------
# Every kernel of the product: up to 8 and up to 16 rows, tiles, tiles that share k, [k, n] weights, and operands
# whose rows are off 16 bytes.
FORMS = [(3, 40, 300, "nk", True), (13, 40, 300, "nk", True), (130, 140, 300, "nk", True), (140, 150, 1100, "nk", True),
         (130, 140, 300, "kn", True), (130, 140, 1100, "kn", True), (3, 140, 300, "nk", False), (130, 70, 300, "kn", False)]


def blocks(rows, cols, kind, aligned, q64):
    held = D.strided(rows, cols, D.FP8[kind], D.up16(cols) if aligned else cols + 1, 0 if aligned else 1)
    held.view(torch.uint8).copy_(q64.float().to(D.FP8[kind]).view(torch.uint8))
    return held


def small_elements(rows, cols, seed):
    """Whole numbers from -2 to 2."""
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-2, 3, (rows, cols), generator=gen).double().cuda()


@pytest.mark.parametrize("m,n,k,layout,aligned", FORMS)
def test_product_of_extreme_scales(m, n, k, layout, aligned):
    """Scales whose product no float holds, in either direction, beside sums that are zero or bring it back. Every
    sum is a small whole number times a power of two: exact in fp32."""
    qa, qb = small_elements(m, k, 1), small_elements(n, k, 2)
    kb, nb = -(-k // 128), -(-n // 128)
    for kind, factor, a_byte, b_byte in (("e4m3", 0, 254, 254), ("e4m3", 1, 1, 1), ("e5m2", 28672, 52, 52), ("e4m3", 224, 1, 254),
                                         ("e4m3", 224, 254, 1), ("e4m3", 224, 200, 60), ("e4m3", 1, 0, 254)):
        a64, b64 = qa * max(factor, 1), qb * max(factor, 1)
        if factor == 0:  # 2^254: only zeros may meet
            a64[:, ::2] = 0
            b64[:, 1::2] = 0
        a = blocks(m, k, kind, aligned, a64)
        b = blocks(n, k, kind, aligned, b64) if layout == "nk" else blocks(k, n, kind, aligned, b64.t())
        sa = torch.full((m, kb), a_byte, dtype=torch.uint8, device="cuda")
        sb = torch.full((nb, kb) if layout == "nk" else (kb, nb), b_byte, dtype=torch.uint8, device="cuda")
        y = torch.full((m, n), float("nan"), device="cuda")
        T.matmul_fp8_blocks(a, sa, b, sb, y, b_layout=layout)
        want = (a64 @ b64.t()) * 2.0 ** (a_byte + b_byte - 254)
        assert torch.equal(y, want.float()), (kind, a_byte, b_byte)


@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
@pytest.mark.parametrize("m,n,k,layout,aligned", FORMS)
def test_product_of_large_values(m, n, k, layout, aligned, kind):
    """The largest finite rows, whose elements stand for 2^128: zeros of b leave them out, and a small b brings them
    into range."""
    x = torch.zeros(m, k, device="cuda")
    x[0::3] = torch.finfo(torch.float32).max
    x[1::3, ::5] = torch.finfo(torch.float32).min
    sa = torch.empty(m, -(-k // 128), dtype=torch.uint8, device="cuda")
    a = blocks(m, k, kind, aligned, torch.zeros(m, k))
    T.quantize_blocks_fp8(x, a, sa)
    want_q, want_s = D.quantize(x, kind)
    assert torch.equal(a.double(), want_q) and torch.equal(sa, want_s)
    b64 = torch.zeros(n, k, device="cuda", dtype=torch.float64)
    b64[::2, 35], b64[1::4, 260] = 1.0, -0.5
    nb, kb = -(-n // 128), -(-k // 128)
    b = blocks(n, k, "e4m3", aligned, b64) if layout == "nk" else blocks(k, n, "e4m3", aligned, b64.t())
    sb = torch.full((nb, kb) if layout == "nk" else (kb, nb), 127 - 20, dtype=torch.uint8, device="cuda")
    y = torch.full((m, n), float("nan"), device="cuda")
    T.matmul_fp8_blocks(a, sa, b, sb, y, b_layout=layout)
    want = D.values(a, sa) @ b64.t() * 2.0 ** -20
    assert torch.equal(y.double(), want) and want.abs().max() == 2.0 ** 108
