"""The dense operators on 8-bit blocks against their definitions in 64 bits."""
from __future__ import annotations

import math

import pytest
import torch

import tcc_spmm_b200 as T
from tests import dense8_util as D

pytestmark = pytest.mark.gpu


def same(got, want):
    return torch.equal(torch.nan_to_num(got.double(), nan=1e300), torch.nan_to_num(want.double(), nan=1e300))


# ---- quantizer ----------------------------------------------------------------------------------
SHAPES = [(1, 1), (1, 128), (3, 127), (130, 129), (257, 384), (64, 1000), (5, 4100), (1000, 16)]


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_blocks(rows, cols, dtype, kind, block_rows):
    x = D.make(rows, cols, D.TYPES[dtype], rows + cols)
    for stride, offset, x_stride, x_offset in ((D.up16(cols), 0, D.up16(cols), 0), (cols + 3, 1, cols + 5, 1),
                                               (D.up16(cols) + 8, 8, D.up16(cols) + 4, 4),
                                               (D.up16(cols) + 4, 4, D.up16(cols) + 2, 2)):
        q = D.strided(rows, cols, D.FP8[kind], stride, offset)
        scales = torch.zeros(-(-rows // block_rows), -(-cols // 128), dtype=torch.uint8, device="cuda")
        xs = D.strided(rows, cols, x.dtype, x_stride, x_offset)
        xs.copy_(x)
        T.quantize_blocks_fp8(xs, q, scales, block_rows=block_rows)
        want, bytes_ = D.quantize(x, kind, block_rows)
        assert torch.equal(scales, bytes_)
        assert same(q, want)


def test_quantize_leaves_the_rest_alone():
    """Padding between the rows and behind the last row keeps its bytes."""
    rows, cols, stride = 37, 200, 224
    whole = torch.full((rows + 2, stride), 0x55, dtype=torch.uint8, device="cuda")
    q = whole[1:rows + 1, :cols].view(torch.float8_e4m3fn)
    scales = torch.full((rows + 1, 2), 0x55, dtype=torch.uint8, device="cuda")
    T.quantize_blocks_fp8(D.make(rows, cols, torch.bfloat16, 1), q, scales[:rows])
    assert (whole[1:rows + 1, cols:] == 0x55).all() and (whole[0] == 0x55).all() and (whole[-1] == 0x55).all()
    assert (scales[rows] == 0x55).all()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
def test_quantize_extremes(kind, block_rows):
    """The largest and smallest values, the borders of the scale rule, and blocks that are not finite."""
    big = torch.finfo(torch.float32).max
    tiny = 2.0 ** -149
    edge = D.LARGEST[kind]
    rows = [big, tiny, 2.0 ** -126, 2.0 ** -130, edge, math.nextafter(edge, 1e9) * (1 + 2 ** -22), edge * 2.0 ** -60,
            edge * 2.0 ** -126, float("inf"), float("nan"), -float("inf"), -big, 0.0]
    x = torch.zeros(len(rows) * (1 if block_rows == 1 else 128), 256, device="cuda")
    for i, v in enumerate(rows):
        r = i if block_rows == 1 else 128 * i + 77
        x[r, 130] = v
        x[r, 131:140] = torch.linspace(-1, 1, 9, device="cuda") * (abs(v) if math.isfinite(v) else 1.0)
        x[r, 0] = 1.0
    q = torch.empty(x.shape, dtype=torch.uint8, device="cuda").view(D.FP8[kind])
    scales = torch.empty(len(rows), 2, dtype=torch.uint8, device="cuda")
    T.quantize_blocks_fp8(x, q, scales, block_rows=block_rows)
    want, bytes_ = D.quantize(x, kind, block_rows)
    assert torch.equal(scales, bytes_)
    bad = D.spread(scales, block_rows, *x.shape).isnan()
    assert q[bad].double().isnan().all() and bad.sum() == 3 * 128 * block_rows
    assert torch.equal(q.double()[~bad], want[~bad])


# ---- product ------------------------------------------------------------------------------------
def product_case(m, n, k, a_kind="e4m3", b_kind="e4m3", layout="nk", a_rows=1, b_rows=128, seed=0, aligned=True):
    def operand(rows, cols, kind, block_rows, seed, scale):
        x = D.make(rows, cols, torch.float32, seed, scale=scale)
        q, scales = D.quantize(x, kind, block_rows)
        held = D.strided(rows, cols, D.FP8[kind], D.up16(cols) if aligned else cols + 1, 0 if aligned else 1)
        held.view(torch.uint8).copy_(q.float().to(D.FP8[kind]).view(torch.uint8))
        return held, scales.contiguous()

    a, a_scales = operand(m, k, a_kind, a_rows, seed, 1.0)
    b, b_scales = operand(*((n, k) if layout == "nk" else (k, n)), b_kind, b_rows, seed + 1, 0.1)
    av = D.values(a, a_scales, a_rows)
    bv = D.values(b, b_scales, b_rows)
    bv = bv.t() if layout == "nk" else bv
    return a, a_scales, b, b_scales, av @ bv, av.abs() @ bv.abs()


def check_product(out, want, size, k, bias=None):
    """|error| <= what k + 4 additions and the last rounding may lose: half a step of the type, which below 2^-14
    is 2^-25 for fp16."""
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    limit = (k + 4) * D.U * size + D.half_step(out.dtype) * (want.abs() + (k + 4) * D.U * size)
    if out.dtype == torch.float16:
        limit = limit + 2.0 ** -25
    off = (out.double() - want).abs()
    if out.dtype == torch.float16:  # beyond the largest fp16 value and half a step, infinity is the rounded value
        over = want.abs() + limit >= 65520
        assert (out[over].isinf() | (off[over] <= limit[over])).all()
        off, limit = off[~over], limit[~over]
    assert (off <= limit).all(), f"{int((off > limit).sum())} outside, worst {float((off / limit).max())}"


MNK = [(1, 1, 1), (1, 128, 128), (2, 16, 64), (7, 130, 129), (16, 256, 1024), (17, 100, 300), (64, 512, 512),
       (128, 128, 128), (129, 257, 384), (200, 1000, 1000), (300, 64, 2050), (513, 384, 640), (1000, 130, 16)]


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("out", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("m,n,k", MNK)
def test_product(m, n, k, out, layout, aligned):
    a, sa, b, sb, want, size = product_case(m, n, k, layout=layout, aligned=aligned, seed=m + n)
    y = torch.full((m, n), float("nan"), device="cuda", dtype=D.TYPES[out])
    bias = torch.randn(n, generator=torch.Generator().manual_seed(k)).cuda() if (m + n) % 2 else None
    T.matmul_fp8_blocks(a, sa, b, sb, y, bias=bias, b_layout=layout)
    check_product(y, want, size, k, bias)
    assert T.device_status() == 0


@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("m,n,k", [(2500, 2100, 200), (2500, 1000, 300), (1000, 1217, 640), (9000, 128, 1152), (40000, 260, 128),
                                   (20, 9000, 136), (700, 4000, 1030), (2500, 2100, 2200), (2500, 1000, 2500), (1000, 1217, 4200)])
def test_product_many_tiles(m, n, k, layout):
    """More output tiles than SMs, so that a CTA computes several in turn, at every width of tile; several times,
    and with every width of output (a CTA reuses its output buffers while copies read them)."""
    a, sa, b, sb, want, size = product_case(m, n, k, layout=layout, seed=m)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for _ in range(4):
            y = torch.full((m, n), float("nan"), device="cuda", dtype=dtype)
            T.matmul_fp8_blocks(a, sa, b, sb, y, b_layout=layout)
            check_product(y, want, size, k)
    assert T.device_status() == 0


@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("n", [5, 21, 32, 33, 64, 100, 128, 129, 256])
@pytest.mark.parametrize("k", [1, 65, 128, 256, 300, 500, 640, 700])
def test_product_tall(n, k, layout):
    """Few columns and so many rows that a CTA's stages come round several times, with one to six blocks of k; the
    output's rows end on 16, 4 and 2 bytes."""
    m = 150001 if n <= 128 else 400001
    a, sa, b, sb, want, size = product_case(m, n, k, layout=layout, seed=n)
    for dtype in (torch.float32, torch.bfloat16):
        y = torch.full((m, n), float("nan"), device="cuda", dtype=dtype)
        T.matmul_fp8_blocks(a, sa, b, sb, y, b_layout=layout)
        check_product(y, want, size, k)
    assert T.device_status() == 0


@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("m,n,k", [(20, 130, 1024), (100, 500, 2100), (40, 64, 4300), (130, 1000, 8192), (600, 900, 1500),
                                   (17, 2000, 3333), (256, 4096, 1152)])
def test_product_split(m, n, k, layout):
    """Few output tiles and a long k, which several CTAs share."""
    a, sa, b, sb, want, size = product_case(m, n, k, layout=layout, seed=m)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(k)).cuda()
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for stride in (n, D.up16(n) + 16):
            y = torch.full((m, stride), float("nan"), device="cuda", dtype=dtype)
            T.matmul_fp8_blocks(a, sa, b, sb, y[:, :n], bias=bias, b_layout=layout)
            check_product(y[:, :n], want, size, k, bias)
            assert y[:, n:].isnan().all()
            again = torch.empty(m, n, device="cuda", dtype=dtype)
            T.matmul_fp8_blocks(a, sa, b, sb, again, bias=bias, b_layout=layout)
            assert torch.equal(again, y[:, :n])
    assert T.device_status() == 0


@pytest.mark.parametrize("a_rows,b_rows", [(1, 1), (128, 1), (128, 128)])
@pytest.mark.parametrize("a_kind,b_kind", [("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("m", [5, 40, 300])
def test_product_blocks_and_types(m, a_kind, b_kind, a_rows, b_rows):
    a, sa, b, sb, want, size = product_case(m, 300, 520, a_kind, b_kind, "nk", a_rows, b_rows, seed=3)
    y = torch.full((m, 300), float("nan"), device="cuda")
    T.matmul_fp8_blocks(a, sa, b, sb, y)
    check_product(y, want, size, 520)


@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("n", [200, 201, 203, 1])
@pytest.mark.parametrize("m", [1, 3, 30, 260])
def test_product_writes_its_rows_only(m, n, layout):
    k = 256
    a, sa, b, sb, want, size = product_case(m, n, k, seed=9, layout=layout)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for stride, offset in (((n + 15) // 8 * 8, 8), (n + 1, 3)):
            whole = torch.full((m + 3, stride), 7.0, device="cuda", dtype=dtype)
            y = whole.view(-1)[offset + stride:offset + stride + m * stride].view(m, stride)[:, :n]
            T.matmul_fp8_blocks(a, sa, b, sb, y, b_layout=layout)
            check_product(y, want, size, k)
            left = whole.clone().view(-1)
            left[offset + stride:offset + stride + m * stride].view(m, stride)[:, :n] = 7.0
            assert (left == 7.0).all()


@pytest.mark.parametrize("m", [2, 40, 200])
def test_product_nan_blocks(m):
    """A NaN scale or element makes the rows (columns) that read it NaN, and no others."""
    a, sa, b, sb, want, size = product_case(m, 256, 384, seed=5)
    sa[1, 1] = 255
    sb[1, 2] = 255
    y = torch.empty(m, 256, device="cuda")
    T.matmul_fp8_blocks(a, sa, b, sb, y)
    bad = torch.zeros(m, 256, dtype=torch.bool, device="cuda")
    bad[1] = True
    bad[:, 128:] = True
    assert y[bad].isnan().all()
    assert not y[~bad].isnan().any()


def test_product_large_and_small_scales():
    """Scales at the ends of their range meet, where their product is still a float."""
    m, n, k = 130, 140, 256
    a, sa, b, sb, _, _ = product_case(m, n, k, seed=11)
    sa[:, 0], sb[:, 0] = 1, 240
    sa[:, 1], sb[:, 1] = 235, 12
    want = D.values(a, sa) @ D.values(b, sb, 128).t()
    size = D.values(a, sa).abs() @ D.values(b, sb, 128).abs().t()
    y = torch.empty(m, n, device="cuda")
    T.matmul_fp8_blocks(a, sa, b, sb, y)
    check_product(y, want, size, k)


# ---- checkpoint and backward ----------------------------------------------------------------------
def slope(x, kind):
    x = x.clone().requires_grad_(True)
    D.activation(x, kind).sum().backward()
    g = x.grad
    return torch.where(x > 0, 1.0, 0.0).double() if kind == "relu" else g


def function_bound(x, kind):
    """Relative error of an activation or of a slope's terms in fp32: a few roundings, and the rounding of the
    exponential's argument u, which counts |u| times (u = x^2 / 2 for the normal distribution's tail)."""
    u = {"relu": 0 * x, "silu": x.abs(), "gelu": x * x, "gelu_tanh": 1.6 * (x.abs() + 0.05 * x.abs() ** 3)}[kind]
    return (16 + 4 * u) * D.U


@pytest.mark.parametrize("kind", ["relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 129), (33, 128), (130, 257), (50, 1001)])
def test_checkpoint_and_backward(rows, cols, dtype, kind):
    dt = D.TYPES[dtype]
    for stride, offset in ((D.up16(cols), 0), (cols + 1, 1), (D.up16(cols) + 4, 4), (D.up16(cols) + 2, 2)):
        def held(t):
            return D.strided(rows, cols, t, stride, offset)

        x, y, q, dy, dx = held(dt), held(dt), held(torch.int8), held(dt), held(dt)
        x.copy_(D.make(rows, cols, dt, rows * cols))
        dy.copy_(D.make(rows, cols, dt, 7, scale=0.01))
        scales = torch.zeros(rows, -(-cols // 128), dtype=torch.uint8, device="cuda")
        T.activation_checkpoint_int8(x, y, q, scales, activation=kind)
        want_q, want_scales = D.quantize(x, "int8")
        assert torch.equal(scales, want_scales) and same(q, want_q)
        want = D.activation(x.double(), kind)
        off = (y.double() - want).abs()
        # an exponential below 2^-126 counts as zero: less than |x| 2^-126 of y; and the type's own smallest step
        least = x.double().abs() * 2.0 ** -126 + (2.0 ** -24 if dt == torch.float16 else 2.0 ** -120)
        assert (off <= (function_bound(x.double(), kind) + D.half_step(dt)) * want.abs() + least).all()

        T.activation_backward_int8(dy, q, scales, dx, activation=kind)
        xh = D.values(q, scales)
        want = dy.double() * slope(xh, kind)
        # the slope's two terms, each at most 1 + |x| times the falling factor; their sum may cancel
        terms = torch.special.expit(-xh.abs()) * xh.abs() * (2 if kind != "gelu_tanh" else 2 + 0.5 * xh * xh) + \
            slope(xh, kind).abs() if kind != "relu" else slope(xh, kind)
        limit = dy.double().abs() * function_bound(xh, kind) * terms + D.half_step(dt) * want.abs() + \
            (2.0 ** -24 if dt == torch.float16 else 2.0 ** -120)
        assert ((dx.double() - want).abs() <= limit).all()


def test_checkpoint_identity_in_place_and_not_finite():
    x = D.make(40, 300, torch.float32, 3)
    q = torch.zeros(40, 300, dtype=torch.int8, device="cuda")
    scales = torch.zeros(40, 3, dtype=torch.uint8, device="cuda")
    T.activation_checkpoint_int8(x, None, q, scales, activation="identity")
    want_q, want_scales = D.quantize(x, "int8")
    assert torch.equal(scales, want_scales) and same(q, want_q)
    y = torch.empty_like(x)
    T.activation_checkpoint_int8(x, y, q, scales, activation="gelu")
    z = x.clone()
    T.activation_checkpoint_int8(z, z, q, scales, activation="gelu")
    assert torch.equal(y, z) and torch.equal(scales, want_scales)
    g = D.make(40, 300, torch.float32, 4)
    dx = torch.empty_like(g)
    T.activation_backward_int8(g, q, scales, dx, activation="gelu")
    T.activation_backward_int8(g, q, scales, g, activation="gelu")
    assert torch.equal(dx, g)
    x[3, 5], x[7, 290] = float("inf"), float("nan")
    T.activation_checkpoint_int8(x, y, q, scales, activation="silu")
    assert (scales == 255).nonzero().tolist() == [[3, 0], [7, 2]]
    assert (q[3, :128] == 0).all() and (q[7, 256:] == 0).all()
    T.activation_backward_int8(torch.ones_like(x), q, scales, dx, activation="silu")
    assert dx[3, :128].isnan().all() and dx[7, 256:].isnan().all() and int(dx.isnan().sum()) == 128 + 44


@pytest.mark.parametrize("kind", ["gelu", "gelu_tanh", "silu"])
def test_backward_against_differences(kind):
    """The slope is the function's: central differences of the definition, h = 2^-10 (third derivatives below 4)."""
    x = torch.arange(-127, 128, device="cuda", dtype=torch.float32).repeat(1, 1) * 2.0 ** -4
    q = torch.arange(-127, 128, device="cuda").to(torch.int8)[None].contiguous()
    scales = torch.full((1, 2), 127 - 4, dtype=torch.uint8, device="cuda")
    dx = torch.empty_like(x)
    T.activation_backward_int8(torch.ones_like(x), q, scales, dx, activation=kind)
    h = 2.0 ** -10
    want = (D.activation(x.double() + h, kind) - D.activation(x.double() - h, kind)) / (2 * h)
    assert (dx.double() - want).abs().max() <= 4 * h * h / 6 + 1e-5


# ---- weight gradient --------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 128, 128), (31, 16, 64), (64, 128, 256), (65, 130, 129), (200, 100, 1000),
                                      (1000, 256, 384), (5000, 48, 130), (333, 520, 264)])
@pytest.mark.parametrize("pad", [0, 1, 2, 4, 8])  # elements that rows lie off a multiple of 16
def test_weight_grad(rows, n, k, dtype, pad):
    dt = D.TYPES[dtype]
    q64, scales = D.quantize(D.make(rows, k, torch.float32, rows + k), "int8")
    q = D.strided(rows, k, torch.int8, D.up16(k) + pad, pad)
    q.copy_(q64.to(torch.int8))
    dy = D.strided(rows, n, dt, D.up16(n) + pad, pad)
    dy.copy_(D.make(rows, n, dt, 5, scale=0.01))
    xv = D.values(q, scales)
    want, size = dy.double().t() @ xv, dy.double().abs().t() @ xv.abs()
    for accumulate in (False, True):
        width = (k + 3) // 4 * 4 + (0 if pad in (0, 2) else 1)  # rows of dw on 16 bytes, or not
        start = torch.randn(n, width, generator=torch.Generator().manual_seed(rows))[:, :k].cuda()
        dw = torch.full((n, width), 7.0, device="cuda")[:, :k].copy_(start)
        T.weight_grad_int8(dy, q, scales, dw, accumulate=accumulate)
        target = want + (start.double() if accumulate else 0)
        limit = (rows + 8) * D.U * (size + (start.double().abs() if accumulate else 0)) + 2.0 ** -140
        off = (dw.double() - target).abs()
        assert (off <= limit).all(), f"{int((off > limit).sum())} outside, worst {float((off / limit).max())}"
        assert (dw.as_strided((n, width - k), (width, 1), k) == 7.0).all()  # between the rows
    assert T.device_status() == 0


def test_weight_grad_same_bits_and_workspace():
    rows, n, k = 20000, 130, 200
    q64, scales = D.quantize(D.make(rows, k, torch.float32, 1), "int8")
    q = q64.to(torch.int8)
    dy = D.make(rows, n, torch.float32, 2)
    size = T.weight_grad_int8_workspace_size(rows, n, k)
    assert size > 0
    dw = [torch.empty(n, k, device="cuda") for _ in range(3)]
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    for out, w in zip(dw, (None, ws, ws)):
        T.weight_grad_int8(dy, q, scales, out, workspace=w)
    assert torch.equal(dw[0], dw[1]) and torch.equal(dw[0], dw[2])
    with pytest.raises(T.InvalidArgument, match="workspace"):
        T.weight_grad_int8(dy, q, scales, dw[0], workspace=ws[:size - 16])


def test_weight_grad_nan_block():
    """A checkpoint block that is not finite makes the 128 columns that read it NaN."""
    q = torch.ones(300, 256, dtype=torch.int8, device="cuda")
    scales = torch.full((300, 2), 127, dtype=torch.uint8, device="cuda")
    scales[77, 1] = 255
    dw = torch.empty(20, 256, device="cuda")
    T.weight_grad_int8(torch.ones(300, 20, device="cuda"), q, scales, dw)
    assert (dw[:, :128] == 300).all() and dw[:, 128:].isnan().all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_weight_grad_not_finite_gradient(dtype):
    """Infinities and NaN of dy arrive as such: inf times a positive element is inf, times zero NaN. So does the
    largest finite value."""
    rows, n, k = 300, 40, 130
    dt = D.TYPES[dtype]
    q = torch.ones(rows, k, dtype=torch.int8, device="cuda")
    q[:, 1] = -3
    q[:, 2] = 0
    scales = torch.full((rows, 2), 127, dtype=torch.uint8, device="cuda")
    dy = torch.zeros(rows, n, device="cuda", dtype=dt)
    dy[5, 0], dy[6, 1], dy[7, 2], dy[200, 3] = float("inf"), -float("inf"), float("nan"), torch.finfo(dt).max
    dy[8, 4] = 1.0
    dw = torch.empty(n, k, device="cuda")
    T.weight_grad_int8(dy, q, scales, dw)
    want = dy.float().t() @ q.float()
    want[3] = torch.finfo(dt).max * q[0].float()
    assert torch.equal(torch.nan_to_num(dw, nan=1.5), torch.nan_to_num(want, nan=1.5))
    if dtype == "fp32":  # a NaN whose upper half alone would be an infinity
        dy[7, 2] = torch.tensor([0x7F800001], dtype=torch.int32, device="cuda").view(torch.float32)[0]
        T.weight_grad_int8(dy, q, scales, dw)
        assert dw[2].isnan().all()


# ---- alignments -----------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("cols", [1, 3, 50, 64, 127, 130, 255, 300])
def test_rows_of_any_alignment(kind, cols):
    """Every pair of alignments of a float matrix and an 8-bit one: the bytes are those of packed copies, nothing
    beyond a row is written."""
    rows, dtype = 131, D.TYPES[kind]
    x = D.make(rows, cols, dtype, cols)

    def place(dtype, stride, offset):
        whole = torch.full((rows * stride + offset + 16,), 5.0, device="cuda").to(dtype)
        return whole, whole[offset:offset + rows * stride].view(rows, stride)[:, :cols]

    q0 = torch.empty(rows, D.up16(cols), dtype=torch.int8, device="cuda")[:, :cols]
    s0 = torch.empty(rows, -(-cols // 128), dtype=torch.uint8, device="cuda")
    y0, g0 = torch.empty_like(x), torch.empty_like(x)
    T.activation_checkpoint_int8(x, y0, q0, s0, activation="silu")
    T.activation_backward_int8(x, q0, s0, g0, activation="silu")
    want_rows = D.quantize(x, "e4m3", 1)
    want_squares = D.quantize(x, "e4m3", 128)
    wide = (cols + 31) // 16 * 16
    for x_stride, x_offset in ((wide, 0), (wide + 4, 4), (wide + 2, 2), (wide + 1, 1)):
        xs = place(dtype, x_stride, x_offset)[1]
        xs.copy_(x)
        for q_stride, q_offset in ((wide, 0), (wide + 8, 8), (wide + 4, 4), (wide + 2, 2), (wide + 1, 1)):
            whole_q, q = place(torch.int8, q_stride, q_offset)
            whole_y, y = place(dtype, x_stride, x_offset)
            whole_g, g = place(dtype, x_stride, x_offset)
            s = torch.empty_like(s0)
            T.activation_checkpoint_int8(xs, y, q, s, activation="silu")
            assert torch.equal(s, s0) and torch.equal(q, q0) and torch.equal(y, y0)
            T.activation_backward_int8(xs, q, s, g, activation="silu")
            assert torch.equal(g, g0)
            for whole, part in ((whole_q, q), (whole_y, y), (whole_g, g)):
                part.fill_(5)
                assert (whole == 5).all()
            f = q.view(torch.float8_e4m3fn)
            for block_rows, (want, scales) in ((1, want_rows), (128, want_squares)):
                got = torch.empty_like(scales)
                whole_q.fill_(5)
                T.quantize_blocks_fp8(xs, f, got, block_rows=block_rows)
                assert torch.equal(got, scales) and torch.equal(f.double(), want)
                q.fill_(5)
                assert (whole_q == 5).all()


# ---- sizes of zero, refusals ------------------------------------------------------------------------
def test_empty():
    e4 = torch.float8_e4m3fn

    def z(r, c, t):
        return torch.empty(r, c, dtype=torch.uint8 if t == e4 else t, device="cuda").view(t)

    for r, c in ((0, 128), (4, 0), (0, 0)):
        s = torch.empty(r, -(-c // 128), dtype=torch.uint8, device="cuda")
        T.quantize_blocks_fp8(z(r, c, torch.float32), z(r, c, e4), s)
        T.activation_checkpoint_int8(z(r, c, torch.float32), z(r, c, torch.float32), z(r, c, torch.int8), s)
        T.activation_backward_int8(z(r, c, torch.float32), z(r, c, torch.int8), s, z(r, c, torch.float32))
    for m, n, k in ((0, 128, 128), (5, 0, 128), (5, 130, 0), (300, 130, 0)):
        y = torch.full((m, n), 3.0, device="cuda")
        bias = torch.arange(n, device="cuda", dtype=torch.float32)
        sa = torch.empty(m, -(-k // 128), dtype=torch.uint8, device="cuda").fill_(127)
        sb = torch.empty(-(-n // 128), -(-k // 128), dtype=torch.uint8, device="cuda").fill_(127)
        T.matmul_fp8_blocks(z(m, k, e4), sa, z(n, k, e4), sb, y, bias=bias)
        if k == 0:
            assert torch.equal(y, bias.expand(m, n))
    for accumulate in (False, True):
        dw = torch.full((20, 30), 3.0, device="cuda")
        T.weight_grad_int8(z(0, 20, torch.float32), z(0, 30, torch.int8), z(0, 1, torch.uint8), dw, accumulate=accumulate)
        assert (dw == (3.0 if accumulate else 0.0)).all()


def test_refusals():
    e4 = torch.float8_e4m3fn
    x = torch.zeros(8, 256, device="cuda")
    q = torch.zeros(8, 256, dtype=torch.uint8, device="cuda").view(e4)
    s = torch.full((8, 2), 127, dtype=torch.uint8, device="cuda")
    w = torch.zeros(128, 256, dtype=torch.uint8, device="cuda").view(e4)
    ws = torch.full((1, 2), 127, dtype=torch.uint8, device="cuda")
    y = torch.zeros(8, 128, device="cuda")
    i8 = torch.zeros(8, 256, dtype=torch.int8, device="cuda")
    bad = [
        lambda: T.quantize_blocks_fp8(x.double(), q, s),
        lambda: T.quantize_blocks_fp8(x, i8, s),
        lambda: T.quantize_blocks_fp8(x, q, s, block_rows=64),
        lambda: T.quantize_blocks_fp8(x, q, s, block_rows=128),
        lambda: T.quantize_blocks_fp8(x, q[:, :128], s),
        lambda: T.quantize_blocks_fp8(x.cpu(), q, s),
        lambda: T.quantize_blocks_fp8(x, q, s.cpu()),
        lambda: T.quantize_blocks_fp8(x, q, s.float()),
        lambda: T.quantize_blocks_fp8(x.t(), q.t(), s),
        lambda: T.quantize_blocks_fp8(x[0], q[0], s),
        lambda: T.quantize_blocks_fp8(x[:1].expand(8, 256), q, s),
        lambda: T.matmul_fp8_blocks(q, s, w, ws, y, b_layout="tn"),
        lambda: T.matmul_fp8_blocks(q, s, w, ws, y.double()),
        lambda: T.matmul_fp8_blocks(q, s, w, ws, y[:, :100]),
        lambda: T.matmul_fp8_blocks(q, s, w, ws, y, bias=torch.zeros(127, device="cuda")),
        lambda: T.matmul_fp8_blocks(q, s, w, ws, y, bias=torch.zeros(128, device="cuda").bfloat16()),
        lambda: T.matmul_fp8_blocks(q, s[:, :1], w, ws, y),
        lambda: T.matmul_fp8_blocks(q, s, w, ws, y, b_layout="kn"),
        lambda: T.matmul_fp8_blocks(x, s, w, ws, y),
        lambda: T.activation_checkpoint_int8(x, x.clone(), i8, s, activation="tanh"),
        lambda: T.activation_checkpoint_int8(x, x.clone(), i8, s, activation="identity"),
        lambda: T.activation_checkpoint_int8(x, x.bfloat16(), i8, s),
        lambda: T.activation_checkpoint_int8(x, x.clone(), q, s),
        lambda: T.activation_backward_int8(x, i8, s, x.clone(), activation="identity"),
        lambda: T.activation_backward_int8(x, i8, s, x.half()),
        lambda: T.weight_grad_int8(x, i8[:7], s, torch.zeros(256, 256, device="cuda")),
        lambda: T.weight_grad_int8(x, i8, s, torch.zeros(256, 255, device="cuda")),
        lambda: T.weight_grad_int8(x, i8, s, torch.zeros(256, 256, device="cuda").half()),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(T.InvalidArgument):
            call()
            pytest.fail(f"call {i} was not refused")


def test_refuses_what_is_no_tensor():
    x = torch.zeros(8, 256, device="cuda")
    q = torch.zeros(8, 256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.full((8, 2), 127, dtype=torch.uint8, device="cuda")
    i8 = torch.zeros(8, 256, dtype=torch.int8, device="cuda")
    dw = torch.zeros(256, 256, device="cuda")
    bad = [
        lambda: T.quantize_blocks_fp8(x, q, None),
        lambda: T.quantize_blocks_fp8([[1.0]], q, s),
        lambda: T.quantize_blocks_fp8(x, None, s),
        lambda: T.matmul_fp8_blocks(q, None, q, s, x[:, :8]),
        lambda: T.matmul_fp8_blocks(q, s, q, s, x[:, :8], bias=[0.0] * 8),
        lambda: T.activation_checkpoint_int8(x, None, i8, s),
        lambda: T.activation_checkpoint_int8(x, x.clone(), i8, 127),
        lambda: T.activation_backward_int8(x, i8, s, None),
        lambda: T.weight_grad_int8(x, i8, None, dw),
        lambda: T.weight_grad_int8(x, i8, s, dw, workspace=1 << 20),
    ]
    for call in bad:
        with pytest.raises(T.InvalidArgument):
            call()


# ---- streams and graphs -------------------------------------------------------------------------------
def layer(x, w, ws, grad, bias, stages=False):
    """One layer forward and backward, as a training step runs it: quantize, product, activation with its input
    kept, the input kept for the weight gradient, and the gradients."""
    m, k = x.shape
    n = w.shape[0]
    dev = x.device
    xq = torch.empty(m, k, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    xs = torch.empty(m, -(-k // 128), dtype=torch.uint8, device=dev)
    T.quantize_blocks_fp8(x, xq, xs)
    z = torch.empty(m, n, device=dev, dtype=torch.bfloat16)
    T.matmul_fp8_blocks(xq, xs, w, ws, z, bias=bias)
    kept = torch.empty(m, k, dtype=torch.int8, device=dev)
    kept_s = torch.empty_like(xs)
    T.activation_checkpoint_int8(x, None, kept, kept_s, activation="identity")
    y, zq = torch.empty_like(z), torch.empty(m, n, dtype=torch.int8, device=dev)
    zs = torch.empty(m, -(-n // 128), dtype=torch.uint8, device=dev)
    T.activation_checkpoint_int8(z, y, zq, zs, activation="gelu")
    dz = torch.empty_like(y)
    T.activation_backward_int8(grad, zq, zs, dz, activation="gelu")
    dzq = torch.empty(m, n, dtype=torch.uint8, device=dev).view(torch.float8_e5m2)
    dzs = torch.empty_like(zs)
    T.quantize_blocks_fp8(dz, dzq, dzs)
    dx = torch.empty(m, k, device=dev, dtype=torch.bfloat16)
    T.matmul_fp8_blocks(dzq, dzs, w, ws, dx, b_layout="kn")
    dw = torch.empty(n, k, device=dev)
    T.weight_grad_int8(dz, kept, kept_s, dw)
    if stages:
        return dict(xq=xq, xs=xs, z=z, kept=kept, kept_s=kept_s, y=y, zq=zq, zs=zs, dz=dz, dzq=dzq, dzs=dzs, dx=dx, dw=dw)
    return y, dx, dw


def layer_inputs(seed=0, m=700, n=256, k=384):
    x = D.make(m, k, torch.bfloat16, seed)
    w64, ws = D.quantize(D.make(n, k, torch.float32, seed + 1, scale=0.05), "e4m3", 128)
    w = w64.float().to(torch.float8_e4m3fn)
    return x, w, ws, D.make(m, n, torch.bfloat16, seed + 2, scale=0.01), torch.randn(n, device="cuda")


def test_layer_against_64_bits():
    """A run of all operators, each stage against the 64-bit definition of what it was given: the elements and scales
    equal, the sums and functions within their rounding bounds. (The distance of the whole step from an unquantized
    one has no useful bound here: e5m2 moves a gradient by up to 2^-3 of itself, and where a block holds an outlier
    its INT8 step is as large as its other values.)"""
    x, w, ws, g, bias = layer_inputs()
    s = layer(x, w, ws, g, bias, stages=True)
    (n, k), m = w.shape, x.shape[0]
    wv = D.values(w, ws, 128)
    for got, scales, source, kind in ((s["xq"], s["xs"], x, "e4m3"), (s["kept"], s["kept_s"], x, "int8"),
                                      (s["zq"], s["zs"], s["z"], "int8"), (s["dzq"], s["dzs"], s["dz"], "e5m2")):
        q, bytes_ = D.quantize(source, kind)
        assert torch.equal(scales, bytes_) and same(got, q)
    xv, dzv = D.values(s["xq"], s["xs"]), D.values(s["dzq"], s["dzs"])
    check_product(s["z"], xv @ wv.t(), xv.abs() @ wv.abs().t(), k, bias)
    check_product(s["dx"], dzv @ wv, dzv.abs() @ wv.abs(), n)
    want = D.activation(s["z"].double(), "gelu")
    assert ((s["y"].double() - want).abs() <= (function_bound(s["z"].double(), "gelu") + 2.0 ** -8) * want.abs() +
            2.0 ** -120).all()  # below 2^-126 a float has fewer bits: |x| 2^-126 and less is lost there
    zh = D.values(s["zq"], s["zs"])
    want = g.double() * slope(zh, "gelu")
    terms = slope(zh, "gelu").abs() + 2 * zh.abs() * torch.special.expit(-zh.abs())
    assert ((s["dz"].double() - want).abs() <=
            g.double().abs() * function_bound(zh, "gelu") * terms + 2.0 ** -8 * want.abs() + 2.0 ** -120).all()
    kept = D.values(s["kept"], s["kept_s"])
    size = s["dz"].double().abs().t() @ kept.abs()
    assert ((s["dw"].double() - s["dz"].double().t() @ kept).abs() <= (m + 8) * D.U * size).all()


@pytest.mark.parametrize("features", [128, 256])
def test_graph_layer(features):
    """A graph layer and its weight gradient: the aggregated features (the SpMM's fp32 output) quantized and
    multiplied by the layer's weights, kept for the backward pass as well."""
    from tests.cases import EDGE_CASES
    from tests.gpu_util import build_case, run_spmm

    y = run_spmm(build_case(EDGE_CASES["random_local"](), features, seed=3))
    rows, n = y.shape[0], 96
    q = torch.empty(rows, features, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.empty(rows, features // 128, dtype=torch.uint8, device="cuda")
    T.quantize_blocks_fp8(y, q, scales)
    kept, kept_s = torch.empty(rows, features, dtype=torch.int8, device="cuda"), torch.empty_like(scales)
    T.activation_checkpoint_int8(y, None, kept, kept_s, activation="identity")
    w64, ws = D.quantize(D.make(n, features, torch.float32, 8, scale=0.1), "e4m3", 128)
    w = w64.float().to(torch.float8_e4m3fn)
    z = torch.empty(rows, n, device="cuda")
    T.matmul_fp8_blocks(q, scales, w, ws, z)
    for got, got_s, kind in ((q, scales, "e4m3"), (kept, kept_s, "int8")):
        want, bytes_ = D.quantize(y, kind)
        assert torch.equal(got_s, bytes_) and same(got, want)
    yv, wv = D.values(q, scales), D.values(w, ws, 128)
    check_product(z, yv @ wv.t(), yv.abs() @ wv.abs().t(), features)
    grad = D.make(rows, n, torch.float32, 9, scale=0.01)
    dw = torch.empty(n, features, device="cuda")
    T.weight_grad_int8(grad, kept, kept_s, dw)
    kv = D.values(kept, kept_s)
    limit = (rows + 8) * D.U * (grad.double().abs().t() @ kv.abs())
    assert ((dw.double() - grad.double().t() @ kv).abs() <= limit).all()


def test_streams_and_graph():
    args = layer_inputs(3)
    want = layer(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(*args)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    static = [a.clone() for a in args]
    with torch.cuda.graph(graph):
        out = layer(*static)
    for seed in (3, 9):
        fresh = layer_inputs(seed)
        for s, f in zip(static, fresh):
            s.view(torch.uint8).copy_(f.view(torch.uint8)) if s.element_size() == 1 else s.copy_(f)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, layer(*fresh)))


def test_explicit_stream_argument():
    rows, n, k = 20000, 64, 128
    q64, scales = D.quantize(D.make(rows, k, torch.float32, 1), "int8")
    q, dy = q64.to(torch.int8), D.make(rows, n, torch.bfloat16, 2)
    want = torch.empty(n, k, device="cuda")
    T.weight_grad_int8(dy, q, scales, want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        dw = torch.empty(n, k, device="cuda")
        torch.cuda.synchronize()
        T.weight_grad_int8(dy, q, scales, dw, stream=stream)
        side.synchronize()
        assert torch.equal(dw, want)
