"""Long sums of the dense operators on 8-bit blocks. All terms are positive, so that what an accumulator cuts off
adds up and shows as a bias.

The tensor core cuts off at most about a last bit of the accumulator (2^-23 of it) for every MMA of 32 of k, and the
accumulator is half of the sum on average; N MMAs lose at most N 2^-23 / 2 of the sum, twice that is allowed. An
accumulator is emptied after 64 MMAs (fp32 outputs, and long sums of any type), into registers that round each of P
sums to nearest (2^-24 of the sum at most). 16-bit outputs keep one accumulator for up to 512 (fp16) or 4096 (bf16)
MMAs. Without that, 32768 MMAs lose 2.4e-3."""
from __future__ import annotations

import pytest
import torch

import tcc_spmm_b200 as T
from tests import dense8_util as D

pytestmark = pytest.mark.gpu


def positive(rows, cols, low, high, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.rand(rows, cols, device="cuda", generator=gen) * (high - low) + low
    q = x.to(torch.float8_e4m3fn)
    held = D.strided(rows, cols, q.dtype, D.up16(cols))
    held.view(torch.uint8).copy_(q.view(torch.uint8))
    return held


# few rows, narrow and wide tiles, tiles that share k, pairs of CTAs, [k, n] weights
@pytest.mark.parametrize("m,n,k,layout", [(5, 40, 65536, "nk"), (20, 30, 1 << 20, "nk"), (20, 130, 1 << 20, "kn"), (300, 64, 150000, "nk"),
                                          (20, 30, 16384, "nk"), (20, 30, 131072, "nk"), (150, 200, 40000, "nk"),
                                          (2500, 2100, 20000, "nk"), (2500, 2100, 20000, "kn"), (130, 18900, 17000, "nk"),
                                          (20, 140, 131073, "kn"), (20, 30, 16385, "nk")])
def test_product_long_sums(m, n, k, layout):
    a = positive(m, k, 0.5, 2.0, 1)
    b = positive(n, k, 0.01, 0.12, 2) if layout == "nk" else positive(k, n, 0.01, 0.12, 2)
    sa = torch.full((m, -(-k // 128)), 127, dtype=torch.uint8, device="cuda")
    sb = torch.full((-(-b.shape[0] // 128), -(-b.shape[1] // 128)), 127 - (k.bit_length() - 13), dtype=torch.uint8, device="cuda")
    wide = b.double() if layout == "kn" else b.double().t()
    want = a.double() @ wide * 2.0 ** -(k.bit_length() - 13)
    assert want.max() < 30000 and want.min() > 100
    passes = -(-k // 2048)
    for dtype, kept in ((torch.float32, 64), (torch.bfloat16, 4096), (torch.float16, 512)):
        y = torch.full((m, n), float("nan"), device="cuda", dtype=dtype)
        T.matmul_fp8_blocks(a, sa, b, sb, y, b_layout=layout)
        limit = D.half_step(dtype) + min(kept, -(-k // 32)) * D.U + passes * 2.0 ** -24
        off = ((y.double() - want).abs() / want).max()
        assert off <= limit, (dtype, float(off), limit)
    assert T.device_status() == 0


def test_product_long_sums_shared_by_ctas():
    """fp32 outputs of few tiles of [n, k] weights: CTAs that share k and empty their accumulators on the way."""
    m, n, k = 600, 900, 8192
    a, b = positive(m, k, 0.5, 2.0, 3), positive(n, k, 0.01, 0.12, 4)
    sa = torch.randint(125, 130, (m, k // 128), generator=torch.Generator().manual_seed(5)).to(torch.uint8).cuda()
    sb = torch.randint(125, 130, (8, k // 128), generator=torch.Generator().manual_seed(6)).to(torch.uint8).cuda()
    want = D.values(a, sa) @ D.values(b, sb, 128).t()
    for dtype, kept in ((torch.float32, 64), (torch.bfloat16, 256), (torch.float16, 256)):
        y = torch.full((m, n), float("nan"), device="cuda", dtype=dtype)
        T.matmul_fp8_blocks(a, sa, b, sb, y)
        # sums of up to four passes, then of up to eight CTAs
        assert ((y.double() - want).abs() <= (D.half_step(dtype) + kept * D.U + 12 * 2.0 ** -24) * want).all(), dtype
    assert T.device_status() == 0


# one CTA a tile of dW and two: so many tiles that each range of rows is all of them; and so few that ranges are many
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,n,k,ranges", [(6000, 100, 148 * 256, 1), (6001, 512, 37 * 256, 1), (1000000, 30, 70, 100)])
def test_weight_grad_long_sums(rows, n, k, ranges, dtype, pad):
    """A range of rows whose accumulator is emptied several times (every 60 MMAs of 16 rows, of which bf16 takes one,
    fp16 two and fp32 three; 56 at least, since stages are whole), the ranges' sums added in eight sums and those in
    order."""
    dt, parts = D.TYPES[dtype], {"bf16": 1, "fp16": 2, "fp32": 3}[dtype]
    gen = torch.Generator(device="cuda").manual_seed(rows)
    q = D.strided(rows, k, torch.int8, D.up16(k) + pad, pad)
    q.copy_(torch.randint(1, 128, (rows, k), device="cuda", generator=gen, dtype=torch.int8))
    scales = torch.full((rows, -(-k // 128)), 127 - 7, dtype=torch.uint8, device="cuda")
    dy = D.strided(rows, n, dt, D.up16(n) + pad, pad)
    dy.copy_(torch.rand(rows, n, device="cuda", generator=gen) * 1.5 + 0.5)
    cg, size = 1 if n <= 128 else 2, T.weight_grad_int8_workspace_size(rows, n, k)
    splits = max(1, size // (-(-n // (128 * cg)) * -(-k // 256) * cg * 128 * 256 * 4))
    assert splits == 1 if ranges == 1 else splits >= ranges
    flushes = -(-(-(-rows // splits) + 64) * parts // (16 * 56))
    assert flushes >= 6 * parts
    dw = torch.full((n, k), float("nan"), device="cuda")
    T.weight_grad_int8(dy, q, scales, dw)
    want = dy.double().t() @ q.double() * 2.0 ** -7
    added = splits if splits <= 8 else -(-splits // 8) + 8
    limit = 60 * D.U + (flushes + added) * 2.0 ** -24
    off = ((dw.double() - want).abs() / want).max()
    assert off <= limit, (float(off), limit)
    assert T.device_status() == 0


@pytest.mark.parametrize("layout", ["nk", "kn"])
@pytest.mark.parametrize("k", [1152, 3200, 4096, 4100, 4224, 8193, 8320])  # 9, 25, 32, 33, 33, 65 and 65 blocks
def test_product_parts_of_any_length(k, layout):
    """CTAs that share k, whose parts are unlike: every block counts once."""
    m, n = 200, 500
    a = positive(m, k, 0.5, 2.0, 1)
    b = positive(n, k, 0.01, 0.12, 2) if layout == "nk" else positive(k, n, 0.01, 0.12, 2)
    sa = torch.randint(125, 130, (m, -(-k // 128)), generator=torch.Generator().manual_seed(5)).to(torch.uint8).cuda()
    sb = torch.randint(125, 130, (-(-b.shape[0] // 128), -(-b.shape[1] // 128)), generator=torch.Generator().manual_seed(6))
    sb = sb.to(torch.uint8).cuda()
    wide = D.values(b, sb, 128)
    want = D.values(a, sa) @ (wide.t() if layout == "nk" else wide)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        y = torch.full((m, n), float("nan"), device="cuda", dtype=dtype)
        T.matmul_fp8_blocks(a, sa, b, sb, y, b_layout=layout)
        # up to 12 blocks in one accumulator, eight sums
        assert ((y.double() - want).abs() <= (D.half_step(dtype) + 48 * D.U + 8 * 2.0 ** -24) * want).all(), dtype
    assert T.device_status() == 0
