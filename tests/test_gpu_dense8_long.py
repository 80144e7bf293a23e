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
