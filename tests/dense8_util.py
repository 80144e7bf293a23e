"""The 8-bit block operators' definitions in 64 bits, and the rounding bounds their tests use."""
from __future__ import annotations

import math

import torch

LARGEST = {"e4m3": 448.0, "e5m2": 57344.0, "int8": 127.0}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -23  # one addition or product in fp32, rounded either way or cut off


def pow2(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def spread(scales, block_rows, rows, cols):
    """The scale of every element, from the scale bytes."""
    s = torch.where(scales == 255, torch.full_like(scales, float("nan"), dtype=torch.float64),
                    pow2(scales.long() - 127))
    return s.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def values(q, scales, block_rows=1):
    """What 8-bit blocks stand for."""
    return q.double() * spread(scales, block_rows, *q.shape)


def quantize(x, kind, block_rows=1):
    """(elements as doubles, scale bytes): the least power of two that holds the block, then the nearest element."""
    rows, cols = x.shape
    x = x.double()
    rb, cb = -(-rows // block_rows), -(-cols // 128)
    scales = torch.full((rb, cb), 127, dtype=torch.uint8, device=x.device)
    top = torch.nn.functional.pad(x.abs(), (0, cb * 128 - cols, 0, rb * block_rows - rows))
    top = top.reshape(rb, block_rows, cb, 128).amax((1, 3))
    powers = pow2(torch.arange(-126, 128, device=x.device)) * LARGEST[kind]
    e = torch.bucketize(top, powers) + 1
    e = torch.where(top == 0, torch.full_like(e, 127), e)
    scales = torch.where(torch.isfinite(top), e, torch.full_like(e, 255)).to(torch.uint8)
    v = x / spread(scales, block_rows, rows, cols)
    if kind == "int8":
        q = torch.round(v)
    else:
        kept, lowest = (3, -6) if kind == "e4m3" else (2, -14)
        step = pow2((torch.frexp(torch.nan_to_num(v))[1] - 1).clamp(min=lowest) - kept)
        q = torch.round(v / step) * step
    return q, scales


def make(rows, cols, dtype, seed, device="cuda", scale=1.0):
    """Rows of differing sizes, a few large columns, a row of zeros, the last rows zero."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen)) * scale
    x *= torch.where(torch.rand(1, cols, generator=gen) < 0.02, 30.0, 1.0)
    if rows > 3:
        x[2] = 0
    if rows > 40:
        x[-rows // 16:] = 0
    return x.to(dtype).to(device)


def strided(rows, cols, dtype, stride=None, offset=0, device="cuda", fill=0):
    """A [rows, cols] tensor whose rows are `stride` elements apart, `offset` elements into an allocation."""
    stride = stride or cols
    whole = torch.zeros(rows * stride + offset + 64, dtype=torch.uint8, device=device)
    if dtype.itemsize != 1:
        whole = torch.zeros(rows * stride + offset + 64, dtype=dtype, device=device)
        whole.fill_(fill)
        return whole[offset:offset + rows * stride].view(rows, stride)[:, :cols]
    whole.fill_(fill)
    return whole[offset:offset + rows * stride].view(rows, stride)[:, :cols].view(dtype)


def up16(n):
    return -(-n // 16) * 16


def activation(x, kind):
    if kind == "relu":
        return x.clamp(min=0)
    if kind == "silu":
        return x * torch.special.expit(x)
    if kind == "gelu":
        return x * 0.5 * torch.special.erfc(-x * math.sqrt(0.5))  # ndtr's 1 + erf loses the left tail
    return x * torch.special.expit(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2
