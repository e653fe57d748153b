"""64-bit reference of microscaled rows: quantization, storage and products (torch float64, test infrastructure).

Exponents come from math on exact doubles, codes from comparing with the middles between the format's values, so neither
shares a step with the kernels' conversions."""
from __future__ import annotations

import math

import torch

from . import product_oracle as orx

BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E4M3 = tuple(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
             for e in range(16) for m in range(8) if (e, m) != (15, 7))
VALUES = {"e2m1": E2M1, "e4m3": E4M3}


def exponent(amax: float, fmt: str) -> int:
    """The smallest X >= -127 with amax 2^-X below the middle between the format's largest value and what would follow it
    with a longer range; 0 for a block of zeros, 128 for one that is not finite."""
    if not math.isfinite(amax):
        return 128
    if amax == 0:
        return 0
    v = VALUES[fmt]
    past = v[-1] + (v[-1] - v[-2]) / 2
    x = math.frexp(amax / past)[1]                      # 2^(x - 1) <= amax / past < 2^x
    return max(x, -127)


def quantize(x: torch.Tensor, fmt: str):
    """(codes uint8 [M, K] with the sign in bit 3 or 7, scales uint8 [M, ceil(K / 32)]) of fp32 / bf16 [M, K]."""
    M, K = x.shape
    nb = -(-K // BLOCK)
    v = torch.nn.functional.pad(x.double(), (0, nb * BLOCK - K)).view(M, nb, BLOCK)
    amax = v.abs().amax(2)
    amax = torch.where(torch.isnan(v).any(2), math.nan, amax)
    X = torch.tensor([[exponent(float(a), fmt) for a in row] for row in amax], dtype=torch.float64).view(M, nb)
    bad = X == 128
    s = torch.where(bad[..., None], 0.0, v / torch.exp2(torch.where(bad, 0.0, X))[..., None])
    table = torch.tensor(VALUES[fmt], dtype=torch.float64)
    middle = (table[1:] + table[:-1]) / 2
    mag = s.abs().contiguous()
    code = torch.bucketize(mag, middle, right=True)      # a middle belongs to the code above it
    tie = (code > 0) & (mag == middle[(code - 1).clamp(min=0)]) & (code % 2 == 1)
    code = (code - tie.long()).to(torch.uint8)
    sign = torch.signbit(s) & ~bad[..., None]
    code = code | (sign.to(torch.uint8) << (3 if fmt == "e2m1" else 7))
    return code.view(M, nb * BLOCK)[:, :K], (X + 127).to(torch.uint8)


def store(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    """Codes as the package stores them."""
    if fmt == "e4m3":
        return codes.contiguous().view(torch.float8_e4m3fn)
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def decode(q: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What stored values stand for, float64; NaN where the scale is 255."""
    if q.dtype == torch.uint8:
        table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device=q.device)
        v = torch.stack((table[(q & 15).long()], table[(q >> 4).long()]), -1).flatten(-2)
    else:
        v = q.double()
    power = torch.exp2(scales.double() - 127)
    power = torch.where(scales == 255, math.nan, power).repeat_interleave(BLOCK, -1)[..., :v.shape[-1]]
    return v * power


def random_operand(shape, fmt, gen, low=118, high=128):
    """Stored values of random codes and scales low .. high (bytes): every finite code, both zeros."""
    K = shape[-1]
    if fmt == "e2m1":
        q = torch.randint(0, 256, tuple(shape[:-1]) + (K // 2,), generator=gen, dtype=torch.int16).to(torch.uint8)
    else:
        c = torch.randint(0, 127, tuple(shape), generator=gen, dtype=torch.int16)
        q = (c | torch.randint(0, 2, tuple(shape), generator=gen, dtype=torch.int16) << 7).to(torch.uint8)
        q = q.view(torch.float8_e4m3fn)
    s = torch.randint(low, high + 1, tuple(shape[:-1]) + (-(-K // BLOCK),), generator=gen, dtype=torch.int16)
    return q, s.to(torch.uint8)


def product(a, b, fmt, offs, bias, activation, residual, **options):
    """(z, out, bound) of decoded float64 operands a [M, K], b [G, N, K]; rows of no group NaN. bound: how far the
    kernels' z may be off. e2m1 products are multiples of 1/4 up to 36, which the matrix cores add without loss: what is
    left are fp32 sums of block sums. With e4m3 on one side they drop bits 2^-9 below the largest product of the blocks
    that an instruction adds, for each of them: two or four blocks out of 256 columns, so 2^-6 of the largest product
    there for every 256."""
    M, (G, N, K) = a.shape[0], b.shape

    def tops(t):
        pad = torch.nn.functional.pad(t.abs(), (0, -K % 256))
        return pad.view(t.shape[0], -1, 256).amax(2)

    z = torch.full((M, N), math.nan, dtype=torch.float64, device=a.device)
    size = torch.zeros((M, N), dtype=torch.float64, device=a.device)
    for g, (lo, hi) in enumerate(zip(offs, offs[1:])):
        if hi <= lo:
            continue
        z[lo:hi] = a[lo:hi] @ b[g].t()
        size[lo:hi] = (K / 16 + 4) * 2.0 ** -24 * a[lo:hi].abs() @ b[g].abs().t()
        if fmt == "e4m3":
            size[lo:hi] += 2.0 ** -6 * tops(a[lo:hi]) @ tops(b[g]).t()
        if bias is not None:
            z[lo:hi] += bias[g].double()
            size[lo:hi] += 2.0 ** -23 * (bias[g].double().abs() + z[lo:hi].abs())
    out = orx.act(z, activation, **options)
    return z, out if residual is None else out + residual.double(), size
