"""Plain restatement in 64 bits of the block-scaled cache (pccl_hip_cache_write / _read): every step is exact up to the one
rounding, so results are compared bit for bit."""
import math

import torch

BLOCK = 32
BITS = {"f8e4m3": 8, "f8e5m2": 8, "i8": 8, "f4e2m1": 4}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def values(fmt):
    """The value of every code, NaN and infinities of the 8-bit floats included."""
    if fmt == "i8":
        return [(c - 256 if c > 127 else c) / 64 for c in range(256)]
    exponent_bits, mantissa_bits = {"f8e4m3": (4, 3), "f8e5m2": (5, 2), "f4e2m1": (2, 1)}[fmt]
    bias, found = (1 << (exponent_bits - 1)) - 1, []
    for c in range(1 << (1 + exponent_bits + mantissa_bits)):
        e, m = (c >> mantissa_bits) & ((1 << exponent_bits) - 1), c & ((1 << mantissa_bits) - 1)
        v = math.ldexp(m, 1 - bias - mantissa_bits) if e == 0 else math.ldexp((1 << mantissa_bits) + m, e - bias - mantissa_bits)
        if fmt == "f8e5m2" and e == 31:
            v = math.nan if m else math.inf
        if fmt == "f8e4m3" and e == 15 and m == 7:
            v = math.nan
        found.append(-v if c >> (exponent_bits + mantissa_bits) else v)
    return found


def grid(fmt):
    """Magnitudes from 0 up; the index is the code without its sign."""
    top = {"f8e4m3": 448.0, "f8e5m2": 57344.0, "i8": 127 / 64, "f4e2m1": 6.0}[fmt]
    return sorted({abs(v) for v in values(fmt) if abs(v) <= top})


def encode(fmt, x):
    """x [..., dim], 64 bits -> (codes [..., bytes of a head], scales [..., blocks]) as uint8."""
    dim = x.shape[-1]
    x = torch.cat([x, x.new_zeros(*x.shape[:-1], -dim % BLOCK)], -1).reshape(*x.shape[:-1], -1, BLOCK)
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, 0.0)
    g = torch.tensor(grid(fmt), dtype=torch.float64)
    most = x.abs().amax(-1)
    s = torch.full(most.shape, 254, dtype=torch.long)
    for k in range(253, -1, -1):  # the smallest power of two with which nothing passes the format's largest value
        s[most <= g[-1] * math.ldexp(1.0, k - 127)] = k
    scale = torch.tensor([math.ldexp(1.0, k - 127) for k in range(255)], dtype=torch.float64)[s]
    a = (x.abs() / scale[..., None]).clamp(max=float(g[-1]))
    between = (g[1:] + g[:-1]) / 2
    low, high = torch.searchsorted(between, a.contiguous()), torch.searchsorted(between, a.contiguous(), right=True)
    code = torch.where(low % 2 == 0, low, high)  # they differ at a tie: the even one
    negative = torch.signbit(x)
    if fmt == "i8":
        code = torch.where(negative, (256 - code) % 256, code)
    else:
        code = code + torch.where(negative, 1 << (BITS[fmt] - 1), 0)
    code = torch.where(fine[..., None], code, 0).flatten(-2)[..., :dim]
    if BITS[fmt] == 4:
        code = torch.cat([code, code.new_zeros(*code.shape[:-1], dim % 2)], -1)
        code = code[..., 0::2] + 16 * code[..., 1::2]
    return code.to(torch.uint8), torch.where(fine, s, 255).to(torch.uint8)


def decode(fmt, codes, scales, dim, dtype):
    """codes, scales as encode gives them -> [..., dim] of `dtype`; the product is exact in 32 bits, so there is one rounding."""
    if BITS[fmt] == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :dim]
    v = torch.tensor(values(fmt), dtype=torch.float64)[codes.long()]
    scale = torch.tensor([math.ldexp(1.0, k - 127) for k in range(255)] + [math.nan], dtype=torch.float64)[scales.long()]
    return (v * scale.repeat_interleave(BLOCK, -1)[..., :dim]).float().to(TYPES[dtype])


def same(got, want):
    """Equal bit for bit, any NaN standing for any other."""
    got, want = got.cpu(), want.cpu()
    nan = torch.isnan(want)
    kind = torch.int32 if got.dtype == torch.float32 else torch.int16
    return torch.equal(torch.isnan(got), nan) and torch.equal(got.view(kind)[~nan], want.view(kind)[~nan])
