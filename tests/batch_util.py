"""Plain 64-bit forms of the batch operators, on the CPU, and the bounds their
outputs are held to."""
from __future__ import annotations

import math

import torch

from gpu_util import DEV

U8, F64 = torch.uint8, torch.float64
BF16_HALF = 2.0 ** -8   # half a step of bf16, relative to the value


def cu_of(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def normal(shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(torch.bfloat16)


def attend64(q, k, v, scale):
    """q [hq, d], k and v [keys, hkv, d] -> (out [hq, d], sum of |p v| [hq, d]); float64.
    No keys: zeros."""
    hq, hkv = q.shape[0], k.shape[1]
    if not k.shape[0]:
        z = torch.zeros(q.shape, dtype=F64)
        return z, z
    qg = q.to(F64).view(hkv, hq // hkv, -1)
    s = torch.matmul(qg, k.to(F64).permute(1, 2, 0)) * scale
    p = torch.softmax(s, -1)
    vv = v.to(F64).permute(1, 0, 2)
    return torch.matmul(p, vv).reshape(q.shape), torch.matmul(p, vv.abs()).reshape(q.shape)


def assert_attention(got, want, weight, smax):
    """Bound of an output: half a bf16 step of it; P rounded to bf16, half a step
    of every weight, so of sum |p v|; and the fp32 of the scores, sums and exponents:
    a score of size smax (log2 units, before the reference is taken off) is off by at
    most 2^-24 per operation of its dot product and scaling, taken as 32 of
    them, which moves every weight by ln 2 times that."""
    soft = 32 * 2.0 ** -24 * max(1.0, smax)
    tol = BF16_HALF * want.abs() + (BF16_HALF + 2 * soft) * weight + 1e-30
    err = (got.to(F64) - want).abs()
    assert torch.isfinite(got).all()
    worst = (err / tol).max().item()
    assert worst <= 1.0, worst


def score_size(q, k, scale):
    """A bound of the scores in log2 units."""
    return float(q.to(F64).norm(dim=-1).max() * k.to(F64).norm(dim=-1).max() * abs(scale) / math.log(2))


def quantize(x):
    """(codes uint8, scale) of bf16 rows in the cache's format. (448.0 / amax is a reciprocal times 448
    here, so a code may lie a step from the append's at a tie.)"""
    x = x.float()
    amax = x.abs().amax(-1)
    inv = torch.where(amax > 0, 448.0 / amax, torch.zeros_like(amax))
    return (x * inv[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(U8), amax / 448.0


def dequantize(codes, scale):
    return codes.view(torch.float8_e4m3fn).to(F64) * scale.to(F64)[..., None]
