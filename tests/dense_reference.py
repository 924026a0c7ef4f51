"""The dense layers' operators from their definitions in 64 bits, and how far a kernel may be from them."""
import math

import torch

BLOCK = 128
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def floor_power(v):
    """2^floor(log2 v), v > 0, in 64 bits: without the fraction's bits"""
    return ((v.contiguous().view(torch.int64) >> 52) << 52).view(torch.float64)


def held(x):
    """what the 8-bit form of x's rows stands for, blocks of 128 along the last axis; what is not finite becomes NaN"""
    x = x.detach().double()
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at:at + BLOCK]
        finite = torch.where(torch.isfinite(part), part, torch.zeros_like(part))
        top = finite.abs().amax(dim=1, keepdim=True) / 448.0
        scale = floor_power(top.clamp(min=2.0 ** -126))
        scale = torch.where(scale < top, 2 * scale, scale)
        v = finite / scale
        grid = floor_power(v.abs().clamp(min=2.0 ** -6)) / 8
        out[:, at:at + BLOCK] = torch.where(torch.isfinite(part), torch.round(v / grid) * grid * scale, torch.full_like(part, math.nan))
    return out


def product_tolerance(a, b, y, dtype):
    """a [M, K], b [N, K] held values, y = a b^T (+ bias): the result's rounding, and its sum's.  In halves the products are exact and a
    block's 128 terms, the blocks and at most 512 parts are added in 32 bits: every addition is off by at most 2^-24 of what is added up.
    The 8-bit instruction cuts each product of a step at 2^-13 of the largest or below."""
    size = a.abs() @ b.abs().t()
    terms = 128 + (a.shape[1] + 127) // 128 + 4
    return HALF_STEP[dtype] * y.abs() + (terms * 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -13) * size + 2.0 ** -140


def newton_schulz(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    u = u.detach().double()
    x = u.t() if u.shape[0] > u.shape[1] else u
    x = x / (x.square().sum().sqrt() + eps)
    if not isinstance(coefficients[0], (tuple, list)):
        coefficients = [coefficients] * steps
    for a, b, c in coefficients:
        s = x @ x.t()
        x = a * x + (b * s + c * s @ s) @ x
    return x.t() if u.shape[0] > u.shape[1] else x


def orthogonal_tolerance(dtype, steps=5):
    """of the result's 2-norm.  A step adds at most the rounding of X (one half step of what it is held in) and of the polynomial's
    matrices (coefficients that add up to 10.3 at singular values near 1, each held to 2^-22): with pairs of halves
    (1 + 1 + 10.3) 2^-22 a step.  bf16 results: X and the polynomial in halves, 2^-11 each, after every second step, and the
    result's own rounding.  Later steps enlarge what is lost by at most what they enlarge small singular values by, and the
    matrices here have at least a third of their norm in those: a factor 3."""
    pair = 3 * 12.3 * 2.0 ** -22 * steps
    return pair + (3 * 2 * 2.0 ** -11 * ((steps + 1) // 2) if dtype == torch.bfloat16 else 0.0) + HALF_STEP[dtype]


def off(x, y):
    """2-norm of the difference over the 2-norm"""
    y = y.double()
    return float((x.double() - y).norm() / y.norm().clamp(min=1e-300))


def gradient(shape, seed, dtype=torch.float32, scale=1e-3):
    g = torch.Generator().manual_seed(seed)
    r, c = shape
    x = torch.randn(r, c, generator=g) * torch.exp(0.5 * torch.randn(1, c, generator=g))
    x = x + torch.randn(r, 2, generator=g) @ torch.randn(2, c, generator=g)
    return (scale * x).to(dtype)
