"""Inputs and 64-bit definitions for the tests of the 4-bit-weight products and the expert routing."""
import torch

HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def codes(shape, gen):
    """Random signed 4-bit values [..., k] and their packed form [..., k/2] (even element in the low nibble)."""
    q = torch.randint(-8, 8, shape, generator=gen, dtype=torch.int32)
    packed = ((q[..., 0::2] & 15) | ((q[..., 1::2] & 15) << 4)).to(torch.uint8).view(torch.int8)
    return q, packed


def dequantised(q, scales, group):
    """float64 weights: code(i) * scale(i // group)."""
    at = torch.arange(q.shape[-1]) // group
    return q.double() * scales.double()[..., at]


def whole_case(m, n, k, group, dtype, scale_dtype, seed, lead=()):
    """Inputs whose products and sums are exact: small whole x, scales that are powers of two.  All partial sums are multiples of
    1/4 below 2^22, so fp32 holds them, and code * scale is exact in 16 bits: every output is the definition's value rounded once."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randint(-3, 4, (m, k), generator=gen).to(dtype)
    q, packed = codes((*lead, n, k), gen)
    scales = torch.exp2(torch.randint(-2, 2, (*lead, n, -(-k // group)), generator=gen).double()).to(scale_dtype)
    return x, q, packed, scales


def normal_case(m, n, k, group, dtype, scale_dtype, seed, lead=()):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=gen).to(dtype)
    q, packed = codes((*lead, n, k), gen)
    scales = (0.01 * torch.exp(0.5 * torch.randn(*lead, n, -(-k // group), generator=gen))).to(scale_dtype)
    return x, q, packed, scales


def close_to(got, x, w):
    """got [m, n] against x [m, k] @ w[n, k]^T in 64 bits.  With u = half a step of the type, an output is off by at most
      u |y|                        its own rounding,
      u S                          code * scale rounded to the type before the product (S = sum of |x| |w|), where that is done,
      (k / 16 + 16) 2^-22 S        fp32 sums of sixteen products at a time, each good to two of its last places,
    and, as roundings are independent, the 2-norm of the difference is within 2 u of the result's: one lost product in 4096
    would be 1.6 % of it."""
    u = HALF_STEP[got.dtype]
    ref = x.double() @ w.T
    size = x.double().abs() @ w.abs().T
    k = x.shape[1]
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double().cpu() - ref).abs()
    limit = u * ref.abs() + (u + (k / 16 + 16) * 2.0**-22) * size + tiny
    assert bool((off <= limit).all()), f"{int((off > limit).sum())} of {off.numel()} outputs off, worst {float((off / limit).max())} of the limit"
    if ref.numel() >= 256:
        assert float(off.norm()) <= 2 * u * float(ref.norm()), float(off.norm() / ref.norm())
