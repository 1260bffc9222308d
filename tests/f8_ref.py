"""The 8-bit float operators in 64 bits, from their definitions, and the
error that a 32-bit evaluation with one rounding per output may have.

Bounds, with u = 2^-24 (one f32 rounding, relative):
  codes    e4m3 rounds to within half a step: 2^-4 of the value, 2^-10 below
           the smallest normal code (times the scale), on a y that is itself
           off by Y · |y|.
  Y        norm: up to 32 squares per thread, 5 shuffles and 16 warps make
           under 60 roundings of the sum, halved by the root, and 4 more to y:
           34 u < 2^-18. SwiGLU: the exponent's rounding, |g| u, and a few u:
           2^-18 for |g| ≤ 40. GELU: erfc(z) moves by 2 z² of z's relative
           error, 2 u: 72 u at |x| = 6, and erfc's own 4 u: 2^-17.
  product  one rounding or truncation (2 u) of the running sum for each 16
           values of k that enter the accumulator, and 32 more for the join of
           blocks and splits, each relative to sum |a||b|; then the output's
           rounding.
"""
from __future__ import annotations

import torch

BLOCK = 128
Y_NORM, Y_SWIGLU, Y_GELU, Y_NONE = 2.0 ** -18, 2.0 ** -18, 2.0 ** -17, 2.0 ** -23


def blocks_max(y, block_rows):
    r, k = y.shape
    p = torch.nn.functional.pad(y.abs(), (0, -k % BLOCK, 0, -r % block_rows))
    p = p.view(p.shape[0] // block_rows, block_rows, p.shape[1] // BLOCK, BLOCK)
    return p.amax(dim=(1, 3)).clamp_min(2.0 ** -100)


def spread(scales, rows, k, block_rows):
    s = scales.double().repeat_interleave(BLOCK, 1)[:, :k]
    return s.repeat_interleave(block_rows, 0)[:rows]


def check_quantised(y, q, scales, block_rows, rel):
    """q, scales against the exact y (float64)."""
    want = blocks_max(y, block_rows) / 448.0
    assert scales.shape == want.shape
    off = ((scales.double() - want).abs() / want).max().item()
    assert off <= rel + 2.0 ** -23, f"scales off by {off:.3g}"
    s = spread(scales, *y.shape, block_rows)
    err = (q.double() * s - y).abs()
    # The code is the rounding of y · inv, inv and the scale off by u each.
    tol = y.abs() * (2.0 ** -4 + 2 * rel + 2.0 ** -22) + s * 2.0 ** -10 * (1 + 2.0 ** -10)
    worst = (err - tol).max().item()
    assert worst <= 0, f"codes off by {worst:.3g} more than half a step"


def values(q, scales, block_rows):
    return q.double() * spread(scales, q.shape[0], q.shape[1], block_rows)


def check_product(got, want, mag, k, bias=None):
    """got (its own type) against want = a · bᵀ (+ bias) in float64, with
    mag = |a| · |b|ᵀ (+ |bias|)."""
    u = 2.0 ** -24
    half = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[got.dtype]
    tiny = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[got.dtype]
    acc = 2 * u * (k / 16 + 32) * mag
    err = (got.double() - want).abs()
    worst = (err - (acc * (1 + half) + want.abs() * half + tiny)).max().item()
    assert worst <= 0, f"product off by {worst:.3g} more than its bound, max error {err.max().item():.3g}"


def pitched(t):
    """t with rows that start at multiples of 16 bytes (the room between them
    filled with the bytes of NaN, which nothing may read)."""
    k, e = t.shape[-1], t.element_size()
    wide = -(-k * e // 16) * 16 // e
    if wide == k:
        return t.contiguous()
    room = torch.full((*t.shape[:-1], wide * e), 0xFF, dtype=torch.uint8, device=t.device).view(t.dtype)
    room[..., :k] = t
    return room[..., :k]


def quantised(y, block_rows):
    """Plain quantisation of float32 y (inputs of the product tests)."""
    r, k = y.shape
    amax = blocks_max(y, block_rows)
    s = (amax / 448.0).float()
    inv = spread(448.0 / amax, r, k, block_rows)
    return (y.double() * inv).float().to(torch.float8_e4m3fn), s
