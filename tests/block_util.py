"""Plain 64-bit forms of the block-scaled operators, for the tests (numpy, no library code)."""
from __future__ import annotations

import math

import numpy as np

from ccglib_b200 import capi

BLOCK = 128
FMAX = {capi.FLOAT8E4M3: 448.0, capi.FLOAT8E5M2: 57344.0}
TINY = np.float32(2.0 ** -126)
U24 = 2.0 ** -24


def ceil(a, b):
    return -(-a // b)


def torch_type(code):
    import torch

    return {capi.FLOAT16: torch.float16, capi.BFLOAT16: torch.bfloat16,
            capi.FLOAT32: torch.float32, capi.FLOAT8E4M3: torch.float8_e4m3fn,
            capi.FLOAT8E5M2: torch.float8_e5m2}[code]


def round_fp8(v, code):
    """Nearest fp8 value (ties to even) of finite v, as float64; v must not exceed the format."""
    bits, low = (3, -6) if code == capi.FLOAT8E4M3 else (2, -14)
    v = np.asarray(v, np.float64)
    _, e = np.frexp(v)
    step = np.exp2(np.maximum(e - 1, low).astype(np.float64) - bits)
    return np.clip(np.rint(v / step) * step, -FMAX[code], FMAX[code])


def block_scales(x, code, block_rows):
    """x: planar [batch][2][rows][k] float32 -> (scales, factors) [batch][kb][rb] float32 by the
    definition."""
    batch, _, rows, k = x.shape
    kb, rb = ceil(k, BLOCK), ceil(rows, block_rows)
    mag = np.zeros((batch, rb * block_rows, kb * BLOCK), np.float32)
    mag[:, :rows, :k] = np.where(np.isfinite(x), np.abs(x), np.float32(0)).max(axis=1)
    amax = mag.reshape(batch, rb, block_rows, kb, BLOCK).max(axis=(2, 4))
    scale = np.maximum(amax / np.float32(FMAX[code]), TINY)
    with np.errstate(divide="ignore", over="ignore"):
        factor = np.where(scale > TINY, np.float32(FMAX[code]) / amax, np.float32(2.0 ** 126))
    return (np.ascontiguousarray(scale.transpose(0, 2, 1)),
            np.ascontiguousarray(factor.transpose(0, 2, 1)))


def per_element(scale, block_rows, rows, k):
    """[batch][kb][rb] -> [batch][rows][k]."""
    full = np.repeat(np.repeat(scale.transpose(0, 2, 1), block_rows, 1), BLOCK, 2)
    return full[:, :rows, :k]


def quantize(x, code, block_rows):
    """Planar float32 x -> (values [batch][2][rows][k] float64, scales), the definition's steps in
    float32 (numpy's division and product are correctly rounded)."""
    scale, factor = block_scales(x, code, block_rows)
    with np.errstate(invalid="ignore", over="ignore"):
        v = x * per_element(factor, block_rows, x.shape[2], x.shape[3])[:, None]
    finite = np.isfinite(v)
    q = round_fp8(np.where(finite, v, 0), code)
    special = v.astype(np.float64) if code == capi.FLOAT8E5M2 else np.full(v.shape, np.nan)
    return np.where(finite, q, special), scale


def scaled_product(a, sa, ga, b, sb, gb):
    """Values and scales -> (C complex128 [batch][m][n], S_re, S_im), S the sums of absolute
    products that bound the rounding errors."""
    def side(v, s, g):
        f = per_element(s.astype(np.float64), g, v.shape[2], v.shape[3])
        return v[:, 0] * f, v[:, 1] * f

    ar, ai = side(a.astype(np.float64), sa, ga)
    br, bi = (x.transpose(0, 2, 1) for x in side(b.astype(np.float64), sb, gb))
    c = ar @ br - ai @ bi + 1j * (ar @ bi + ai @ br)
    ar, ai, br, bi = abs(ar), abs(ai), abs(br), abs(bi)
    return c, ar @ br + ai @ bi, ar @ bi + ai @ br


def product_tolerance(c, s, k, type_out):
    """|C - C64| bound per real value.  fp8 products and their scale factors enter exactly; what
    rounds is float32 addition.  A block of 128 k takes 8 MMAs into its accumulator, each of which may
    lose one unit (2^-23) of a running sum below the block's share of S: 16 * 2^-24 S over all
    blocks.  Two float32 roundings per block for the scales: 2 * 2^-24 S.  Adding the k/128 blocks
    rounds running sums that are at most S: (k / 128) * 2^-24 S, and twice that where a tile's
    parts are added.  Last the rounding of the output, half a step."""
    u = {capi.FLOAT32: U24, capi.FLOAT16: 2.0 ** -11, capi.BFLOAT16: 2.0 ** -8}[type_out]
    small = {capi.FLOAT32: 2.0 ** -149, capi.FLOAT16: 2.0 ** -25, capi.BFLOAT16: 2.0 ** -133}[type_out]
    inner = (18 + 2 * ceil(k, BLOCK)) * U24 * s
    return inner * (1 + u) + u * np.abs(c) + small


def lay_out(x, axis, order):
    """Planar [batch][2][rows][k] -> the caller's layout (numpy or torch)."""
    perm = (0, 1, 2, 3)
    if order == capi.COL_MAJOR:
        perm = (0, 1, 3, 2)
    if axis == capi.INTERLEAVED:
        perm = (perm[0], perm[2], perm[3], perm[1])
    return x.permute(*perm).contiguous()


def canonical_c(c, axis, order):
    """C as stored -> [batch][2][m][n]."""
    if axis == capi.INTERLEAVED:
        c = c.permute(0, 3, 1, 2)
    if order == capi.COL_MAJOR:
        c = c.transpose(2, 3)
    return c.contiguous()


def c_shape(batch, m, n, axis, order):
    if order == capi.COL_MAJOR:
        m, n = n, m
    return (batch, m, n, 2) if axis == capi.INTERLEAVED else (batch, 2, m, n)


def random_operand(rng, batch, rows, k, code, block_rows):
    """fp8 values drawn over the format and positive scales over a few decades:
    (float8 tensor [batch][2][rows][pitch] whose padding is NaN, scale tensor), on the CPU."""
    import torch

    v = rng.standard_normal((batch, 2, rows, k)) * math.sqrt(FMAX[code])
    q = torch.from_numpy(round_fp8(np.clip(v, -FMAX[code], FMAX[code]), code)).float()
    pitch = capi.operand_pitch(k)
    buf = torch.full((batch, 2, rows, pitch), 0x7F, dtype=torch.uint8)
    buf[..., :k] = q.to(torch_type(code)).view(torch.uint8)
    s = np.exp(rng.uniform(-4, 4, (batch, ceil(k, BLOCK), ceil(rows, block_rows))))
    s /= FMAX[code]
    return buf.view(torch_type(code)), torch.from_numpy(s.astype(np.float32))
