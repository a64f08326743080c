"""Plain 64-bit forms of the serving operators (rotary positions, the paged
cache, attention over it), on the CPU, for the tests.  The quantiser is the
oracle's, which is pinned to the reference."""
import math

import numpy as np
import torch

import oracle

EPS16, EPS32 = 2.0 ** -11, 2.0 ** -24  # half a step of FP16 and FP32, relative


def angles(table, positions):
    """cos, sin [..., pairs] float64 of the float32 table at integer positions."""
    t = table.double()[positions.long()]
    return t[..., 0], t[..., 1]


def rotate(x, cos, sin, interleaved):
    """(y, bound): the rotation in 64 bits and the sum of |products| of every element."""
    x = x.double()
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2 : r])
    ya, yb = a * cos - b * sin, a * sin + b * cos
    size_a, size_b = (a * cos).abs() + (b * sin).abs(), (a * sin).abs() + (b * cos).abs()

    def put(ta, tb, rest):
        t = torch.stack((ta, tb), -1).flatten(-2) if interleaved else torch.cat((ta, tb), -1)
        return torch.cat((t, rest), -1)

    return put(ya, yb, x[..., r:]), put(size_a, size_b, x[..., r:] * 0)


def rotary_bound(y, size, dtype):
    """Two rounded FP32 products and their rounded sum (at most 2^-23 of the
    products' sizes), then one rounding to the type; below FP16's normal range
    half a step is 2^-25."""
    arithmetic = 2 * EPS32 * size
    return arithmetic + (EPS16 * (y.abs() + arithmetic) + 2.0 ** -25 if dtype == torch.float16 else 0)


def quantized(x, ocp=False):
    """float64 values of rows after the quantiser (a scale byte of 255 comes with zero codes only)."""
    codes, scales = oracle.quantize(x.float().numpy(), int(ocp))
    return torch.from_numpy(oracle.dequantize(codes, np.minimum(scales, 254))).double()


def unpack(k_codes, k_scales):
    """float64 values of packed codes [..., D/2] with scales [..., D/32]."""
    c = torch.stack((k_codes & 15, k_codes >> 4), -1).flatten(-2).numpy()
    return torch.from_numpy(oracle.dequantize(c, k_scales.numpy())).double()


def read(cache, table_row, start, length):
    """float64 K, V [kv_heads, length, D] of one sequence (CPU tensors of a cache)."""
    codes, scales, v = cache
    page = v.shape[2]
    pos = torch.arange(start, start + length)
    at, off = table_row.long()[pos // page], pos % page
    return unpack(codes[at, :, off], scales[at, :, off]).transpose(0, 1), v[at, :, off].double().transpose(0, 1)


def attend(q, k, v, scale=None):
    """(out, lse, size) for q [heads, D] (quantised, 64 bits) over k, v
    [kv_heads, n, D]: size = softmax . |v|, what rounding P is relative to."""
    hk, n, d = k.shape
    if n == 0:
        z = torch.zeros(q.shape, dtype=torch.float64)
        return z, torch.full((q.shape[0],), math.inf, dtype=torch.float64), z
    g = q.shape[0] // hk
    z = torch.einsum("hgd,hnd->hgn", q.view(hk, g, d), k) * (scale or 1 / math.sqrt(d))
    p = torch.softmax(z, -1)
    return ((p @ v).flatten(0, 1), torch.logsumexp(z, -1).flatten(), (p @ v.abs()).flatten(0, 1))


def attend_bound(out, size, n, vmax, zmax, out_dtype):
    """How far the kernel may be off, element by element.

    The scores are exact sums of few-bit products; scaling them rounds
    (2^-23 |z|, twice) and the exponential is good to 2^-21, so every p is off
    by at most e = 2^-21 + 2^-22 |z| relative, and so are sum and quotient
    together by 3 e; the FP32 sums add n / 128 + 64 roundings.  FP16 output: p
    is rounded to FP16 (2^-11); FP32 output: to two FP16 parts (2^-21).  Below
    FP16's normal range a part's half step is 2^-25, while the sum of all p is
    at least 1.  Last the result is rounded to its type."""
    e = 3 * (2.0 ** -21 + 2.0 ** -22 * zmax) + (n / 128 + 64) * EPS32
    e += EPS16 if out_dtype == torch.float16 else 2.0 ** -21
    bound = e * size + n * 2.0 ** -25 * vmax
    if out_dtype == torch.float16:
        bound = bound + EPS16 * (out.abs() + bound) + 2.0 ** -25
    else:
        bound = bound + EPS32 * out.abs()
    return bound


def lse_bound(lse, n, zmax):
    """The errors of p above, in the logarithm, and FP32 roundings of the result."""
    return 2.0 ** -21 + 2.0 ** -22 * zmax + (n / 128 + 64) * EPS32 + 4 * EPS32 * (lse.abs() + 1)
