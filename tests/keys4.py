"""Whether the keys that a 4-bit arena holds are those of given positions, exactly up to what the fp32 rotation
before the rounding may differ by.

A rotated value in fp32 is off by at most 4.5 * 2^-24 times the larger of its pair (half steps of cos or sin, of
two products and of their sum).  So a held value is that of the value in 64 bits, or of that value moved by the
bound either way, under the scale of the block's largest magnitude moved by its bound either way, one scale
for all 32 values of a block."""

import numpy as np

from checks4 import VALUES, rotate


def scale_of(top):
    """The power of two (its exponent) of a block by its largest magnitude."""
    e = -127
    while e < 125 and top > 6 * 2.0 ** e:
        e += 1
    return e


def rounded(x, e):
    """x in the 4-bit form under 2^e: the nearest value, ties to the even code."""
    a = np.abs(x) / 2.0 ** e
    gap = np.abs(a[..., None] - VALUES)
    near = gap == gap.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    pick = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    return np.where(x < 0, -1.0, 1.0) * VALUES[pick] * 2.0 ** e


def wrong_keys(got, k, positions, f, interleaved):
    """How many blocks of 32 of the held rows got [n, heads, d] are not those of k, in fp32, at the positions."""
    k = k.astype(np.float64)
    x = rotate(k, positions, f, 1.0, interleaved)
    rd = 2 * len(f)
    p = np.abs(k[..., :rd])
    big = (np.maximum(p[..., 0::2], p[..., 1::2]).repeat(2, -1) if interleaved else
           np.tile(np.maximum(p[..., :rd // 2], p[..., rd // 2:]), 2))
    err = np.zeros(x.shape)
    err[..., :rd] = 4.5 * 2.0 ** -24 * big
    wrong = 0
    for g, v, e in zip(got.reshape(-1, 32), x.reshape(-1, 32), err.reshape(-1, 32)):
        scales = {scale_of(np.max(np.abs(v) + s * e)) for s in (-1, 0, 1)}
        wrong += not any(all(np.any([rounded(v + s * e, at) == g for s in (-1, 0, 1)], axis=0))
                         for at in scales)
    return wrong
