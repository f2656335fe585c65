"""Oracle of the 8-bit linear layer, in float64 numpy from the operators' definitions.

The reference has no 8-bit path, so nothing here restates it: a group's scale is the least power of two
s >= 2^-127 with max |v| <= 448 s, a code is v / s rounded to the nearest e4m3 value, ties to even.
"""

from __future__ import annotations

import numpy as np

GROUP = 128


def group_scales(values: np.ndarray) -> np.ndarray:
    """Scales [rows, ceil(cols / 128)] of float64 rows; NaN for groups with an infinity or a NaN."""
    rows, cols = values.shape
    scales = np.empty((rows, -(-cols // GROUP)))
    for g in range(scales.shape[1]):
        largest = np.abs(values[:, g * GROUP : (g + 1) * GROUP]).max(axis=1)
        for r in range(rows):
            a = largest[r]
            if not np.isfinite(a):
                scales[r, g] = np.nan
            elif a == 0:
                scales[r, g] = 1.0
            else:
                e = -127
                fraction, exponent = np.frexp(a)  # a = fraction 2^exponent, fraction in [0.5, 1)
                e = max(e, int(exponent) - 10)
                while 448.0 * 2.0**e < a:
                    e += 1
                scales[r, g] = 2.0**e
    return scales


def round_e4m3(values: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value of |v| <= 448, ties to even: three mantissa bits, steps of 2^-9 below 2^-6."""
    _, exponent = np.frexp(np.maximum(np.abs(values), 2.0**-6))
    step = np.exp2(exponent - 1.0 - 3.0)
    return np.rint(values / step) * step


def quantize(values: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes, scales) of float64 rows, both as the values they stand for."""
    values = np.asarray(values, dtype=np.float64)
    scales = group_scales(values)
    with np.errstate(invalid="ignore"):
        codes = round_e4m3(values / expand(scales, values.shape[1]))
    codes[np.isnan(expand(scales, values.shape[1]))] = np.nan
    return codes, scales


def expand(scales: np.ndarray, cols: int) -> np.ndarray:
    return np.repeat(scales, GROUP, axis=1)[:, :cols]


def silu_and_mul(x: np.ndarray) -> np.ndarray:
    gate, up = np.split(np.asarray(x, dtype=np.float64), 2, axis=1)
    with np.errstate(over="ignore"):
        return gate / (1.0 + np.exp(-gate)) * up


def rms_norm(x: np.ndarray, weight: np.ndarray, epsilon: float, residual: np.ndarray | None = None) -> tuple[np.ndarray, np.ndarray]:
    """(normalised rows, x + residual) in float64."""
    h = np.asarray(x, dtype=np.float64)
    if residual is not None:
        h = h + np.asarray(residual, dtype=np.float64)
    return h / np.sqrt((h * h).mean(axis=1, keepdims=True) + epsilon) * np.asarray(weight, dtype=np.float64), h


def matmul(lhs_codes, lhs_scales, rhs_codes, rhs_scales) -> np.ndarray:
    lhs = np.asarray(lhs_codes, dtype=np.float64) * expand(np.asarray(lhs_scales, dtype=np.float64), lhs_codes.shape[1])
    rhs = np.asarray(rhs_codes, dtype=np.float64) * expand(np.asarray(rhs_scales, dtype=np.float64), rhs_codes.shape[1])
    return lhs @ rhs.T
