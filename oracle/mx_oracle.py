"""Float64 restatement of the microscaled formats and of the operators on them.

Test infrastructure only: values, codes and the storage layout are written here
from the formats' definitions, apart from the package's code.
"""

from __future__ import annotations

import numpy as np

BLOCK = {"mxfp4": 32, "nvfp4": 16, "mxfp8": 32}
TOP = {"mxfp4": 2, "mxfp8": 8}


def _code_values(exp_bits: int, man_bits: int, bias: int) -> np.ndarray:
    """Magnitudes of a small float format by code (no infinities)."""
    out = []
    for e in range(2 ** exp_bits):
        for m in range(2 ** man_bits):
            frac = m / 2 ** man_bits
            out.append(frac * 2.0 ** (1 - bias) if e == 0 else (1 + frac) * 2.0 ** (e - bias))
    return np.array(out)


E2M1 = _code_values(2, 1, 1)
E4M3 = _code_values(4, 3, 7)[:-1]  # the last code is NaN


def nearest(v: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the nearest magnitude of the grid, ties to the even code, saturating."""
    a = np.abs(v)
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    lo = hi - 1
    down, up = a - grid[lo], grid[hi] - a
    return np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)


def quantize(x: np.ndarray, fmt: str, g: float = 1.0) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """(codes without the sign, scale bytes, values) of x [M, K] padded to whole 32-column blocks.

    The quotients of nvfp4 are those of float32, as the format's operator states them.
    """
    m, k = x.shape
    size = BLOCK[fmt]
    kp = -(-k // 32) * 32
    p = np.zeros((m, kp))
    p[:, :k] = x
    b = p.reshape(m, -1, size)
    bad = ~np.isfinite(b).all(axis=2)
    b = np.where(bad[:, :, None], 0.0, b)
    amax = np.abs(b).max(axis=2)
    if fmt == "nvfp4":
        f = np.float32
        byte = nearest((amax.astype(f) / (f(6) * f(g))).astype(np.float64), E4M3)
        unit = E4M3[byte].astype(f) * f(g)
        with np.errstate(over="ignore"):
            y = np.where(unit[:, :, None] > 0, b.astype(f) / np.where(unit > 0, unit, 1)[:, :, None], 0)
        codes = nearest(y.astype(np.float64), E2M1)
        val = E2M1[codes] * E4M3[byte][:, :, None] * float(f(g))
        byte = np.where(bad, 0x7F, byte)
    else:
        e = np.maximum(np.frexp(amax)[1] - 1 - TOP[fmt], -127)
        e = np.where(amax == 0, -127, e)
        grid = E2M1 if fmt == "mxfp4" else E4M3
        codes = nearest(np.ldexp(b, -e[:, :, None]), grid)
        val = np.ldexp(grid[codes], e[:, :, None])
        byte = np.where(bad, 255, e + 127)
    val = np.where(bad[:, :, None], np.nan, np.copysign(val, b))
    codes = np.where(bad[:, :, None], 0, codes)
    return codes.reshape(m, kp), byte, val.reshape(m, kp)[:, :k]


def scale_layout(byte: np.ndarray) -> np.ndarray:
    """Scale bytes [M, blocks] at their places in the 512-byte chunks."""
    m, nb = byte.shape
    gb = -(-nb // 4)
    out = np.zeros((-(-m // 128)) * gb * 512, dtype=np.uint8)
    for r in range(m):
        for g in range(nb):
            out[((r // 128) * gb + g // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + g % 4] = byte[r, g]
    return out


def product_bound(ref: np.ndarray, mass: np.ndarray, k: int, dtype: str, extra: np.ndarray | float = 0.0) -> np.ndarray:
    """Elementwise error bound of a tensor-core product rounded once to ``dtype``.

    Half an ulp of the result (8 significant bits in bf16, 11 in fp16: 2^-8 and 2^-11 of it); one float32 rounding (2^-23 for a truncating adder)
    per 16-deep step of the accumulation, relative to the sum of magnitudes
    ``mass``, plus a few for the epilogue; ``extra`` for operands that were rounded.
    """
    half_ulp = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11
    tiny = 2.0 ** -133 if dtype == "bf16" else 2.0 ** -25
    acc = (k / 16 + 8) * 2.0 ** -23 * mass + extra
    return half_ulp * (np.abs(ref) + acc) + acc + tiny
