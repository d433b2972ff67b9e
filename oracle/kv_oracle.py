"""The paged key/value cache and its attention in numpy, in 64 bits.

TEST INFRASTRUCTURE ONLY (see the package docstring).  Written from the
definitions in include/lmoe.h; there is no counterpart in the reference.
"""

from __future__ import annotations

import numpy as np

FINITE_MAX = {"bf16": 3.3895313892515355e38, "f16": 65504.0}
HALF_STEP = {"bf16": 2.0**-8, "f16": 2.0**-11}  # largest relative rounding error of the type


def round_to(x: np.ndarray, dtype: str) -> np.ndarray:
    """Values of the 16-bit type nearest to x (ties to even), as float64."""
    x = np.asarray(x, np.float64)
    if dtype == "f16":
        return x.astype(np.float16).astype(np.float64)
    # 8 significant bits, from 64 bits in one step
    with np.errstate(invalid="ignore"):
        m, e = np.frexp(x)
        e = np.maximum(e, -125)  # subnormals of the type
        step = np.ldexp(1.0, e - 8)
        y = np.where(np.isfinite(x), np.rint(x / step) * step, x)
    return np.where(np.abs(y) > FINITE_MAX["bf16"], np.copysign(np.inf, y), y)


def _below(s: np.ndarray, dtype: str) -> np.ndarray:
    """The next lower value of the type (positive s)."""
    if dtype == "f16":
        return np.nextafter(s.astype(np.float16), np.float16(0)).astype(np.float64)
    m, e = np.frexp(s)
    low = s - np.ldexp(1.0, e - 8)
    return np.where(m == 0.5, s - np.ldexp(1.0, e - 9), low)


def quantise(x: np.ndarray, bits: int, group: int, dtype: str):
    """(codes, scales, biases) of the last dimension's groups of x (values of the type)."""
    n = 2**bits - 1
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, group)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    b = g.min(-1)
    s = round_to(((g.max(-1) - b) / n).astype(np.float32), dtype)
    s = np.where(s * n + b > FINITE_MAX[dtype], _below(np.where(s > 0, s, 1.0), dtype), s)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.rint((g - b[..., None]) / s[..., None])
    q = np.where(s[..., None] > 0, np.clip(q, 0, n), 0.0)
    codes = np.where(bad[..., None], 0, np.nan_to_num(q)).astype(np.int64).reshape(x.shape)
    return codes, np.where(bad, np.nan, s), np.where(bad, np.nan, b)


def pack(codes: np.ndarray, bits: int) -> np.ndarray:
    per = 32 // bits
    c = codes.reshape(*codes.shape[:-1], -1, per).astype(np.uint64) << (np.arange(per, dtype=np.uint64) * bits)
    return c.sum(-1).astype(np.uint32)


def unpack(words: np.ndarray, bits: int) -> np.ndarray:
    per = 32 // bits
    c = words.astype(np.uint64)[..., None] >> (np.arange(per, dtype=np.uint64) * bits)
    return (c & (2**bits - 1)).astype(np.int64).reshape(*words.shape[:-1], -1)


def dequantise(codes, scales, biases, group):
    """scale * code + bias in 64 bits, not rounded."""
    c = codes.reshape(*codes.shape[:-1], -1, group).astype(np.float64)
    return (c * scales[..., None] + biases[..., None]).reshape(codes.shape)


def visible(pos: np.ndarray, keys: int, window: int, sinks: int) -> np.ndarray:
    """[rows, keys]: what a row at each position sees."""
    p, j = np.asarray(pos)[:, None], np.arange(keys)[None, :]
    see = (j <= p) & (p >= 0)
    if window > 0:
        see &= (j > p - window) | (j < sinks)
    return see


def attention(q, k, v, see, scale):
    """o [rows, d], and the sums the tolerance is made of: A [rows, d] = sum_j
    p_j |v_j|, B [rows] = the largest scale * sum |q| |k_j| of a visible j,
    N [rows, d] = sum_j |v_j| / sum_j exp(s_j - max s).  q [rows, d], k and v
    [keys, d] in 64 bits, see [rows, keys].  A row that sees nothing is 0;
    hidden keys are not looked at."""
    rows, d = q.shape
    o, A, N, B = np.zeros((rows, d)), np.zeros((rows, d)), np.zeros((rows, d)), np.zeros(rows)
    for r in range(rows):
        j = np.flatnonzero(see[r])
        if j.size == 0:
            continue
        with np.errstate(invalid="ignore", over="ignore"):
            s = scale * (k[j] @ q[r])
            e = np.exp(s - s.max())
            o[r] = (e @ v[j]) / e.sum()
            A[r], N[r] = (e @ np.abs(v[j])) / e.sum(), np.abs(v[j]).sum(0) / e.sum()
            B[r] = (scale * (np.abs(k[j]) @ np.abs(q[r]))).max()
    return o, A, B, N


def tolerance(o, A, B, N, dtype: str, quantised: bool, keys: int):
    """Largest error of the kernels' arithmetic.  With u the largest relative
    rounding error of the type:
      softmax terms rounded to the type       u A   (and 2^-25 N below f16's normal range)
      quantised values rounded to the type    u A
      quantised keys rounded to the type      a score moves by u B at most, a
                                              normalised term by a factor within exp(+-2 u B)
      the result rounded to the type          u |o|
      fp32: scores of d terms 2^-24 each step of sums of d and of `keys` terms,
      exp2 of a scaled score: (2 B + 8) 2^-22 A + keys 2^-24 A
    """
    u = HALF_STEP[dtype]
    uk = u if quantised else 0.0
    t = A * (u + uk + np.expm1(2 * uk * B)[:, None] + ((2 * B + 8) * 2.0**-22)[:, None] + keys * 2.0**-24)
    t = 1.01 * t + u * np.abs(o) * 1.01
    if dtype == "f16":
        t = t + N * 2.0**-25 + 2.0**-25
    return t + 1e-37


def expected_error(q, k, v, see, scale, dtype: str, values: bool, keys: bool):
    """(squared norm of the error that independent roundings leave, squared
    norm of the result) over all rows.

    A value x of mantissa m in [1, 2) is off by x times an error uniform in
    +-u / m; with log m uniform the mean of 1 / m^2 is 3 / (8 ln 2), so the
    error's deviation is g |x|, g = u sqrt(1 / (8 ln 2)) = 0.4247 u.  Rounded
    are the result, the softmax terms, the values (``values``) and the keys
    (``keys``: a score is then off by g scale sqrt(sum (q k)^2), and its term by
    as much of itself).  What fp32 leaves is below a hundredth of that."""
    g2 = HALF_STEP[dtype] ** 2 / (8 * np.log(2))
    err = norm = 0.0
    for r in range(q.shape[0]):
        j = np.flatnonzero(see[r])
        if j.size == 0:
            continue
        s = scale * (k[j] @ q[r])
        p = np.exp(s - s.max())
        p /= p.sum()
        o = p @ v[j]
        p2 = p * p
        e = (o * o).sum() + (1 + values) * (p2 @ (v[j] ** 2)).sum()
        if keys:
            off = scale**2 * ((k[j] * q[r]) ** 2).sum(1)
            e += (p2 * off) @ ((v[j] - o) ** 2).sum(1)
        err += g2 * e
        norm += (o * o).sum()
    return err, norm
