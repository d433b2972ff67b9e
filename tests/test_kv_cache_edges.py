"""Refusals of the key/value cache's C entries at the ends of their ranges (no
kernel runs), and the oracle's expected error against roundings made in numpy."""

import numpy as np
import pytest

from locali_b200 import _lib
from oracle import kv_oracle as K
from tests.test_kv_cache import FAKE, _attend, _cache, _rows


def test_results_past_what_the_kernels_count(built):
    """Results of more than 2^38 bytes (with one query row broadcast to all, nothing else need be large)."""
    c = _cache(kv_heads=128, head_dim=128)
    for n, heads in ((2**22 + 1, 256), (2**29, 128), (2**30, 128)):
        assert n * heads * 256 > 2**38 and n * (heads // 128) <= 2**30
        assert _attend(c, _rows(n_rows=n, row_start=FAKE), heads=heads, qt=0, qh=0) == _lib.LMOE_EUNSUPPORTED


# ------------------------------------------------------------------ the oracle's expected error
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,d", [(16, 64), (8, 64), (4, 128)])
def test_expected_error_tells_rounded_keys_apart(dtype, bits, d):
    """The kernels' roundings, made here one by one, come within a quarter of the expected error's norm, and keys that
    are rounded where they should not be, or values scaled by 1.01, pass it."""
    rng = np.random.default_rng(5)
    L, rows, scale = 300, 60, d**-0.5
    # channels with offsets, as trained projections have them: a key's rounding goes by its size, the softmax by what varies
    k = K.round_to(0.5 * rng.standard_normal((L, d)) + 6.0 * rng.choice([-1, 1], d), dtype)
    v = K.round_to(rng.standard_normal((L, d)), dtype)
    if bits < 16:
        k, v = (K.dequantise(*K.quantise(x, bits, 32, dtype), 32) for x in (k, v))
    q = K.round_to(1.5 * rng.standard_normal((rows, d)), dtype)
    see = K.visible(np.arange(L - rows, L), L, 0, 0)

    def made(keys, factor=1.0):
        kk = K.round_to(k, dtype) if keys else k
        vv = K.round_to(v, dtype) * factor
        out = np.zeros((rows, d))
        for r in range(rows):
            j = np.flatnonzero(see[r])
            s = scale * (kk[j] @ q[r])
            p = np.exp(s - s.max())
            out[r] = K.round_to((K.round_to(p, dtype) @ vv[j]) / p.sum(), dtype)
        return out

    exact = np.stack([K.attention(q[r:r + 1], k, v, see[r:r + 1], scale)[0][0] for r in range(rows)])

    def ratio(x, keys):
        err, norm = K.expected_error(q, k, v, see, scale, dtype, bits < 16, keys)
        assert np.isclose(norm, (exact**2).sum())
        return np.sqrt(((x - exact) ** 2).sum() / err)

    assert 0.75 < ratio(made(False), False) < 1.25
    if bits < 16:
        assert 0.75 < ratio(made(True), True) < 1.25
        assert ratio(made(True), False) > 1.5
    assert ratio(made(False, 1.01), False) > 1.5
