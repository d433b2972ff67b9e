"""Refusals of the key/value cache's C entries at the ends of their ranges (no
kernel runs)."""

from locali_b200 import _lib
from tests.test_kv_cache import FAKE, _attend, _cache, _rows


def test_results_past_what_the_kernels_count(built):
    """Results of more than 2^38 bytes (with one query row broadcast to all, nothing else need be large)."""
    c = _cache(kv_heads=128, head_dim=128)
    for n, heads in ((2**22 + 1, 256), (2**29, 128), (2**30, 128)):
        assert n * heads * 256 > 2**38 and n * (heads // 128) <= 2**30
        assert _attend(c, _rows(n_rows=n, row_start=FAKE), heads=heads, qt=0, qh=0) == _lib.LMOE_EUNSUPPORTED
