"""The paged key/value cache on the host: refusals of the C entry points and
of PagedKVCache (no kernel runs), and the oracle against itself."""

import ctypes
import random

import numpy as np
import pytest
import torch

from locali_b200 import _lib, kv_cache
from oracle import kv_oracle as K

FAKE = 256  # a non-null, aligned address that nothing on the host follows


def _cache(**kw):
    f = dict(n_pages=4, page_size=16, kv_heads=2, head_dim=64, dtype=_lib.LMOE_BF16, bits=8, group_size=32)
    f.update(kw)
    p = {n: f.pop(n, FAKE) for n in ("k", "v", "k_scales", "k_biases", "v_scales", "v_biases")}
    return _lib.KVCache(p["k"], p["v"], p["k_scales"], p["k_biases"], p["v_scales"], p["v_biases"], f["n_pages"],
                        f["page_size"], f["kv_heads"], f["head_dim"], f["dtype"], f["bits"], f["group_size"])


def _rows(**kw):
    f = dict(page_table=FAKE, table_stride=8, table_width=8, n_seqs=3, lens=FAKE, row_start=None, n_rows=3)
    f.update(kw)
    return _lib.KVRows(*f.values())


def _append(c, r, **kw):
    f = dict(k=FAKE, kt=128, kh=64, v=FAKE, vt=128, vh=64)
    f.update(kw)
    return _lib.lmoe().lmoe_kv_append(ctypes.byref(c), ctypes.byref(r), *f.values(), None, None)


def _read(c, r, k=FAKE, v=FAKE):
    return _lib.lmoe().lmoe_kv_read(ctypes.byref(c), ctypes.byref(r), k, v, None, None)


def _attend(c, r, heads=4, **kw):
    f = dict(q=FAKE, qt=256, qh=64, scale=0.125, window=0, sinks=0, out=FAKE, scratch=FAKE, nbytes=1 << 40)
    f.update(kw)
    return _lib.lmoe().lmoe_paged_attention(ctypes.byref(c), ctypes.byref(r), heads, *f.values(), None, None)


BAD_CACHES = [
    (dict(head_dim=96), _lib.LMOE_EUNSUPPORTED), (dict(head_dim=256), _lib.LMOE_EUNSUPPORTED),
    (dict(bits=2), _lib.LMOE_EUNSUPPORTED), (dict(bits=3), _lib.LMOE_EUNSUPPORTED),
    (dict(group_size=128), _lib.LMOE_EUNSUPPORTED), (dict(group_size=16), _lib.LMOE_EUNSUPPORTED),
    (dict(group_size=0), _lib.LMOE_EUNSUPPORTED), (dict(page_size=24), _lib.LMOE_EUNSUPPORTED),
    (dict(page_size=0), _lib.LMOE_EINVAL), (dict(dtype=2), _lib.LMOE_EUNSUPPORTED),
    (dict(n_pages=0), _lib.LMOE_EINVAL), (dict(kv_heads=0), _lib.LMOE_EINVAL),
    (dict(k=None), _lib.LMOE_EINVAL), (dict(v=None), _lib.LMOE_EINVAL), (dict(k=FAKE + 8), _lib.LMOE_EINVAL),
    (dict(k_scales=None), _lib.LMOE_EINVAL), (dict(v_biases=FAKE + 2), _lib.LMOE_EINVAL),
]
BAD_ROWS = [dict(n_seqs=-1), dict(n_rows=-1), dict(n_rows=4), dict(table_width=-1), dict(table_stride=7),
            dict(lens=None), dict(page_table=None)]


@pytest.mark.parametrize("kw,status", BAD_CACHES)
def test_cache_refusals(built, kw, status):
    c, r = _cache(**kw), _rows()
    assert _append(c, r) == status and _read(c, r) == status and _attend(c, r) == status
    assert _lib.lmoe().lmoe_paged_attention_scratch(ctypes.byref(c), ctypes.byref(r), 4) == 0


@pytest.mark.parametrize("kw", BAD_ROWS)
def test_rows_refusals(built, kw):
    c, r = _cache(), _rows(**kw)
    assert _append(c, r) == _read(c, r) == _attend(c, r) == _lib.LMOE_EINVAL


def test_operand_refusals(built):
    c, r = _cache(), _rows()
    for kw in (dict(k=None), dict(v=None), dict(k=FAKE + 2), dict(kt=130), dict(vh=63)):
        assert _append(c, r, **kw) == _lib.LMOE_EINVAL
    for kw in (dict(k=None), dict(v=None), dict(v=FAKE + 8)):
        assert _read(c, r, **kw) == _lib.LMOE_EINVAL
    for kw in (dict(heads=3), dict(heads=0), dict(q=None), dict(q=FAKE + 4), dict(qt=257), dict(out=None),
               dict(out=FAKE + 8), dict(scale=float("nan")), dict(scale=-1.0), dict(scale=float("inf")),
               dict(sinks=-1)):
        assert _attend(c, r, **kw) == _lib.LMOE_EINVAL
    assert _attend(c, _rows(n_rows=1 << 30, row_start=FAKE), heads=64) == _lib.LMOE_EUNSUPPORTED
    lib = _lib.lmoe()
    need = lib.lmoe_paged_attention_scratch(ctypes.byref(c), ctypes.byref(r), 4)
    if need:
        assert _attend(c, r, nbytes=need - 1) == _lib.LMOE_EWORKSPACE
        assert _attend(c, r, scratch=None) == _lib.LMOE_EINVAL


def test_nothing_to_do(built):
    c = _cache()
    for r in (_rows(n_seqs=0, n_rows=0), _rows(n_seqs=0, n_rows=5, row_start=FAKE),
              _rows(n_seqs=3, n_rows=0, row_start=FAKE)):
        assert _append(c, r) == _read(c, r) == _attend(c, r) == _lib.LMOE_OK


def test_no_cpu_fallback(built):
    with pytest.raises(RuntimeError, match="CUDA"):
        kv_cache.PagedKVCache(2, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="bits"):
        kv_cache.PagedKVCache(2, 16, 1, 64, bits=2, device="cpu")
    with pytest.raises(ValueError, match="group_size"):
        kv_cache.PagedKVCache(2, 16, 1, 64, bits=4, group_size=48, device="cpu")


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_oracle_rounding_is_the_types(dtype):
    t = {"bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    rng = np.random.default_rng(0)
    x = (rng.standard_normal(4000) * np.exp2(rng.integers(-20, 14, 4000))).astype(np.float32)
    assert np.array_equal(K.round_to(x, dtype), torch.from_numpy(x).to(t).double().numpy())
    vals = torch.arange(1, 2000, dtype=torch.int16).view(t).double().numpy()
    assert np.array_equal(K.round_to(vals, dtype), vals)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_oracle_quantisation(dtype, bits):
    rng = np.random.default_rng(1)
    x = K.round_to(rng.standard_normal((50, 2, 128)) * 3, dtype)
    codes, s, b = K.quantise(x, bits, 32, dtype)
    assert codes.min() == 0 and codes.max() <= 2**bits - 1
    assert np.array_equal(K.unpack(K.pack(codes, bits), bits), codes)
    y = K.dequantise(codes, s, b, 32)
    # half a step, and the rounding of the scale over the whole range
    lim = np.repeat(s, 32, -1) * (0.5 + (2**bits - 1) * K.HALF_STEP[dtype] * 1.01)
    assert (np.abs(y - x) <= lim).all()
    top = np.zeros((1, 32))
    top[0, :2] = K.FINITE_MAX[dtype], -K.FINITE_MAX[dtype]
    c, s, b = K.quantise(top, bits, 32, dtype)
    assert np.isfinite(K.round_to(K.dequantise(c, s, b, 32), dtype)).all()


def test_oracle_visibility_by_definition():
    rnd = random.Random(2)
    for _ in range(50):
        W, S, keys = rnd.choice([0, 1, 3, 7]), rnd.choice([0, 1, 4]), rnd.randrange(1, 20)
        pos = [rnd.randrange(-2, keys) for _ in range(4)]
        see = K.visible(np.array(pos), keys, W, S)
        for i, p in enumerate(pos):
            for j in range(keys):
                assert see[i, j] == (0 <= j <= p and (W <= 0 or j > p - W or j < S))
