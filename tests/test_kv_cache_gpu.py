"""The paged key/value cache on the GPU: append, read and attend against the
64-bit oracle (oracle/kv_oracle.py).  Tolerances are the oracle's sums of the
roundings the kernels make."""

import numpy as np
import pytest
import torch

from locali_b200 import _lib
from locali_b200.kv_cache import PagedKVCache
from oracle import kv_oracle as K

pytestmark = pytest.mark.gpu

T = {"bf16": torch.bfloat16, "f16": torch.float16}


def np64(t):
    return t.detach().double().cpu().numpy()


class Case:
    """A filled cache, its page tables, and what the sequences hold."""

    def __init__(self, lens, rows, *, dtype="bf16", bits=16, gs=32, page=16, hk=2, d=64, seed=0, width=None, spread=1.0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.lens_l, self.rows_l, self.dtype, self.gs, self.gen = list(lens), list(rows), dtype, gs, g
        B = len(lens)
        need = [max(0, -(-n // page)) for n in lens]
        self.n_pages = sum(need) + 3
        perm = torch.randperm(self.n_pages, generator=g, device="cuda").cpu().tolist()
        W = max(need + [1]) if width is None else width
        tab = torch.full((B, W), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            tab[b, :n] = torch.tensor(perm[at:at + n], dtype=torch.int32)
            at += n
        self.table = tab.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        start = np.concatenate([[0], np.cumsum(rows)])
        self.start_l = start.tolist()
        self.start = torch.tensor(self.start_l, dtype=torch.int32, device="cuda")
        self.n = int(start[-1])
        self.cache = PagedKVCache(self.n_pages, page, hk, d, bits=bits, group_size=gs, dtype=T[dtype])
        # every slot of every page is written first, so slots behind a
        # sequence's end hold other data
        cells = self.n_pages * page
        k = (torch.randn(cells, hk, d, generator=g, device="cuda") * spread + 0.3).to(T[dtype])
        v = torch.randn(cells, hk, d, generator=g, device="cuda").to(T[dtype])
        allt = torch.arange(self.n_pages, dtype=torch.int32, device="cuda").unsqueeze(0)
        self.cache.append(k, v, allt, torch.tensor([cells], dtype=torch.int32, device="cuda"),
                          torch.tensor([0, cells], dtype=torch.int32, device="cuda"))

    def held(self, which):
        """[n_pages, hk, page, d] values in 64 bits (not rounded to the type), from the raw arrays."""
        c = self.cache
        a = c.k if which == "k" else c.v
        if c.bits == 16:
            return np64(a)
        s, b = (c.k_scales, c.k_biases) if which == "k" else (c.v_scales, c.v_biases)
        return K.dequantise(K.unpack(a.cpu().numpy().view(np.uint32), c.bits), np64(s), np64(b), c.group_size)

    def seq(self, held, b, h):
        L, pg = self.lens_l[b], self.cache.page_size
        j = np.arange(max(L, 0))
        pages = self.table.cpu().numpy()[b][j // pg]
        return held[pages, h, j % pg]

    def q(self, heads, seed=1, amp=1.5):
        g = torch.Generator("cuda").manual_seed(seed)
        return (torch.randn(self.n, heads, self.cache.head_dim, generator=g, device="cuda") * amp).to(T[self.dtype])


def attend_and_check(case, heads, *, window=0, sinks=0, scale=None, q=None, out=None, got=None, hk_v=None):
    c = case.cache
    q = case.q(heads) if q is None else q
    if got is None:
        got = c.attend(q, case.table, case.lens, case.start, window=window, sinks=sinks, scale=scale, out=out)
        torch.cuda.synchronize()
        c.check()
    sc = 1.0 / np.sqrt(c.head_dim) if scale is None else scale
    hk, hv = hk_v or (case.held("k"), case.held("v"))
    g, qn = np64(got), np64(q)
    G = heads // c.kv_heads
    for b, (L, n) in enumerate(zip(case.lens_l, case.rows_l)):
        r0 = case.start_l[b]
        pos = np.arange(L - n, L)
        see = K.visible(pos, max(L, 0), window, sinks)
        for h in range(heads):
            k, v = case.seq(hk, b, h // G), case.seq(hv, b, h // G)
            o, A, B, N = K.attention(qn[r0:r0 + n, h], k, v, see, sc)
            tol = K.tolerance(o, A, B, N, case.dtype, c.bits < 16, max(L, 1))
            x = g[r0:r0 + n, h]
            fine = np.isfinite(o)
            assert np.array_equal(np.isfinite(x), fine), (b, h)
            bad = np.abs(np.where(fine, x - o, 0.0)) > np.where(fine, tol, 1.0)
            assert not bad.any(), (b, h, np.argwhere(bad)[:4], np.abs(x - o)[bad].max(), tol[bad].min())
    return got


# ------------------------------------------------------------------ append and read
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,gs,d", [(16, 32, 64), (16, 32, 128), (8, 32, 64), (8, 64, 64), (8, 32, 128), (8, 64, 128),
                                       (8, 128, 128), (4, 32, 64), (4, 64, 64), (4, 32, 128), (4, 64, 128),
                                       (4, 128, 128)])
def test_append_holds_the_defined_codes(built, dtype, bits, gs, d):
    """Codes, scales and biases equal the definition bit for bit; the rest of the pages stays as it was."""
    case = Case([37, 5, 64, 1], [37, 2, 10, 0], dtype=dtype, bits=bits, gs=gs, d=d, hk=3, page=32)
    c = case.cache
    before = [None if t is None else t.clone() for t in (c.k, c.v, c.k_scales, c.k_biases, c.v_scales, c.v_biases)]
    g = torch.Generator("cuda").manual_seed(5)
    new = [(torch.randn(case.n, 3, d, generator=g, device="cuda") * s + o).to(T[dtype]) for s, o in ((2, 0.5), (1, 0))]
    new[0][3] = 1.25  # constant rows
    new[1][4] *= 1e-6
    new[1][5, :, ::2] = 0
    c.append(new[0], new[1], case.table, case.lens, case.start)
    k, v = c.read(case.table, case.lens, case.start, rows=case.n)
    torch.cuda.synchronize()
    c.check()
    tab = case.table.cpu().numpy()
    written = np.zeros((case.n_pages, c.page_size), bool)
    arrays = [None if t is None else t.cpu() for t in (c.k, c.v, c.k_scales, c.k_biases, c.v_scales, c.v_biases)]
    for which, x, got in ((0, new[0], k), (1, new[1], v)):
        xn = np64(x)
        if bits < 16:
            codes, s, b = K.quantise(xn, bits, gs, dtype)
            want = K.round_to(K.dequantise(codes, s, b, gs), dtype)
        else:
            want = xn
        assert np.array_equal(np64(got), want)
        for b_, (L, n) in enumerate(zip(case.lens_l, case.rows_l)):
            for i in range(n):
                p, r = L - n + i, case.start_l[b_] + i
                pg, sl = tab[b_, p // c.page_size], p % c.page_size
                written[pg, sl] = True
                if bits < 16:
                    assert np.array_equal(arrays[which][pg, :, sl].numpy().view(np.uint32), K.pack(codes[r], bits))
                    assert np.array_equal(np64(arrays[2 + 2 * which][pg, :, sl]), s[r])
                    assert np.array_equal(np64(arrays[3 + 2 * which][pg, :, sl]), b[r])
    keep = torch.from_numpy(~written)
    for old, now in zip(before, arrays):
        if old is not None:
            old = old.cpu()
            for h in range(3):
                assert torch.equal(old[:, h][keep].view(torch.int16), now[:, h][keep].view(torch.int16))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_append_next_to_a_half(built, dtype, bits):
    """Values on and one step beside the borders between two codes, extremes of very different size, the largest
    values of the type, subnormals: the exact code every time."""
    n, gs = 2**bits - 1, 32
    fin = K.FINITE_MAX[dtype]
    rng = np.random.default_rng(3)
    rows = []
    for _ in range(200):
        s = K.round_to(np.exp2(rng.uniform(-12, 4)), dtype)
        b = K.round_to(rng.choice([0.0, -s * 7, s * 3, -1e-3]), dtype)
        x = b + s * (rng.integers(0, n, gs) + rng.choice([0.5, 0.5 - 2.0**-9, 0.25], gs))
        x[0], x[1] = b, b + s * n
        rows.append(x)
    tiny = 2.0**-24 if dtype == "f16" else 2.0**-133
    rows += [np.linspace(-fin, fin, gs), np.linspace(0, fin, gs), np.full(gs, fin), np.full(gs, -fin),
             np.arange(gs) * tiny, np.arange(gs) * tiny * 3 - 40 * tiny, np.where(np.arange(gs) == 3, 1.0, tiny),
             np.where(np.arange(gs) % 2, -3.0, tiny * 5), np.zeros(gs)]
    x = K.round_to(np.stack(rows), dtype)
    x = np.concatenate([x, x[::-1]], -1).reshape(-1, 1, 64)
    codes, s, b = K.quantise(x, bits, gs, dtype)
    R = x.shape[0]
    page = 16
    np_ = -(-R // page)
    c = PagedKVCache(np_, page, 1, 64, bits=bits, group_size=gs, dtype=T[dtype])
    t = torch.from_numpy(x).to(T[dtype]).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    tab, lens, st = torch.arange(np_, **i32).unsqueeze(0), torch.tensor([R], **i32), torch.tensor([0, R], **i32)
    c.append(t, t.flip(0), tab, lens, st)
    k, v = c.read(tab, lens, st, rows=R)
    assert np.array_equal(np64(c.k_scales).reshape(-1, 2)[:R], s[:, 0])
    assert np.array_equal(np64(c.k_biases).reshape(-1, 2)[:R], b[:, 0])
    assert np.array_equal(K.unpack(c.k.cpu().numpy().view(np.uint32), bits).reshape(-1, 64)[:R], codes[:, 0])
    want = K.round_to(K.dequantise(codes, s, b, gs), dtype)
    assert np.isfinite(want).all()
    assert np.array_equal(np64(k), want) and np.array_equal(np64(v)[::-1], want)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_append_nonfinite_groups(built, bits):
    c = PagedKVCache(1, 16, 1, 64, bits=bits, group_size=32)
    x = torch.randn(3, 1, 64, device="cuda").to(torch.bfloat16)
    x[0, 0, 3], x[1, 0, 40], x[2, 0, 10] = float("nan"), float("inf"), -float("inf")
    i32 = dict(dtype=torch.int32, device="cuda")
    tab, lens, st = torch.zeros(1, 1, **i32), torch.tensor([3], **i32), torch.tensor([0, 3], **i32)
    c.append(x, x, tab, lens, st)
    k, _ = c.read(tab, lens, st, rows=3)
    if bits == 16:
        assert torch.equal(k.view(torch.int16), x.view(torch.int16))
    else:
        bad = torch.zeros(3, 2, dtype=torch.bool)
        bad[0, 0] = bad[1, 1] = bad[2, 0] = True
        assert torch.equal(torch.isnan(k).view(3, 2, 32).all(-1).cpu(), bad)
        assert torch.equal(torch.isnan(k).view(3, 2, 32).any(-1).cpu(), bad)


def test_append_and_read_strides_and_offsets(built):
    """Slices of a fused projection, transposed heads, odd offsets, a table with a row stride."""
    case = Case([70, 33], [20, 33], bits=8, hk=2, d=64)
    c, n = case.cache, case.n
    fused = torch.randn(n, 6, 64, device="cuda").to(torch.bfloat16)
    want_k, want_v = fused[:, 1:3].clone(), fused[:, 4:6].clone()
    c.append(want_k, want_v, case.table, case.lens, case.start)
    ref = c.read(case.table, case.lens, case.start, rows=n)
    wide = torch.full((2, case.table.shape[1] + 5), 10**6, dtype=torch.int32, device="cuda")
    wide[:, :case.table.shape[1]] = case.table
    heads_first = torch.empty(2, n, 64, dtype=torch.bfloat16, device="cuda").copy_(want_k.transpose(0, 1)).transpose(0, 1)
    odd = torch.empty(n * 2 * 64 + 3, dtype=torch.bfloat16, device="cuda")[3:].view(n, 2, 64).copy_(want_v)
    inner = torch.empty(n, 64, 2, dtype=torch.bfloat16, device="cuda").copy_(want_v.transpose(1, 2)).transpose(1, 2)
    for k, v in ((fused[:, 1:3], fused[:, 4:6]), (heads_first, odd), (heads_first, inner)):
        c.k.zero_(), c.v.zero_()
        c.append(k, v, wide[:, :case.table.shape[1]], case.lens, case.start)
        got = c.read(wide[:, :case.table.shape[1]], case.lens, case.start, rows=n)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


# ------------------------------------------------------------------ attention
GEOMS = [(16, 32, 64), (16, 32, 128), (8, 32, 64), (8, 64, 64), (8, 32, 128), (8, 64, 128), (8, 128, 128), (4, 32, 64),
         (4, 64, 64), (4, 32, 128), (4, 64, 128), (4, 128, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,gs,d", GEOMS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_single_tokens(built, dtype, bits, gs, d, window, sinks):
    case = Case([1, 2, 15, 16, 17, 100, 333, 0], [1] * 8, dtype=dtype, bits=bits, gs=gs, d=d, hk=2, page=48)
    case.start_l = list(range(9))
    attend_and_check(case, 8, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,gs,d", GEOMS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 5)])
def test_chunks(built, dtype, bits, gs, d, window, sinks):
    case = Case([200, 75, 300, 3], [70, 75, 1, 0], dtype=dtype, bits=bits, gs=gs, d=d, hk=2, page=32)
    attend_and_check(case, 6, window=window, sinks=sinks)


@pytest.mark.parametrize("hk,heads", [(1, 1), (1, 5), (1, 16), (1, 24), (2, 6), (4, 4), (1, 130), (3, 27)])
@pytest.mark.parametrize("rows", [1, 3, 9])
def test_head_layouts(built, hk, heads, rows):
    case = Case([90, 140], [rows, rows], bits=8, gs=64, d=64, hk=hk, page=16)
    attend_and_check(case, heads)


@pytest.mark.parametrize("page", [16, 48, 80, 256])
@pytest.mark.parametrize("rows", [1, 40])
def test_pages_that_end_inside_a_tile(built, page, rows):
    lens = [rows, rows + 1, page, page + 1, 2 * page - 1, 3 * page]
    lens = [max(n, rows) for n in lens]
    case = Case(lens, [rows] * len(lens), bits=4, gs=32, d=128, hk=1, page=page)
    attend_and_check(case, 4)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (16, 0), (17, 20), (63, 64), (64, 1), (65, 130), (128, 5),
                                          (1000, 7), (2**31 - 1, 2**31 - 1)])
@pytest.mark.parametrize("rows", [1, 2, 150])
def test_window_and_first_tokens(built, window, sinks, rows):
    case = Case([max(rows, n) for n in (1, 64, 129, 400)], [rows] * 4, bits=16, d=64, hk=1, page=16)
    attend_and_check(case, 3, window=window, sinks=sinks)


@pytest.mark.parametrize("rows", [1, 3, 70])
def test_rows_that_see_nothing(built, rows):
    """Sequences shorter than their rows: rows with a negative position see nothing and are zero; append skips them
    and read gives zeros."""
    lens = [rows - 1, 0, rows // 2, rows + 40]
    case = Case(lens, [rows] * 4, bits=8, gs=32, d=64, hk=2)
    got = attend_and_check(case, 4, window=8, sinks=1)
    for b, L in enumerate(lens):
        for i in range(rows):
            if L - rows + i < 0:
                assert (got[b * rows + i] == 0).all()
    before = case.cache.k.clone()
    x = torch.full((case.n, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    case.cache.append(x, x, case.table, case.lens, case.start)
    k, v = case.cache.read(case.table, case.lens, case.start, rows=case.n)
    case.cache.check()
    assert int((case.cache.k != before).any(-1).sum()) <= 2 * sum(min(n, rows) for n in lens)
    for b, L in enumerate(lens):
        for i in range(rows):
            want = 3.0 if L - rows + i >= 0 else 0.0
            assert (k[b * rows + i] == want).all() and (v[b * rows + i] == want).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("rows", [1, 5, 150])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_hidden_infinities_and_nan(built, bits, rows, window, sinks, bad):
    """What a row does not see does not touch it: non-finite keys and values behind the sequence's end, in other
    pages' slots, and at positions that some rows of the chunk see and others do not."""
    case = Case([rows + 61, rows], [rows, rows], bits=bits, gs=32, d=64, hk=1, page=48)
    c = case.cache
    arrays = [c.k, c.v] if bits == 16 else [c.k_scales, c.v_scales]
    L = case.lens_l[0]
    tab = case.table.cpu()
    for t in arrays:
        used = torch.zeros(case.n_pages, c.page_size, dtype=torch.bool)
        for b, n in enumerate(case.lens_l):
            for j in range(n):
                used[tab[b, j // c.page_size], j % c.page_size] = True
        t.transpose(1, 2)[~used.cuda()] = bad
        for j in {L - 1, L - 1 - rows // 2, 30, 1}:
            t[tab[0, j // c.page_size], 0, j % c.page_size, 0] = bad
    with np.errstate(invalid="ignore"):
        hk = tuple(case.held(w) for w in "kv")
        if window and rows == 1:
            pass
        attend_and_check(case, 2, window=window, sinks=sinks, hk_v=hk)


def test_hidden_values_only(built):
    """Non-finite values (keys finite) at the last positions of a chunk: earlier rows stay finite, later ones do not."""
    for bits, rows in ((16, 150), (8, 150), (4, 7), (16, 7)):
        case = Case([rows + 30], [rows], bits=bits, gs=32, d=64, hk=1, page=16)
        c, j = case.cache, rows + 30 - 3
        pg = int(case.table[0, j // 16])
        t = c.v if bits == 16 else c.v_biases
        t[pg, 0, j % 16, -1] = float("inf")
        got = attend_and_check(case, 2)
        assert torch.isfinite(got[:rows - 3]).all() and not torch.isfinite(got[rows - 3:]).all()


@pytest.mark.parametrize("rows", [1, 4, 100])
def test_large_scores(built, rows):
    """Scores of a few hundred: one key takes all; sharp and flat scales."""
    case = Case([150 + rows], [rows], bits=16, d=128, hk=1, page=16, spread=6.0)
    q = case.q(4, amp=8.0)
    attend_and_check(case, 4, q=q)
    attend_and_check(case, 4, q=q, scale=0.0)
    attend_and_check(case, 4, q=q, scale=1e-3)


@pytest.mark.parametrize("rows", [1, 40])
def test_long_cache(built, rows):
    """Thousands of keys over many blocks and a split key axis."""
    case = Case([9000, 31, 4097], [rows] * 3, bits=4, gs=64, d=128, hk=1, page=64)
    attend_and_check(case, 2)
    attend_and_check(case, 2, window=3000, sinks=4)


def test_offsets_pass_32_bits(built):
    """A cache of more than 2^32 bytes and 2^31 elements; the sequence lives in its last pages."""
    page, hk, d = 256, 8, 128
    n_pages = 2**32 // (page * hk * d * 2) + 40
    c = PagedKVCache(n_pages, page, hk, d)
    i32 = dict(dtype=torch.int32, device="cuda")
    L = 600
    tab = torch.tensor([[n_pages - 1, n_pages - 3, n_pages - 2]], **i32)
    lens, st = torch.tensor([L], **i32), torch.tensor([0, L], **i32)
    k, v = (torch.randn(L, hk, d, device="cuda").to(torch.bfloat16) for _ in range(2))
    c.append(k, v, tab, lens, st)
    a, b = c.read(tab, lens, st, rows=L)
    assert torch.equal(a, k) and torch.equal(b, v)
    small = PagedKVCache(3, page, hk, d)
    small.append(k, v, torch.tensor([[2, 0, 1]], **i32), lens, st)
    for n in (1, 300):
        q = torch.randn(n, 16, d, device="cuda").to(torch.bfloat16)
        s = torch.tensor([0, n], **i32)
        x = c.attend(q, tab, lens, s)
        y = small.attend(q, torch.tensor([[2, 0, 1]], **i32), lens, s)
        c.check()
        assert torch.equal(x, y)
    del c
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 3, 60])
def test_rows_behind_the_last_sequence(built, rows):
    case = Case([100, 64], [rows, rows], bits=8, gs=32, d=64, hk=2)
    c, n = case.cache, case.n
    q = torch.randn(n + 37, 4, 64, device="cuda").to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    c.attend(q, case.table, case.lens, case.start, out=out)
    # the number of rows may choose another kernel than q[:n] alone: held to the oracle, not to those bits
    attend_and_check(case, 4, q=q[:n], got=out[:n])
    assert (out[n:] == 7).all()
    k, v = c.read(case.table, case.lens, case.start, rows=n)
    o = tuple(torch.full((n + 37, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    c.read(case.table, case.lens, case.start, out=o)
    assert torch.equal(o[0][:n], k) and torch.equal(o[1][:n], v) and (o[0][n:] == 7).all() and (o[1][n:] == 7).all()
    before = (c.k.clone(), c.v.clone())
    x = torch.zeros(n + 37, 2, 64, dtype=torch.bfloat16, device="cuda")
    x[:n] = k
    y = torch.zeros_like(x)
    y[:n] = v
    c.append(x, y, case.table, case.lens, case.start)
    c.check()
    del before
    # a batch with no sequences leaves everything
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    out.fill_(7.0)
    c.attend(q, case.table[:0], case.lens[:0], none, out=out)
    assert (out == 7).all()


def test_query_strides(built):
    case = Case([60, 91], [11, 30], bits=16, d=64, hk=2)
    c, n = case.cache, case.n
    fused = torch.randn(n, 10, 64, device="cuda").to(torch.bfloat16)
    want = c.attend(fused[:, 3:7].contiguous(), case.table, case.lens, case.start)
    heads_first = torch.empty(4, n, 64, dtype=torch.bfloat16, device="cuda").copy_(fused[:, 3:7].transpose(0, 1))
    odd = torch.empty(n * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(n, 4, 64).copy_(fused[:, 3:7])
    for q in (fused[:, 3:7], heads_first.transpose(0, 1), odd):
        assert torch.equal(c.attend(q, case.table, case.lens, case.start), want)
    one = case.q(4)[:1].expand(n, 4, 64)  # every row the same
    assert torch.equal(c.attend(one, case.table, case.lens, case.start),
                       c.attend(one.contiguous(), case.table, case.lens, case.start))


# ------------------------------------------------------------------ errors, streams, graphs
@pytest.mark.parametrize("rows", [1, 30])
def test_bad_pages_are_reported(built, rows):
    """A page id out of range, a table too short: the keys there are absent, check() raises once."""
    for bad in (-1, 10**9):
        case = Case([100, 80], [rows, rows], bits=8, gs=32, d=64, hk=1, page=16)
        c = case.cache
        tab = case.table.clone()
        tab[0, 2] = bad
        q = case.q(2)
        got = c.attend(q, tab, case.lens, case.start)
        with pytest.raises(_lib.LmoeError):
            c.check()
        c.check()
        # the same as those 16 keys hidden
        kn, vn, qn = case.held("k"), case.held("v"), np64(q)
        for h in range(2):
            see = K.visible(np.arange(100 - rows, 100), 100, 0, 0)
            see[:, 32:48] = False
            o, A, B, N = K.attention(qn[:rows, h], case.seq(kn, 0, 0), case.seq(vn, 0, 0), see, 0.125)
            assert (np.abs(np64(got)[:rows, h] - o) <= K.tolerance(o, A, B, N, "bf16", True, 100)).all()
        short = case.table[:, :4].contiguous()
        c.attend(q, short, case.lens, case.start)
        with pytest.raises(_lib.LmoeError):
            c.check()
        x = torch.ones(case.n, 1, 64, dtype=torch.bfloat16, device="cuda")
        before = c.k.clone()
        tab[:] = bad
        c.append(x, x, tab, case.lens, case.start)
        with pytest.raises(_lib.LmoeError):
            c.check()
        assert torch.equal(before, c.k)
        k, _ = c.read(tab, case.lens, case.start, rows=case.n)
        with pytest.raises(_lib.LmoeError):
            c.check()
        assert (k == 0).all()


@pytest.mark.parametrize("rows", [1, 4, 60])
def test_lengths_past_the_table_are_reported(built, rows):
    """A length the table has no room for, up to the largest: the positions behind the table are absent (and not
    walked), the others are seen."""
    case = Case([128, 90 + rows], [rows, rows], bits=8, gs=32, d=64, hk=1, page=16, width=12)
    c, q = case.cache, case.q(2)
    for length in (200, 128 + 10**6, 2**31 - 1):
        lens = torch.tensor([length, 90 + rows], dtype=torch.int32, device="cuda")
        tab = case.table[:, :8].contiguous()  # room for 128 positions
        got = c.attend(q, tab, lens, case.start)
        with pytest.raises(_lib.LmoeError):
            c.check()
        kn, vn, qn = case.held("k"), case.held("v"), np64(q)
        for h in range(2):
            pos = np.arange(length - rows, length)
            see = K.visible(np.minimum(pos, 10**6), 128, 0, 0)
            o, A, B, N = K.attention(qn[:rows, h], case.seq(kn, 0, 0), case.seq(vn, 0, 0), see, 0.125)
            assert (np.abs(np64(got)[:rows, h] - o) <= K.tolerance(o, A, B, N, "bf16", True, 128)).all()
        # a window that lies wholly behind the table sees nothing
        if length > 10**5:
            assert (c.attend(q, tab, lens, case.start, window=50)[:rows] == 0).all()
            with pytest.raises(_lib.LmoeError):
                c.check()
        k, v = c.read(tab, lens, case.start, rows=case.n)
        with pytest.raises(_lib.LmoeError):
            c.check()


def test_bad_row_starts_are_reported(built):
    case = Case([50, 60], [5, 6], bits=16, d=64, hk=1)
    c = case.cache
    q = case.q(2)
    x = torch.ones(case.n, 1, 64, dtype=torch.bfloat16, device="cuda")
    for st in ([0, 50, 11], [0, 8, 5], [-3, 5, 11], [0, 5, 12]):
        start = torch.tensor(st, dtype=torch.int32, device="cuda")
        for call in (lambda: c.attend(q, case.table, case.lens, start), lambda: c.append(x, x, case.table, case.lens, start),
                     lambda: c.read(case.table, case.lens, start, rows=case.n)):
            call()
            with pytest.raises(_lib.LmoeError):
                c.check()
    neg = torch.tensor([50, -5], dtype=torch.int32, device="cuda")
    got = c.attend(q, case.table, neg, case.start)
    assert (got[5:] == 0).all()
    with pytest.raises(_lib.LmoeError):
        c.check()


def test_refusals(built):
    case = Case([50, 60], [1, 1], bits=8, gs=32, d=64, hk=2)
    c, q = case.cache, case.q(4)
    t, l, s = case.table, case.lens, case.start
    kv = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: c.attend(q.float(), t, l), lambda: c.attend(q[:, :3], t, l), lambda: c.attend(q[..., :32], t, l),
                lambda: c.attend(q[:1], t, l), lambda: c.attend(q, t.long(), l), lambda: c.attend(q, t, l.long()),
                lambda: c.attend(q, t[:1], l), lambda: c.attend(q, t, l, s[:2]), lambda: c.attend(q, t, l, s.long()),
                lambda: c.attend(q, t, l, scale=float("inf")), lambda: c.attend(q, t, l, scale=-0.1),
                lambda: c.attend(q, t, l, sinks=-1), lambda: c.attend(q, t, l, out=q), lambda: c.attend(q, t, l, out=kv),
                lambda: c.attend(q, t.cpu(), l), lambda: c.attend(q, t, l.cpu()),
                lambda: c.attend(q, t.t().contiguous().t(), l), lambda: c.append(kv, kv[:1], t, l),
                lambda: c.append(kv.half(), kv, t, l), lambda: c.append(kv[:, :1], kv[:, :1], t, l),
                lambda: c.read(t, l, s), lambda: c.read(t, l, rows=3), lambda: c.read(t, l, out=(kv, kv[:, :1])),
                lambda: c.read(t, l, out=(kv.float(), kv))):
        with pytest.raises((ValueError, _lib.LmoeError)):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        c.attend(q.cpu(), t, l)
    k = torch.zeros(2, 1, 16, 96, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(_lib.LmoeError):
        PagedKVCache.from_arrays(k, k)
    with pytest.raises(_lib.LmoeError):
        PagedKVCache(2, 24, 1, 64)
    with pytest.raises(ValueError):
        PagedKVCache.from_arrays(k[..., :64], k[..., :64])
    with pytest.raises(ValueError):
        PagedKVCache.from_arrays(torch.zeros(2, 1, 16, 16, dtype=torch.int32, device="cuda"),
                                 torch.zeros(2, 1, 16, 16, dtype=torch.int32, device="cuda"), bits=8, group_size=32)
    c.check()


@pytest.mark.parametrize("bits,gs", [(16, 32), (8, 32), (4, 64)])
def test_many_short_chunks(built, bits, gs):
    """More tiles than launch blocks, so one tile's results leave while the next one's keys and values arrive: every
    sequence's rows equal those of a call of its own."""
    rng = np.random.default_rng(4)
    rows = rng.integers(20, 60, 150).tolist()
    lens = [int(r + rng.integers(0, 150)) for r in rows]
    case = Case(lens, rows, bits=bits, gs=gs, d=128, hk=3, page=16)
    c, q = case.cache, case.q(12)
    first = c.attend(q, case.table, case.lens, case.start)
    for _ in range(5):
        assert torch.equal(first, c.attend(q, case.table, case.lens, case.start))
    for b in range(0, 150, 7):
        a, e = case.start_l[b], case.start_l[b + 1]
        st = torch.tensor([0, e - a], dtype=torch.int32, device="cuda")
        one = c.attend(q[a:e], case.table[b:b + 1], case.lens[b:b + 1], st)
        # the same arithmetic unless the tile was cut over two launch blocks: then two sums of terms rounded once
        assert float((one.float() - first[a:e].float()).abs().max()) <= 4 * 2.0**-8 * float(c.v.abs().max() if bits == 16
                                                                                           else 6.0)
    c.check()


@pytest.mark.parametrize("rows", [1, 50])
def test_repeatable_and_on_a_side_stream(built, rows):
    case = Case([3000, 500, 40 + rows], [rows] * 3, bits=8, gs=64, d=128, hk=2, page=64)
    q = case.q(8)
    first = case.cache.attend(q, case.table, case.lens, case.start)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(case.cache.attend(q, case.table, case.lens, case.start))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)


@pytest.mark.parametrize("rows", [1, 6, 90])
def test_two_captured_graphs(built, rows):
    """A decode step (append, attend, read) captured twice and replayed on two streams, with lengths that move
    between replays: each replay equals the eager calls."""
    case = Case([700, 90 + rows, rows], [rows] * 3, bits=8, gs=32, d=64, hk=2, page=16, width=64)
    i32 = dict(dtype=torch.int32, device="cuda")
    case2 = Case([64, 1000, rows + 3], [rows] * 3, bits=8, gs=32, d=64, hk=2, page=16, width=80, seed=9)
    graphs = []
    for cs in (case, case2):
        x = torch.randn(cs.n, 2, 64, device="cuda").to(torch.bfloat16)
        q = cs.q(6)

        def step(cs=cs, x=x, q=q):
            cs.cache.append(x, x, cs.table, cs.lens, cs.start)
            return cs.cache.attend(q, cs.table, cs.lens, cs.start), cs.cache.read(cs.table, cs.lens, cs.start, rows=cs.n)

        want = [t.clone() for t in (lambda r: (r[0], *r[1]))(step())]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step()
        graphs.append((g, got, want, cs, step))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for s, (g, *_r) in zip(streams, graphs):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _g, got, want, *_r in graphs:
            for a, b in zip((got[0], *got[1]), want):
                assert torch.equal(a, b)
    g, got, _w, cs, step = graphs[0]
    cs.lens.copy_(torch.tensor([650, rows + 1, rows], **i32))
    g.replay()
    torch.cuda.synchronize()
    a = [t.clone() for t in (got[0], *got[1])]
    r = step()
    for x, y in zip(a, (r[0], *r[1])):
        assert torch.equal(x, y)
    cs.cache.check()


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_decode_loop_equals_whole_prompt(built, bits):
    """Prompt in one chunk, in uneven chunks, and token by token: the cache ends the same and the rows agree; the
    result feeds a routed-MoE block."""
    n, hk, heads, d, page = 53, 2, 4, 64, 16
    i32 = dict(dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(n, hk, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    q = torch.randn(n, heads, d, generator=g, device="cuda").to(torch.bfloat16)
    tab = torch.tensor([[3, 0, 2, 1]], **i32)
    caches, outs = [], []
    for cuts in ([0, n], [0, 1, 20, 22, n], list(range(n + 1))):
        c = PagedKVCache(4, page, hk, d, bits=bits, group_size=32)
        parts = []
        for a, b in zip(cuts, cuts[1:]):
            lens, st = torch.tensor([b], **i32), torch.tensor([0, b - a], **i32)
            if b - a == 1:
                st = None
            c.append(k[a:b], v[a:b], tab, lens, st)
            parts.append(c.attend(q[a:b], tab, lens, st))
        c.check()
        caches.append(c)
        outs.append(torch.cat(parts))
    for c in caches[1:]:
        assert torch.equal(c.k, caches[0].k) and torch.equal(c.v, caches[0].v)
    u = 2.0**-8
    for o in outs[1:]:
        # each within its own tolerance of the same exact rows: terms rounded once each (sum of p |v| is at most max |v|)
        lim = 2 * (float(v.abs().max()) + 1) * (5 * u + np.expm1(2 * u * 40 if bits < 16 else 0.0) + 1e-4)
        assert float((o.float() - outs[0].float()).abs().max()) <= lim
    from locali_b200 import ops, synth
    cfg = synth.config("c0", tokens=n)
    layer = synth.make_layer(cfg, seed=0, device="cuda")
    kern = ops.MoEKernel(layer.router, layer.experts, layer.expert_slot, cfg.swiglu_limit)
    x = outs[0].reshape(n, heads * d).repeat(1, cfg.hidden // (heads * d))
    y = kern.block(x, -1, x)
    torch.cuda.synchronize()
    kern.ws.check()
    assert y.shape == x.shape and torch.isfinite(y).all()
