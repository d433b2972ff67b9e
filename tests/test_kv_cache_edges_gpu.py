"""The paged key/value cache at its edges: lengths and offsets at the ends of
32 bits, sequences across the look-up's blocks, pages that a window has left
behind, extreme values, and how near to 64 bits each path comes."""

import numpy as np
import pytest
import torch

from locali_b200 import _lib
from locali_b200.kv_cache import PagedKVCache
from oracle import kv_oracle as K
from tests.test_kv_cache_gpu import T, Case, attend_and_check, np64

pytestmark = pytest.mark.gpu

I32 = dict(dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ lengths
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("rows", [1, 5, 60])
@pytest.mark.parametrize("window,sinks", [(1, 0), (50, 0), (50, 3), (70, 200)])
def test_windows_of_lengths_far_past_the_table(built, bits, rows, window, sinks):
    """The window of the largest length lies in the last key block that 32 bits can count: nothing of it is there,
    only the first tokens are seen."""
    case = Case([128, 90 + rows], [rows, rows], bits=bits, gs=32, d=64, hk=1, page=16, width=8 + (90 + rows) // 16)
    c, q = case.cache, case.q(2)
    tab = case.table[:, :8].contiguous()  # room for 128 positions
    kn, vn, qn = case.held("k"), case.held("v"), np64(q)
    for length in (2**31 - 1, 2**31 - 40, 2**31 - 128, 2**31 - 256, 2**31 - 300):
        got = c.attend(q, tab, torch.tensor([length, rows], **I32), case.start, window=window, sinks=sinks)
        with pytest.raises(_lib.LmoeError):
            c.check()
        see = np.zeros((rows, 128), bool)
        see[:, :sinks] = True
        for h in range(2):
            o, A, B, N = K.attention(qn[:rows, h], case.seq(kn, 0, 0), case.seq(vn, 0, 0), see, 0.125)
            assert (np.abs(np64(got)[:rows, h] - o) <= K.tolerance(o, A, B, N, "bf16", bits < 16, 128)).all()


@pytest.mark.parametrize("rows", [1, 5, 60])
def test_positions_up_to_the_largest(built, rows):
    """A table that names the same page over and over and has room for every position: windowed attention, append and
    read at the last positions there are; a length behind them is reported."""
    page, d = 1 << 20, 64
    c = PagedKVCache(2, page, 1, d, bits=4, group_size=64)
    tab = torch.zeros(1, 2048, **I32)
    tab[0, -1] = 1  # the last page alone is its own
    start = torch.tensor([0, rows], **I32)
    last = 2**31 - 256
    g = torch.Generator("cuda").manual_seed(0)
    fill = 300
    x, y = (torch.randn(fill, 1, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    c.append(x, y, tab, torch.tensor([last], **I32), torch.tensor([0, fill], **I32))
    c.check()
    lens = torch.tensor([last], **I32)
    k, v = c.read(tab, lens, torch.tensor([0, fill], **I32), rows=fill)
    c.check()
    for t, z in ((x, k), (y, v)):
        codes, s, b = K.quantise(np64(t), 4, 64, "bf16")
        assert np.array_equal(np64(z), K.round_to(K.dequantise(codes, s, b, 64), "bf16"))
    q = torch.randn(rows, 2, d, generator=g, device="cuda").to(torch.bfloat16)
    kn, vn = (np64(t).reshape(fill, d) for t in (k, v))
    for W in (1, 50, 200):
        got = c.attend(q, tab, lens, start, window=W)
        c.check()
        see = K.visible(np.arange(fill - rows, fill), fill, W, 0)
        for h in range(2):
            o, A, B, N = K.attention(np64(q)[:, h], kn, vn, see, 0.125)
            # kn, vn are rounded already: once more the same rounding
            assert (np.abs(np64(got)[:, h] - o) <= 2 * K.tolerance(o, A, B, N, "bf16", True, fill)).all()
    before = c.k.clone()
    for length in (last + 1, 2**31 - 1):
        over = torch.tensor([length], **I32)
        assert torch.isfinite(c.attend(q, tab, over, start, window=3)).all()
        with pytest.raises(_lib.LmoeError):
            c.check()
        c.append(x[:1], y[:1], tab, over)
        with pytest.raises(_lib.LmoeError):
            c.check()
    neg = torch.tensor([-2**31], **I32)
    c.append(x[:1], y[:1], tab, neg)
    with pytest.raises(_lib.LmoeError):
        c.check()
    assert torch.equal(before, c.k)


# ------------------------------------------------------------------ rows of many sequences
@pytest.mark.parametrize("first", [0, 3, 11])
@pytest.mark.parametrize("bits,dtype", [(16, "bf16"), (8, "bf16"), (4, "f16")])
def test_many_rows_across_sequences(built, first, bits, dtype):
    """More rows than get a launch block each, of sequences whose borders lie anywhere, some without rows and some
    shorter than theirs, rows in front of the first sequence and behind the last: every row in its place, the others
    as they were."""
    rng = np.random.default_rng(7)
    B, page, hk, d, gs = 140, 16, 2, 64, 32
    rows = rng.choice([0, 0, 1, 3, 17, 40], B)
    lens = np.where(rng.random(B) < 0.1, rows // 2, rows + rng.integers(0, 50, B))
    start = first + np.concatenate([[0], np.cumsum(rows)])
    n = int(start[-1]) + 13
    assert n > 1024
    need = -(-lens // page)
    tab = np.full((B, max(need)), -7, np.int32)
    perm, at = rng.permutation(int(need.sum()) + 2), 0
    for b in range(B):
        tab[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
    c = PagedKVCache(len(perm), page, hk, d, bits=bits, group_size=gs, dtype=T[dtype])
    g = torch.Generator("cuda").manual_seed(0)
    x, y = (torch.randn(n, hk, d, generator=g, device="cuda").to(T[dtype]) for _ in range(2))
    args = [torch.from_numpy(np.ascontiguousarray(a)).to(**I32) for a in (tab, lens, start)]
    c.append(x, y, *args)
    out = tuple(torch.full((n, hk, d), 7.0, dtype=T[dtype], device="cuda") for _ in range(2))
    c.read(*args, out=out)
    c.check()
    for t, got, held in ((x, out[0], c.k), (y, out[1], c.v)):
        want = np64(t)
        words = want
        if bits < 16:
            codes, s, b = K.quantise(want, bits, gs, dtype)
            want, words = K.round_to(K.dequantise(codes, s, b, gs), dtype), K.pack(codes, bits)
        cells = np.zeros((len(perm), page, hk, words.shape[-1]))
        expect = np.full((n, hk, d), 7.0)
        for b in range(B):
            for r in range(start[b], start[b + 1]):
                p = lens[b] - (start[b + 1] - r)
                expect[r] = want[r] if p >= 0 else 0.0
                if p >= 0:
                    cells[tab[b, p // page], p % page] = words[r]
        assert np.array_equal(np64(got), expect)
        held = np64(held) if bits == 16 else held.cpu().numpy().view(np.uint32)
        assert np.array_equal(held.transpose(0, 2, 1, 3), cells)


# ------------------------------------------------------------------ pages that a window has left behind
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("rows", [1, 7, 150])
@pytest.mark.parametrize("window,sinks", [(40, 4), (100, 0), (129, 20)])
def test_pages_no_row_sees_may_be_gone(built, bits, page, rows, window, sinks):
    """Pages between the first tokens and the window of a sequence's first row are looked up by nothing: a table that
    has them at -1 gives the same bits, and nothing is reported."""
    lens = [rows + 600, rows + 333, rows]
    case = Case(lens, [rows] * 3, bits=bits, gs=32, d=64, hk=2, page=page)
    c, q = case.cache, case.q(4)
    want = c.attend(q, case.table, case.lens, case.start, window=window, sinks=sinks)
    tab, gone = case.table.clone(), 0
    for b, L in enumerate(lens):
        for e in range(-(-L // page)):
            if e * page >= sinks and (e + 1) * page <= L - rows - window + 1:
                tab[b, e] = -1
                gone += 1
    assert gone > 10
    c.check()
    got = c.attend(q, tab, case.lens, case.start, window=window, sinks=sinks)
    c.check()
    assert torch.equal(got, want)
    attend_and_check(case, 4, window=window, sinks=sinks, q=q, got=got)
    # one page further is seen
    tab[0, (lens[0] - rows - window + 1) // page] = -1
    c.attend(q, tab, case.lens, case.start, window=window, sinks=sinks)
    with pytest.raises(_lib.LmoeError):
        c.check()


# ------------------------------------------------------------------ strides and arguments
def test_strides_of_dimensions_of_one(built):
    """A dimension of size one may have any stride: nothing is ever one step along it."""
    i32 = I32
    c = PagedKVCache(2, 16, 4, 64)
    base = torch.randn(5, 257, device="cuda").to(torch.bfloat16)
    one = torch.as_strided(base, (1, 4, 64), (257, 64, 1))  # a token stride of 257
    assert one.is_contiguous()
    tab, lens = torch.tensor([[1]], **i32), torch.tensor([3], **i32)
    c.append(one, one, tab, lens)
    k, v = c.read(tab, lens)
    assert torch.equal(k, one) and torch.equal(v, one)
    assert torch.equal(c.attend(one, tab, lens), c.attend(one.clone(memory_format=torch.contiguous_format), tab, lens))
    c1 = PagedKVCache(2, 16, 1, 64)
    x = torch.as_strided(base.view(-1), (2, 1, 64), (64, 37, 1))  # a head stride of 37
    tab, lens = torch.tensor([[1], [0]], **i32), torch.tensor([3, 9], **i32)
    c1.append(x, x, tab, lens)
    k, v = c1.read(tab, lens)
    assert torch.equal(k, x) and torch.equal(v, x)
    want = c1.attend(base.view(-1)[:128].view(2, 1, 64), tab, lens)
    assert torch.equal(c1.attend(x, tab, lens), want)
    c1.check()


@pytest.mark.parametrize("rows", [1, 40])
def test_windows_of_zero_and_less_are_none(built, rows):
    case = Case([90 + rows], [rows], d=64, hk=1)
    q = case.q(2)
    want = case.cache.attend(q, case.table, case.lens, case.start)
    for window in (0, -1, -2**31, -2**32 + 5, -2**40):
        got = case.cache.attend(q, case.table, case.lens, case.start, window=window, sinks=1)
        assert torch.equal(got, want), window


# ------------------------------------------------------------------ extreme values
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("rows", [1, 5, 60])
def test_keys_near_the_largest_value(built, bits, rows):
    """bf16 keys up to 1e38 and queries so small that the scores are ordinary."""
    case = Case([200 + rows, 70], [rows, min(rows, 50)], bits=bits, gs=32, d=64, hk=1, page=16)
    c, cells = case.cache, case.n_pages * 16
    k = (torch.randn(cells, 1, 64, device="cuda") * 1.5e38).clamp(-3.3e38, 3.3e38).to(torch.bfloat16)
    v = torch.randn(cells, 1, 64, device="cuda").to(torch.bfloat16)
    c.append(k, v, torch.arange(case.n_pages, **I32)[None], torch.tensor([cells], **I32), torch.tensor([0, cells], **I32))
    assert bits == 16 or float(c.k_scales.max()) > 4e38 / 2**bits
    attend_and_check(case, 2, q=case.q(2, amp=2.0**-122), scale=0.02)


@pytest.mark.parametrize("rows", [1, 5, 60])
@pytest.mark.parametrize("scale", [0.0, 1e-38, 3e-39])
def test_smallest_scales(built, rows, scale):
    """A scale of zero makes all terms equal, whatever the scores; a tiny one is taken as it is."""
    case = Case([200 + rows], [rows], d=64, hk=1)
    c = case.cache
    c.k.zero_()
    c.k[..., 0] = (torch.rand(c.k.shape[:3], device="cuda") * 1.5e19).to(torch.bfloat16)
    q = torch.zeros(case.n, 2, 64, dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1e19
    attend_and_check(case, 2, q=q, scale=scale)




@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("rows,seqs", [(1, 1200), (5, 1200), (60, 300)])
@pytest.mark.parametrize("drop", [8.0, 12.0, 17.1])
def test_f16_terms_far_below_the_first_token(built, bits, rows, seqs, drop):
    """One first token far above thousands of others, whose terms together still count: at exp(-17.1) each would be
    near half the smallest f16.  The terms are held 2^7 and more above that.  Many sequences (of the same pages), so
    that a row's keys are not cut over launch blocks, each with a largest term of its own."""
    L, d = 12000, 64
    case = Case([L], [rows], dtype="f16", bits=bits, gs=32, d=d, hk=1, page=16)
    c, g = case.cache, case.gen
    k = torch.randn(L, 1, d, generator=g, device="cuda") * 0.1
    k[:, :, 0] = 0.0
    k[0, 0, :] = 0.0
    k[0, 0, 0] = 4.0
    v = 100.0 + torch.randn(L, 1, d, generator=g, device="cuda")
    v[0] = 0.0
    c.append(k.half(), v.half(), case.table, case.lens, torch.tensor([0, L], **I32))
    q = torch.randn(seqs * rows, 2, d, generator=g, device="cuda")
    q[..., 0] = drop * 8.0 / 4.0
    q = q.half()
    start = torch.arange(seqs + 1, **I32) * rows
    got, qn = np64(c.attend(q, case.table.repeat(seqs, 1), case.lens.repeat(seqs), start)), np64(q)
    hk, hv = case.seq(case.held("k"), 0, 0), case.seq(case.held("v"), 0, 0)
    see = K.visible(np.arange(L - rows, L), L, 0, 0)
    for b in (0, 7, seqs // 2, seqs - 1):
        at = slice(b * rows, (b + 1) * rows)
        for h in range(2):
            o, A, B, N = K.attention(qn[at, h], hk, hv, see, 0.125)
            tol = K.tolerance(o, A, B, N * 2.0**-7, "f16", bits < 16, L)
            err = np.abs(got[at, h] - o)
            assert (err <= tol).all(), ((err / tol).max(), (err / np.abs(o)).max())


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("rows", [1, 5, 60])
@pytest.mark.parametrize("size", [3e38, 2.0**-96])
def test_values_of_the_largest_and_small_sizes(built, bits, rows, size):
    """bf16 values of one sign near the largest one, thousands of them with nearly equal terms: their sum before the
    division is far past the type.  And small ones, which the terms' scaling must not lose."""
    L = 6000 + rows
    case = Case([L, 300], [rows, rows], bits=bits, gs=32, d=64, hk=1, page=64)
    c, cells = case.cache, case.n_pages * 64
    k = torch.randn(cells, 1, 64, device="cuda").to(torch.bfloat16)
    v = (size * (0.9 + 0.1 * torch.rand(cells, 1, 64, device="cuda"))).to(torch.bfloat16)
    c.append(k, v, torch.arange(case.n_pages, **I32)[None], torch.tensor([cells], **I32), torch.tensor([0, cells], **I32))
    got = attend_and_check(case, 2, q=case.q(2, amp=0.3))
    assert (np64(got) > 0.85 * size).all()
    attend_and_check(case, 2, q=case.q(2, amp=0.3), window=500, sinks=3)


@pytest.mark.parametrize("dtype,bits,scale", [("f16", 8, 300.0), ("f16", 4, 8000.0), ("bf16", 8, 2.0**121), ("bf16", 4, 2.0**125)])
@pytest.mark.parametrize("d,gs", [(64, 32), (128, 128)])
@pytest.mark.parametrize("rows", [1, 5, 150])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 2)])
def test_hidden_values_past_the_type(built, dtype, bits, scale, d, gs, rows, window, sinks):
    """Scales and biases that are finite but whose top codes pass the type's largest value (arrays that append did not
    write): rows that see the position get infinities, the others never meet them, and the group's other values count."""
    case = Case([rows + 260, rows + 40], [rows, rows], dtype=dtype, bits=bits, gs=gs, d=d, hk=1, page=16)
    c = case.cache
    tab = case.table.cpu()
    top = 2**bits - 1
    for b, L in enumerate(case.lens_l):
        for i, j in enumerate(sorted({L - 1, L - 1 - rows // 2, L - rows - 52, L - rows - 10, 1, 3})):
            at = (int(tab[b, j // 16]), 0, j % 16)
            for t, x in ((c.v_scales, scale), (c.v_biases, -0.125 * scale)):
                t[at][0] = x
            codes = torch.randint(0, 2, (d,))  # small codes but for two, at other places for each position
            codes[[3 * i, 3 * i + 1]] = top
            words = K.pack(codes.numpy()[None], bits)[0].view(np.int32)
            c.v[at] = torch.from_numpy(words.copy()).cuda()
    hv = K.round_to(case.held("v"), dtype)
    assert np.isinf(hv).any() and np.isfinite(np64(c.v_scales)).all()
    # the finite values of those groups are as large as the type: their rounding is part of the tolerance
    attend_and_check(case, 2, window=window, sinks=sinks, hk_v=(case.held("k"), hv))


# ------------------------------------------------------------------ how near to 64 bits
def error_ratio(got, q, hk, hv, pos, scale, dtype, values, keys):
    """Norm of got's error over the expected one's; got and q [rows, d], pos the rows' positions."""
    see = K.visible(pos, len(hk), 0, 0)
    err, _ = K.expected_error(q, hk, hv, see, scale, dtype, values, keys)
    return ((got - K.attention(q, hk, hv, see, scale)[0]) ** 2).sum(), err


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits,gs,d", [(16, 32, 64), (16, 32, 128), (8, 32, 64), (8, 64, 64), (8, 32, 128), (8, 64, 128),
                                       (8, 128, 128), (4, 32, 64), (4, 64, 64), (4, 32, 128), (4, 64, 128), (4, 128, 128)])
@pytest.mark.parametrize("rows", [1, 7, 90])
def test_error_is_that_of_the_roundings_alone(built, dtype, bits, gs, d, rows):
    """Each path's error against 64 bits has the norm that the roundings it is to make leave, within a quarter: terms
    and result, quantised values, and keys only in chunks, where bf16 heads of 64 bring a second tile with the rest.
    The keys' channels have offsets, so that a rounded key, a tile that lacks or an offset taken off wrongly shows."""
    heads = 2 if rows == 1 else 4
    case = Case([rows + 400, rows + 211, rows + 30], [rows] * 3, dtype=dtype, bits=bits, gs=gs, d=d, hk=2, page=16)
    c, cells = case.cache, case.n_pages * 16
    g = torch.Generator("cuda").manual_seed(11)
    ch = 12.0 * (torch.randint(0, 2, (2, d), generator=g, device="cuda") - 0.5)
    k = (torch.randn(cells, 2, d, generator=g, device="cuda") * 0.5 + ch).to(T[dtype])
    v = torch.randn(cells, 2, d, generator=g, device="cuda").to(T[dtype])
    c.append(k, v, torch.arange(case.n_pages, **I32)[None], torch.tensor([cells], **I32), torch.tensor([0, cells], **I32))
    q = case.q(heads)
    got, qn = np64(c.attend(q, case.table, case.lens, case.start)), np64(q)
    hk, hv = case.held("k"), case.held("v")
    keys = bits < 16 and rows == 90 and not (dtype == "bf16" and d == 64)
    total = expected = 0.0
    for b, (L, n) in enumerate(zip(case.lens_l, case.rows_l)):
        at = slice(case.start_l[b], case.start_l[b + 1])
        for h in range(heads):
            a, e = error_ratio(got[at, h], qn[at, h], case.seq(hk, b, h * 2 // heads), case.seq(hv, b, h * 2 // heads),
                               np.arange(L - n, L), d**-0.5, dtype, bits < 16, keys)
            total, expected = total + a, expected + e
    ratio = np.sqrt(total / expected)
    assert 0.6 < ratio < 1.25, ratio


def test_chunk_terms_are_the_exponentials(built):
    """One-hot values make a row's result its terms: every column of a block, terms over 17 powers of two and up to 2^7
    above the first block's largest, on the exponential unit and the FMA pipe alike."""
    L, rows, d = 128 * 5, 20, 64
    case = Case([L], [rows], dtype="f16", bits=16, d=d, hk=1, page=16)
    c = case.cache
    for half in (0, 1):  # columns 0..63, then 64..127 of the second block
        rng = np.random.default_rng(half)
        a = np.full(L, -60.0)  # terms of exp(-60) and less
        a[0] = 0.0
        first = 128 + 64 * half
        a[first:first + 64] = K.round_to(rng.uniform(-7.0, 4.8, 64), "f16")
        k, v = torch.zeros(L, 1, d), torch.zeros(L, 1, d)
        k[:, 0, 0] = torch.from_numpy(a)
        v[first + torch.arange(64), 0, torch.arange(64)] = 1024.0
        c.append(k.half().cuda(), v.half().cuda(), case.table, case.lens, torch.tensor([0, L], **I32))
        amp = K.round_to(rng.uniform(0.5, 1.0, rows), "f16")
        q = torch.zeros(rows, 1, d)
        q[:, 0, 0] = torch.from_numpy(amp)
        got = np64(c.attend(q.half().cuda(), case.table, case.lens, case.start, scale=1.0))[:, 0]
        e = np.exp(amp[:, None] * a[None, first:first + 64])
        want = 1024.0 * e / (1.0 + e.sum(1, keepdims=True))
        # the term and the result rounded to f16 (the smallest result is 2^-14 and more), the exponential's own error
        # under 2^-18, fp32 scores of up to 7: 2^-20
        assert want.min() > 2.0**-14 and np.log2(e.max()) > 5
        assert (np.abs(got / want - 1.0) <= 2.0**-11 * 2 + 2.0**-17).all(), np.abs(got / want - 1.0).max()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_prompt_chunks_and_tokens_each_near_64_bits(built, dtype, bits):
    """A prompt in one chunk, in uneven chunks and token by token: each within a quarter of its roundings' error."""
    n, hk, heads, d = 300, 2, 4, 64
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.randn(n, hk, d, generator=g, device="cuda").to(T[dtype]) for _ in range(2))
    q = torch.randn(n, heads, d, generator=g, device="cuda").to(T[dtype])
    tab = torch.randperm(19, generator=g, device="cuda").to(torch.int32)[None]
    for cuts in ([0, n], [0, 1, 20, 22, 150, n], list(range(n + 1))):
        c = PagedKVCache(19, 16, hk, d, bits=bits, group_size=32, dtype=T[dtype])
        parts = []
        for a, b in zip(cuts, cuts[1:]):
            lens, st = torch.tensor([b], **I32), torch.tensor([0, b - a], **I32)
            c.append(k[a:b], v[a:b], tab, lens, st)
            parts.append(c.attend(q[a:b], tab, lens, st))
        c.check()
        got, qn = np64(torch.cat(parts)), np64(q)
        total = expected = 0.0
        for h in range(heads):
            held = []
            for x in (k, v):
                x = np64(x)[:, h // 2]
                held.append(K.dequantise(*K.quantise(x, bits, 32, dtype), 32) if bits < 16 else x)
            # f16 keys of chunks are rounded; by the unit scores here that is least for all of them
            e = error_ratio(got[:, h], qn[:, h], *held, np.arange(n), d**-0.5, dtype, bits < 16,
                            bits < 16 and dtype == "f16" and len(cuts) < n)
            total, expected = total + e[0], expected + e[1]
        assert 0.6 < np.sqrt(total / expected) < 1.25, (len(cuts), np.sqrt(total / expected))
