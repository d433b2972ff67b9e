"""The paged key/value cache's operators: their cases, their plain forms and what they cannot do without.

Two groups of cases.  ``cache_*``: new tokens are written into the pages (quantised in affine groups, or kept in 16
bits) and the rows just written are read back.  ``attn_*``: new tokens attend over the pages their sequences hold.

``run`` with ``own`` false computes the plain forms with elementary torch operations; with ``own`` true it makes the
calls of :class:`locali_b200.kv_cache.PagedKVCache`.
"""

import math
import random

import torch

own = False

_T = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ cases
def _cache(name, dtype, bits, group, page, kv_heads, dim, seqs, rows, past, shape):
    """Write ``rows`` new tokens (the longest share of one sequence) after up to ``past`` earlier ones, read them back."""
    return {"name": name, "op": "cache", "dtype": dtype, "bits": bits, "group": group, "page": page,
            "kv_heads": kv_heads, "heads": kv_heads, "dim": dim, "seqs": seqs, "rows": rows, "past": past,
            "window": 0, "sinks": 0, "shape": shape}


def _attn(name, dtype, bits, group, page, heads, kv_heads, dim, seqs, rows, past, window, sinks, shape):
    """``seqs`` sequences of up to ``rows`` new tokens each after up to ``past`` cached ones (the new ones are cached too)."""
    return {"name": name, "op": "attn", "dtype": dtype, "bits": bits, "group": group, "page": page,
            "kv_heads": kv_heads, "heads": heads, "dim": dim, "seqs": seqs, "rows": rows, "past": past,
            "window": window, "sinks": sinks, "shape": shape}


def listed():
    return [
        # one decode step of a small batch: latency alone
        _cache("cache_step", "bf16", 8, 64, 64, 8, 128, 16, 1, 4000, 1),
        # prompts of a batch, 8-bit cache
        _cache("cache_prompts_8bit", "bf16", 8, 64, 64, 8, 128, 5, 8192, 0, 2),
        # prompts on top of earlier turns, 4-bit cache, odd head count and page
        _cache("cache_turns_4bit", "f16", 4, 32, 48, 5, 64, 7, 3000, 900, 3),
        # one user's next token after a short conversation: latency
        _attn("attn_one_token", "bf16", 16, 64, 64, 32, 8, 128, 1, 1, 1000, 0, 0, 4),
        # a serving batch's decode step over an 8-bit cache, ragged lengths
        _attn("attn_batch_8bit", "bf16", 8, 64, 64, 32, 8, 128, 64, 1, 8000, 0, 0, 5),
        # long documents, 4-bit cache
        _attn("attn_long_4bit", "bf16", 4, 64, 128, 32, 8, 128, 4, 1, 131000, 0, 0, 6),
        # a large batch of windowed decode steps with 4 first tokens kept
        _attn("attn_window_step", "f16", 16, 64, 16, 28, 4, 128, 128, 1, 20000, 1024, 4, 7),
        # a few drafted tokens of each sequence verified at once
        _attn("attn_verify_8bit", "bf16", 8, 32, 32, 32, 8, 128, 24, 6, 6000, 0, 0, 8),
        # a whole prompt
        _attn("attn_prompt", "bf16", 16, 64, 64, 32, 8, 128, 1, 4096, 0, 0, 0, 9),
        # the next chunk of a long prompt over an 8-bit cache
        _attn("attn_chunk_8bit", "bf16", 8, 64, 64, 32, 8, 128, 1, 2048, 30000, 0, 0, 10),
        # chunks of several prompts, sliding window with first tokens, small heads
        _attn("attn_chunk_window", "f16", 4, 32, 80, 24, 6, 64, 3, 2500, 3000, 700, 5, 11),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["bf16", "f16"])
    bits = rng.choice([16, 8, 4])
    dim = rng.choice([64, 128])
    group = rng.choice([32, 64] if dim == 64 else [32, 64, 128])
    page = 16 * rng.choice([1, 2, 3, 4, 5, 8, 16])
    kv = rng.choice([1, 2, 3, 4, 6, 8])
    shape = rng.randrange(1 << 30)
    kind = rng.randrange(4)
    if kind == 0:
        seqs, past = _log(rng, 1, 32), _log(rng, 1, 5000)
        rows = 1 if rng.random() < 0.3 else _log(rng, 2, max(2, 30000 // seqs))
        return _cache("draw", dtype, bits, group, page, kv, dim, seqs, rows, past, shape)
    heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    window, sinks = (_log(rng, 16, 4000), rng.choice([0, 1, 4, 17])) if rng.random() < 0.4 else (0, 0)
    if kind == 1:  # single tokens
        seqs = _log(rng, 1, 128)
        rows, past = 1, _log(rng, 10, min(100000, 400000 // seqs))
    elif kind == 2:  # a few tokens each
        seqs = _log(rng, 1, 32)
        rows, past = rng.randrange(2, 17), _log(rng, 10, min(30000, 100000 // seqs))
    else:  # chunks
        seqs = rng.randrange(1, 5)
        rows = _log(rng, 17, 3000)
        past = _log(rng, 1, max(2, min(30000, 600_000_000 // (seqs * rows * heads))))
    return _attn("draw", dtype, bits, group, page, heads, kv, dim, seqs, rows, past, window, sinks, shape)


def _lengths(case):
    """New rows and total length of every sequence: part of the case, not of the seed."""
    r = random.Random(case["shape"])
    B, n, past = case["seqs"], case["rows"], case["past"]
    # the first sequence is the longest: the plain form pads to it
    rows = [n if i == 0 or n == 1 else max(1, int(n * r.uniform(0.4, 1.0))) for i in range(B)]
    earlier = [past if i == 0 else int(past * r.uniform(0.1, 1.0)) for i in range(B)]
    return rows, [a + b for a, b in zip(earlier, rows)]


def _visible(case):
    """(visible key/query pairs of one head, key rows that any query sees) over all sequences."""
    W, S = case["window"], case["sinks"]
    pairs = keys = 0
    for n, L in zip(*_lengths(case)):
        first = L - n
        if W <= 0:
            pairs += n * (first + 1) + n * (n - 1) // 2
            keys += L
            continue
        for p in range(first, L):
            low = max(0, p - W + 1)
            pairs += p + 1 - low + min(S, low)
        low = max(0, first - W + 1)
        keys += L - low + min(S, low)
    return pairs, keys


def work(case):
    rows, lens = _lengths(case)
    n, d, hk = sum(rows), case["dim"], case["kv_heads"]
    held = 2 * hk * (d * case["bits"] // 8 + (4 * (d // case["group"]) if case["bits"] < 16 else 0))
    tables = 4 * sum(-(-L // case["page"]) for L in lens) + 12 * case["seqs"]
    if case["op"] == "cache":
        # the new rows in and the values out, and what the cache holds of them written and read once
        return {"bytes": n * (2 * 2 * hk * d * 2 + 2 * held) + tables, "flops": 8 * 2 * n * hk * d}
    pairs, keys = _visible(case)
    return {"bytes": keys * held + 2 * 2 * n * case["heads"] * d + tables, "flops": 4 * d * case["heads"] * pairs}


# ------------------------------------------------------------------ inputs
def _quantise(x, bits, group):
    """Codes (int32), scales and biases of the last dimension's groups (see PagedKVCache)."""
    n = (1 << bits) - 1
    g = x.unflatten(-1, (-1, group)).double()
    lo, hi = g.amin(-1), g.amax(-1)
    # the scale is the quotient rounded to 32 bits and then to the type; one step lower where the top code would overflow it
    s = ((hi - lo) / n).float().to(x.dtype)
    over = s.double() * n + lo > torch.finfo(x.dtype).max
    s = torch.where(over, (s.view(torch.int16) - over.to(torch.int16)).view(x.dtype), s)
    sd = s.double().unsqueeze(-1)
    q = torch.where(sd > 0, (g - lo.unsqueeze(-1)) / torch.where(sd > 0, sd, 1.0), 0.0)
    return q.round().clamp(0, n).int().flatten(-2), s, lo.to(x.dtype)


def _pack(codes, bits):
    """uint32 words (held as int32), codes LSB first."""
    per = 32 // bits
    c = codes.unflatten(-1, (-1, per)).long() << (bits * torch.arange(per, device=codes.device))
    w = c.sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _unpack(words, bits):
    per = 32 // bits
    c = words.unsqueeze(-1) >> (bits * torch.arange(per, device=words.device, dtype=torch.int32))
    return (c & ((1 << bits) - 1)).flatten(-2)


def prepare(case, seed):
    dev = "cuda"
    T, bits, group, page = _T[case["dtype"]], case["bits"], case["group"], case["page"]
    d, hk, B = case["dim"], case["kv_heads"], case["seqs"]
    rows, lens = _lengths(case)
    gen = torch.Generator(dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    width = max(-(-L // page) for L in lens)
    used = sum(-(-L // page) for L in lens)
    n_pages = used + 3
    # page tables: pages in no order, entries behind a sequence's last page left at -1
    perm = torch.randperm(n_pages, generator=gen, device=dev)[:used].int().cpu()
    table, at = torch.full((B, width), -1, dtype=torch.int32), 0
    for b, L in enumerate(lens):
        k = -(-L // page)
        table[b, :k] = perm[at:at + k]
        at += k
    st = {"case": dict(case), "table": table.to(dev), "lens": torch.tensor(lens, dtype=torch.int32, device=dev),
          "total": sum(rows), "row_start": None}
    if case["rows"] > 1:
        st["row_start"] = torch.tensor([sum(rows[:i]) for i in range(B + 1)], dtype=torch.int32, device=dev)
    # keys: channels of different scale and offset, as trained projections give them; values: unit scale
    ch, off = 0.5 + 0.5 * rnd(hk, 1, d).abs(), 0.7 * rnd(hk, 1, d)
    if case["op"] == "cache":
        st["new_k"] = (rnd(sum(rows), hk, d) * ch[:, 0] + off[:, 0]).to(T)
        st["new_v"] = rnd(sum(rows), hk, d).to(T)
        words = d * bits // 32
        for kv in "kv":
            if bits == 16:
                st[kv] = torch.zeros(n_pages, hk, page, d, dtype=T, device=dev)
            else:
                st[kv] = torch.zeros(n_pages, hk, page, words, dtype=torch.int32, device=dev)
                st[kv + "_scales"] = torch.zeros(n_pages, hk, page, d // group, dtype=T, device=dev)
                st[kv + "_biases"] = torch.zeros(n_pages, hk, page, d // group, dtype=T, device=dev)
        return st
    for kv in "kv":
        x = rnd(n_pages, hk, page, d)
        x = (x * ch + off if kv == "k" else x).to(T)
        if bits == 16:
            st[kv] = x
        else:
            parts = [_quantise(c, bits, group) for c in x.split(max(1, (1 << 25) // (hk * page * d)))]
            st[kv] = torch.cat([_pack(p[0], bits) for p in parts])
            st[kv + "_scales"] = torch.cat([p[1] for p in parts])
            st[kv + "_biases"] = torch.cat([p[2] for p in parts])
    st["q"] = (rnd(sum(rows), case["heads"], d) * 1.5).to(T)
    return st


# ------------------------------------------------------------------ one pass
def _handle(st):
    """The cache handle that a program keeps beside its arrays."""
    if "handle" not in st:
        from locali_b200.kv_cache import PagedKVCache

        st["handle"] = PagedKVCache.from_arrays(st["k"], st["v"], st.get("k_scales"), st.get("k_biases"),
                                                st.get("v_scales"), st.get("v_biases"), bits=st["case"]["bits"],
                                                group_size=st["case"]["group"])
    return st["handle"]


def _new_rows(st):
    """Sequence and position of every new row."""
    B = st["lens"].numel()
    start = st["row_start"]
    if start is None:
        start = torch.arange(B + 1, device=st["lens"].device, dtype=torch.int32)
    i = torch.arange(st["total"], device=start.device)
    b = torch.searchsorted(start[1:].long(), i, right=True)
    return b, st["lens"].long()[b] - start.long()[b + 1] + i, start.long()


def _values(st, kv, page, slot=None):
    """What the pages stand for, in 32 bits: whole pages, or one row of each."""
    at = (lambda a: a[page]) if slot is None else (lambda a: a[page, :, slot])
    c = st["case"]
    if c["bits"] == 16:
        return at(st[kv]).float()
    codes = _unpack(at(st[kv]), c["bits"]).float().unflatten(-1, (-1, c["group"]))
    return (codes * at(st[kv + "_scales"]).float().unsqueeze(-1) + at(st[kv + "_biases"]).float().unsqueeze(-1)).flatten(-2)


def _plain_cache(st):
    c = st["case"]
    b, pos, _ = _new_rows(st)
    page, slot = st["table"][b, pos // c["page"]].long(), pos % c["page"]
    out = []
    for kv in "kv":
        x = st["new_" + kv]
        if c["bits"] == 16:
            st[kv][page, :, slot] = x
        else:
            codes, s, lo = _quantise(x, c["bits"], c["group"])
            st[kv][page, :, slot] = _pack(codes, c["bits"])
            st[kv + "_scales"][page, :, slot] = s
            st[kv + "_biases"][page, :, slot] = lo
        out.append(_values(st, kv, page, slot).to(x.dtype))
    return out


def _plain_attention(st):
    c, q = st["case"], st["q"]
    d, hk, G = c["dim"], c["kv_heads"], c["heads"] // c["kv_heads"]
    b, pos, start = _new_rows(st)
    B, n = st["lens"].numel(), c["rows"]
    # every sequence's rows and keys, padded to the longest
    local = torch.arange(st["total"], device=q.device) - start[b]
    qp = torch.zeros(B, n, hk, G, d, device=q.device)
    qp[b, local] = q.float().unflatten(1, (hk, G))
    at = torch.full((B, n), -1, device=q.device, dtype=torch.long)
    at[b, local] = pos
    table = st["table"].clamp(min=0).long()
    k = _values(st, "k", table).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [B, hk, keys, d]
    j = torch.arange(k.shape[2], device=q.device)
    see = j <= at.unsqueeze(-1)
    if c["window"] > 0:
        see &= (j > at.unsqueeze(-1) - c["window"]) | (j < c["sinks"])
    qp = qp.permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, hk, G * n, d]
    s = qp @ k.transpose(2, 3) * (1.0 / math.sqrt(d))
    del k
    hide = ~see.unsqueeze(1).unsqueeze(1)
    s.unflatten(2, (G, n)).masked_fill_(hide, -math.inf)
    s -= s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    v = _values(st, "v", table).permute(0, 2, 1, 3, 4).flatten(2, 3)
    o = s @ v / torch.where(total > 0, total, 1.0)
    return o.unflatten(2, (G, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)[b, local].to(q.dtype)


def run(state):
    st = state
    if own:
        cache = _handle(st)
        if st["case"]["op"] == "cache":
            cache.append(st["new_k"], st["new_v"], st["table"], st["lens"], st["row_start"])
            return list(cache.read(st["table"], st["lens"], st["row_start"], rows=st["total"]))
        return cache.attend(st["q"], st["table"], st["lens"], st["row_start"], window=st["case"]["window"],
                            sinks=st["case"]["sinks"])
    return _plain_cache(st) if st["case"]["op"] == "cache" else _plain_attention(st)


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definition in 64 bits: sequence by sequence and head by head."""
    st = prepare(case, seed)
    rows, lens = _lengths(case)
    bits, gs, page, d = case["bits"], case["group"], case["page"], case["dim"]
    if case["op"] == "cache":
        out = []
        for x in (st["new_k"], st["new_v"]):
            if bits == 16:
                out.append(x.double())
                continue
            n = 2 ** bits - 1
            top = torch.finfo(x.dtype).max
            g = x.double().reshape(*x.shape[:-1], d // gs, gs)
            b = g.min(-1, keepdim=True).values
            # the held scale is a value of the type, as the bias is
            s = ((g.max(-1, keepdim=True).values - b) / n).float().to(x.dtype)
            low = (s.view(torch.int16) - 1).view(x.dtype).double()
            s = torch.where(s.double() * n + b > top, low, s.double())
            code = torch.nan_to_num(torch.round((g - b) / s), nan=0.0).clamp(0, n)
            out.append((code * s + b).reshape(x.shape))
        return out
    G, W, S = case["heads"] // case["kv_heads"], case["window"], case["sinks"]
    out = torch.zeros(sum(rows), case["heads"], d, dtype=torch.float64, device="cuda")
    word_at = torch.arange(d, device="cuda") * bits // 32
    shift = torch.arange(d, device="cuda") * bits % 32
    group_at = torch.arange(d, device="cuda") // gs
    first = 0
    for b, (n, L) in enumerate(zip(rows, lens)):
        p = torch.arange(L - n, L, device="cuda").unsqueeze(1)
        j = torch.arange(L, device="cuda")
        hidden = j > p
        if W > 0:
            hidden |= (j <= p - W) & (j >= S)
        pg, sl = st["table"][b].long()[j // page], j % page
        for h in range(case["kv_heads"]):
            held = []
            for kv in "kv":
                if bits == 16:
                    held.append(st[kv][pg, h, sl].double())
                else:
                    code = ((st[kv][pg, h, sl].long()[:, word_at] >> shift) & (2 ** bits - 1)).double()
                    held.append(code * st[kv + "_scales"][pg, h, sl].double()[:, group_at]
                                + st[kv + "_biases"][pg, h, sl].double()[:, group_at])
            for g in range(h * G, h * G + G):
                z = st["q"][first:first + n, g].double() @ held[0].T / math.sqrt(d)
                z = z.masked_fill(hidden, -math.inf)
                out[first:first + n, g] = torch.softmax(z, -1) @ held[1]
        first += n
    return out
