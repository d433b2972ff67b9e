"""Paged key/value cache: the attention state next to the routed-MoE layer.

The cache is held the way the arena holds experts: stacked arrays indexed by a
page id, head rows in the affine format of the expert rows (codes LSB first in
32-bit words, one scale and bias per group in the activation dtype), or kept
in 16 bits.  :class:`PagedKVCache` binds the arrays to the kernels of
``liblmoe.so`` (include/lmoe.h, ``lmoe_kv_*`` and ``lmoe_paged_attention``):

* ``append`` writes new tokens' keys and values, quantising them on the way;
* ``read`` gives them back;
* ``attend`` lets new tokens (a prompt's chunk, or one token of each sequence)
  attend over what their sequences hold, with an optional sliding window and
  first tokens that stay visible.

Which page holds what is the caller's: a call names its sequences by their
page tables and lengths.  Like the layer calls, the calls enqueue on the
current stream of the cache's device and do not wait for it; a page id or
length the kernels could not follow is reported by :meth:`PagedKVCache.check`.
The reference has no counterpart (its cache comes from oMLX with the dense
backbone, dsv4_engine.py:22-42).
"""

from __future__ import annotations

import contextlib
import ctypes
import math

import torch

from . import _lib
from ._lib import check, lmoe
from .ops import _ACT, Workspace, _need_cuda, _ptr


_HERE = contextlib.nullcontext()


def _on(device: torch.device):
    """Context that makes ``device`` current (the C calls launch there)."""
    return _HERE if torch._C._cuda_getDevice() == device.index else torch.cuda.device(device)


class PagedKVCache:
    """Keys and values of ``n_pages`` pages of ``page_size`` tokens.

    ``bits`` 16 keeps rows in ``dtype`` (bf16 or f16): ``k``, ``v`` are
    [n_pages, kv_heads, page_size, head_dim].  ``bits`` 8 or 4 holds them
    quantised: ``k``, ``v`` int32 [n_pages, kv_heads, page_size, head_dim *
    bits / 32] and ``k_scales``, ``k_biases``, ``v_scales``, ``v_biases``
    ``dtype`` [n_pages, kv_heads, page_size, head_dim / group_size].

    head_dim is 64 or 128, page_size a multiple of 16, group_size 32, 64 or
    128.  Pages start zeroed; what a page holds behind a sequence's length is
    never looked at, so a page needs no clearing before another sequence takes
    it.

    The calls below share their arguments: ``page_table`` int32 [n_seqs,
    width] (position p of sequence b is slot ``p % page_size`` of page
    ``page_table[b, p // page_size]``), ``lens`` int32 [n_seqs] the
    sequences' lengths with the rows of the call, and ``row_start`` int32
    [n_seqs + 1]: rows ``row_start[b]`` to ``row_start[b + 1] - 1`` are
    sequence b's last positions.  Without ``row_start`` each sequence has one
    row.  Rows in front of ``row_start[0]`` and from ``row_start[n_seqs]`` on
    (padding of a captured batch) belong to no sequence: they are left as they
    were.
    The three arrays are device arrays, so a captured call replays with the
    values they hold then.
    """

    def __init__(self, n_pages: int, page_size: int, kv_heads: int, head_dim: int, *, bits: int = 16,
                 group_size: int = 64, dtype: torch.dtype = torch.bfloat16, device=None):
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if bits not in (16, 8, 4) or dtype not in _ACT:
            raise ValueError("bits must be 16, 8 or 4 and dtype bf16 or f16")
        if min(n_pages, page_size, kv_heads, head_dim) < 1 or (bits < 16 and (group_size < 1 or head_dim % group_size)):
            raise ValueError("cache sizes must be positive and head_dim a multiple of group_size")
        lead = (n_pages, kv_heads, page_size)

        def zeros(last, t):
            return torch.zeros((*lead, last), dtype=t, device=dev)

        if bits == 16:
            kv = [zeros(head_dim, dtype) for _ in range(2)]
            self._bind(kv[0], kv[1], None, None, None, None, 16, group_size)
        else:
            kv = [zeros(head_dim * bits // 32, torch.int32) for _ in range(2)]
            sb = [zeros(head_dim // group_size, dtype) for _ in range(4)]
            self._bind(*kv, *sb, bits, group_size)

    @classmethod
    def from_arrays(cls, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor | None = None,
                    k_biases: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                    v_biases: torch.Tensor | None = None, *, bits: int = 16, group_size: int = 64) -> "PagedKVCache":
        """The cache over arrays that the caller holds (see the class for their shapes)."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scales, k_biases, v_scales, v_biases, bits, group_size)
        return self

    def _bind(self, k, v, k_scales, k_biases, v_scales, v_biases, bits, group_size) -> None:
        sb = (k_scales, k_biases, v_scales, v_biases)
        quant = bits != 16
        if bits not in (16, 8, 4):
            raise ValueError("bits must be 16, 8 or 4")
        if quant and any(t is None for t in sb):
            raise ValueError("a quantised cache needs scales and biases")
        if not quant:
            sb = (None,) * 4
        arrays = [t for t in (k, v, *sb) if t is not None]
        _need_cuda(*arrays)
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("k and v must be [n_pages, kv_heads, page_size, row] of one type")
        if any(t.device != k.device for t in arrays):
            raise ValueError("cache arrays must be on one device")
        if any(not t.is_contiguous() or t.data_ptr() % 16 for t in arrays):
            raise ValueError("cache arrays must be contiguous and 16-byte aligned")
        self.bits, self.group_size = int(bits), int(group_size)
        if quant:
            if k.dtype not in (torch.int32, torch.uint32):
                raise ValueError("quantised k and v hold 32-bit words")
            self.dtype = sb[0].dtype
            self.head_dim = int(k.shape[3]) * 32 // bits
            want = (*k.shape[:3], self.head_dim // group_size)
            if any(tuple(t.shape) != want or t.dtype != self.dtype for t in sb):
                raise ValueError(f"scales and biases must be {want} of one type")
        else:
            self.dtype, self.head_dim = k.dtype, int(k.shape[3])
        if self.dtype not in _ACT:
            raise ValueError(f"unsupported cache dtype {self.dtype}")
        if self.head_dim not in (64, 128) or k.shape[2] % 16 or (quant and (group_size not in (32, 64, 128)
                                                                             or self.head_dim % group_size)):
            raise _lib.LmoeError(_lib.LMOE_EUNSUPPORTED, "cache geometry")
        if k.numel() == 0:
            raise ValueError("the cache needs at least one page")
        self.k, self.v = k, v
        self.k_scales, self.k_biases, self.v_scales, self.v_biases = sb
        self.n_pages, self.kv_heads, self.page_size = (int(n) for n in k.shape[:3])
        self.device = k.device
        self.desc = _lib.KVCache(k.data_ptr(), v.data_ptr(), *(_ptr(t) for t in sb), self.n_pages, self.page_size,
                                 self.kv_heads, self.head_dim, _ACT[self.dtype], self.bits, self.group_size)
        self._desc_ref = ctypes.byref(self.desc)
        # status word of the kernels; they only ever raise it, so calls on any stream may share it
        with _on(self.device):
            self.ws = Workspace(self.device).ensure(256)
        self._scratch_bytes: dict[tuple, int] = {}

    def check(self) -> None:
        """Wait for the current stream and raise if a kernel met a page id, length or row start out of range, or gave up
        a wait.  Calls on other streams are covered once that stream waits for them."""
        with _on(self.device):
            self.ws.check()

    # ------------------------------------------------------------ arguments
    def _rows(self, page_table: torch.Tensor, lens: torch.Tensor, row_start: torch.Tensor | None,
              n_rows: int) -> _lib.KVRows:
        i32 = torch.int32
        B = lens.shape[0] if lens.dim() == 1 else -1
        if page_table.dim() != 2 or page_table.shape[0] != B:
            raise ValueError("page_table must be [n_seqs, width] and lens [n_seqs]")
        if page_table.dtype is not i32 or lens.dtype is not i32:
            raise ValueError("page_table and lens must be int32")
        dev = self.device
        if page_table.device != dev or lens.device != dev:
            raise ValueError(f"page_table and lens must be on {dev}")
        width = page_table.shape[1]
        stride = page_table.stride(0) if B > 1 else width
        if (width > 1 and page_table.stride(1) != 1) or stride < width or not lens.is_contiguous():
            raise ValueError("page_table rows and lens must be contiguous")
        if row_start is None:
            if n_rows != B:
                raise ValueError(f"{n_rows} rows for {B} sequences: give row_start")
            start = None
        else:
            if row_start.dtype is not i32 or row_start.dim() != 1 or row_start.shape[0] != B + 1 \
                    or row_start.device != dev or not row_start.is_contiguous():
                raise ValueError(f"row_start must be contiguous int32 [{B + 1}] on {dev}")
            start = row_start.data_ptr()
        return _lib.KVRows(page_table.data_ptr(), stride, width, B, lens.data_ptr(), start, n_rows)

    def _heads(self, x: torch.Tensor, what: str, heads: int | None) -> torch.Tensor:
        """x as rows the kernels can read: [rows, heads, head_dim], any token and head strides of whole 16 bytes."""
        if x.dim() != 3 or x.shape[2] != self.head_dim or (heads is not None and x.shape[1] != heads):
            raise ValueError(f"{what} must be [rows, {heads or 'heads'}, {self.head_dim}], got {tuple(x.shape)}")
        if x.dtype is not self.dtype:
            raise ValueError(f"{what} must be {self.dtype}, got {x.dtype}")
        if x.device != self.device:
            raise ValueError(f"{what} must be on {self.device}")
        if x.stride(2) != 1 or x.stride(0) % 8 or x.stride(1) % 8 or x.data_ptr() % 16:
            x = x.contiguous()
            if x.data_ptr() % 16:  # a contiguous view that starts between two 16-byte lines
                x = x.clone()
            x = x.view(-1).view(x.shape)  # a dimension of size one may have kept any stride
        return x

    def _out(self, out: torch.Tensor, shape: tuple, what: str) -> torch.Tensor:
        if tuple(out.shape) != tuple(shape) or out.dtype is not self.dtype or out.device != self.device \
                or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError(f"{what} must be contiguous {tuple(shape)} {self.dtype} on {self.device}, 16-byte aligned")
        return out

    def _stream(self) -> int:
        return torch._C._cuda_getCurrentRawStream(self.device.index)

    # ------------------------------------------------------------ calls
    def append(self, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor,
               row_start: torch.Tensor | None = None) -> None:
        """Write the rows' keys and values ([rows, kv_heads, head_dim], any
        strides) into their sequences' last positions.  A quantised cache
        keeps, for each group, ``bias`` = its minimum, ``scale`` = its range
        over ``2^bits - 1`` rounded to ``dtype``, and the nearest codes; a
        group with an infinity or a NaN reads back as NaN.  No two rows of a
        call may share a place: pages that several sequences share (a common
        prefix) are for reading."""
        _need_cuda(k, v)
        k, v = self._heads(k, "k", self.kv_heads), self._heads(v, "v", self.kv_heads)
        if v.shape != k.shape:
            raise ValueError("k and v must have the same rows")
        rows = self._rows(page_table, lens, row_start, k.shape[0])
        with _on(self.device):
            check(lmoe().lmoe_kv_append(self._desc_ref, ctypes.byref(rows), k.data_ptr(), k.stride(0), k.stride(1),
                                        v.data_ptr(), v.stride(0), v.stride(1), self.ws.ptr(), self._stream()),
                  "lmoe_kv_append")

    def read(self, page_table: torch.Tensor, lens: torch.Tensor, row_start: torch.Tensor | None = None, *,
             rows: int | None = None, out: tuple[torch.Tensor, torch.Tensor] | None = None):
        """(k, v) [rows, kv_heads, head_dim] of the sequences' last positions
        as the cache holds them.  ``rows`` is the number of rows to return
        (``row_start[n_seqs]``; one for each sequence without ``row_start``);
        a row in front of its sequence's first position is zero."""
        if out is not None:
            if rows is not None and out[0].shape[0] != rows:
                raise ValueError("out must hold `rows` rows")
            rows = int(out[0].shape[0])
        elif rows is None:
            if row_start is not None:
                raise ValueError("give rows (or out) with row_start: it is on the device")
            rows = int(lens.shape[0])
        shape = (rows, self.kv_heads, self.head_dim)
        if out is None:
            k, v = (torch.empty(shape, dtype=self.dtype, device=self.device) for _ in range(2))
        else:
            k, v = self._out(out[0], shape, "out[0]"), self._out(out[1], shape, "out[1]")
        r = self._rows(page_table, lens, row_start, rows)
        with _on(self.device):
            check(lmoe().lmoe_kv_read(self._desc_ref, ctypes.byref(r), k.data_ptr(), v.data_ptr(), self.ws.ptr(),
                                      self._stream()), "lmoe_kv_read")
        return k, v

    def attend(self, q: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor,
               row_start: torch.Tensor | None = None, *, scale: float | None = None, window: int = 0,
               sinks: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of q [rows, heads, head_dim] over the rows' sequences, up
        to and with each row's own position (append the rows first).  heads is
        a multiple of kv_heads; ``scale`` is head_dim ** -0.5 by default.  With
        ``window`` > 0 a row sees its own and the ``window - 1`` positions
        before it, and the sequence's first ``sinks`` positions; table entries
        of pages that no row sees a position of may hold anything.  A row that
        sees nothing is zero.  ``out`` must not share memory with q; rows of
        no sequence are left as ``out`` has them (undefined without it)."""
        _need_cuda(q)
        q = self._heads(q, "q", None)
        n, heads = int(q.shape[0]), int(q.shape[1])
        if heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads are no multiple of {self.kv_heads} key/value heads")
        if scale is None:
            scale = 1.0 / math.sqrt(self.head_dim)
        if not (math.isfinite(scale) and scale >= 0.0) or sinks < 0:
            raise ValueError("scale must be finite and not negative, sinks not negative")
        if out is None:
            out = torch.empty((n, heads, self.head_dim), dtype=self.dtype, device=self.device)
        else:
            out = self._out(out, q.shape, "out")
            if out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
                a, b = out.data_ptr(), q.data_ptr()
                last = sum((s - 1) * st for s, st in zip(q.shape, q.stride()))
                if n and a <= b + 2 * last and b < a + 2 * out.numel():
                    raise ValueError("out must not share memory with q")
        r = self._rows(page_table, lens, row_start, n)
        key = (r.n_seqs, n, heads)
        need = self._scratch_bytes.get(key)
        lib = lmoe()
        with _on(self.device):
            if need is None:
                need = int(lib.lmoe_paged_attention_scratch(self._desc_ref, ctypes.byref(r), heads))
                if len(self._scratch_bytes) > 4096:
                    self._scratch_bytes.clear()
                self._scratch_bytes[key] = need
            # from the caching allocator, call by call: a call on another
            # stream or in another captured graph has its own
            scratch = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            check(lib.lmoe_paged_attention(self._desc_ref, ctypes.byref(r), heads, q.data_ptr(), q.stride(0),
                                           q.stride(1), scale, min(max(int(window), 0), 2**31 - 1),
                                           min(int(sinks), 2**31 - 1), out.data_ptr(), _ptr(scratch), need,
                                           self.ws.ptr(), self._stream()),
                  "lmoe_paged_attention")
        return out
