"""A paged 8-bit key/value cache, for models that attend to tokens of earlier calls: video generated chunk by chunk,
text token by token.  ``ops.kv_append`` writes into it, ``ops.kv_attention`` reads it.

``KVCache`` is the memory of one attention layer, ``KVPlan`` the batch: which rows of the packed inputs belong to which
sequence, how many tokens each has, and where its pages are.  The plan's three arrays are int32 tensors on the device
that the caller goes on owning and may rewrite in place between calls (also between replays of a captured graph); the
two numbers ``max_rows`` and ``max_kv_len`` bound what they may come to hold.  One plan serves every layer of a model.

The reference keeps no keys or values between calls; there is no counterpart in it.
"""
import ctypes
from typing import Optional

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu
HEAD_DIM = 128
PAGE_SIZES = (16, 32, 64, 128)
EXPONENTS = (-48, 48)  # of a block's scale


class _Fixed:
    """Attributes that are set once: the library is handed the addresses and sizes that they had then."""

    def __setattr__(self, name, value):
        if "_ref" in self.__dict__:
            raise AttributeError("%s.%s is fixed; make a new one" % (type(self).__name__, name))
        super().__setattr__(name, value)


def _apart(shape, strides, inner: int) -> bool:
    """Whether blocks of `inner` elements at these (page, head) strides lie apart."""
    (p, h), (sp, sh) = shape, strides
    return (p == 1 or sp >= inner) and (h == 1 or sh >= inner) \
        and (p == 1 or h == 1 or sp >= (h - 1) * sh + inner or sh >= (p - 1) * sp + inner)


class KVCache(_Fixed):
    """Codes ``k``, ``v``: (pages, heads, page_size, 128) e4m3, any page and head strides that are multiples of 16, each
    (page, head) block contiguous.  Scales ``k_scale``, ``v_scale``: (pages, heads) e8m0, heads contiguous, from 2^-48 to
    2^48 (or NaN) wherever a token lies: others give inexact results, and nothing but ``KVPlan.check`` looks for them.  A
    value is code * scale.  The tensors stay the caller's and are used in place; which they are is fixed when the cache is
    made."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dim() != 4 or k.shape[3] != HEAD_DIM or k.shape[2] not in PAGE_SIZES or k.shape != v.shape \
                or min(k.shape) < 1:
            raise ValueError("KVCache: k and v must be (pages, heads, page_size, 128) of one shape, page_size one of %s; "
                             "got %s and %s" % (PAGE_SIZES, tuple(k.shape), tuple(v.shape)))
        for t in (k, v):
            if t.dtype != E4M3:
                raise ValueError("KVCache: codes must be float8_e4m3fn, got %s" % t.dtype)
            if t.stride(3) != 1 or t.stride(2) != HEAD_DIM or t.stride(1) % 16 or t.stride(0) % 16 or t.data_ptr() % 16:
                raise ValueError("KVCache: every (page, head) block must be contiguous and 16-byte aligned")
            if t.stride(0) > 0x7fffffff:
                raise ValueError("KVCache: page strides must be below 2^31")
            if not _apart(t.shape[:2], t.stride()[:2], t.shape[2] * HEAD_DIM):
                raise ValueError("KVCache: blocks overlap in memory")
        for t in (k_scale, v_scale):
            if t.dtype != E8M0 or t.shape != k.shape[:2]:
                raise ValueError("KVCache: scales must be float8_e8m0fnu of shape (pages, heads)")
            if t.shape[1] > 1 and t.stride(1) != 1:
                raise ValueError("KVCache: the scales of a page must be contiguous")
            if not _apart(t.shape, t.stride(), 1):
                raise ValueError("KVCache: scales overlap in memory")
        if any(t.device != k.device for t in (v, k_scale, v_scale)):
            raise ValueError("KVCache: all four tensors must be on one device")
        if k.shape[0] > 0x7fffffff:
            raise ValueError("KVCache: too many pages")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.pages, self.heads, self.page_size, _ = k.shape
        self.device, self._index = k.device, k.get_device()
        self._c = _lib.KVCacheParams(
            k=k.data_ptr(), v=v.data_ptr(), k_scale=k_scale.data_ptr(), v_scale=v_scale.data_ptr(),
            k_sp=k.stride(0), k_sh=k.stride(1), v_sp=v.stride(0), v_sh=v.stride(1), ks_sp=k_scale.stride(0),
            vs_sp=v_scale.stride(0), pages=self.pages, heads=self.heads, page_size=self.page_size)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, pages: int, heads: int, page_size: int = 64, device="cuda:0") -> "KVCache":
        """A cache of zero codes and scales of 1."""
        codes = [torch.zeros((pages, heads, page_size, HEAD_DIM), dtype=torch.uint8, device=device).view(E4M3)
                 for _ in range(2)]
        scales = [torch.full((pages, heads), 127, dtype=torch.uint8, device=device).view(E8M0) for _ in range(2)]
        return cls(*codes, *scales)


class KVPlan(_Fixed):
    """A packed batch: rows [row_start[b], row_start[b + 1]) of q, k and v are the newest tokens of sequence b, which
    has kv_len[b] tokens with them; token t of it is in page page_table[b, t // page_size].

    page_table (B, P), row_start (B + 1), kv_len (B): int32 on one device.  Table entries that no row sees a token of may
    hold anything: those behind a sequence's end and, for attention with a window, pages that lie in front of every row's
    (``check`` knows of no window and reports these).  max_rows, max_kv_len: no sequence will have more rows in a call, or
    more tokens.  They size launches (and, with kv_len, how attention splits its work), so they should be near what is used.
    Nothing else about the rows is known to the host: every sequence is worked on as if it had max_rows of them.  Prompts
    and sequences with a token or a few belong in plans and calls of their own (``ops.kv_attention`` has the figures).

    The arrays are not read on the host.  What breaks a bound on the device is left out there: see ``check`` and the
    notes of ``ops.kv_append`` and ``ops.kv_attention``."""

    def __init__(self, page_table: torch.Tensor, row_start: torch.Tensor, kv_len: torch.Tensor, *, max_rows: int,
                 max_kv_len: int):
        if page_table.dim() != 2 or row_start.dim() != 1 or kv_len.dim() != 1 or kv_len.shape[0] < 1 \
                or page_table.shape[0] != kv_len.shape[0] or row_start.shape[0] != kv_len.shape[0] + 1 \
                or page_table.shape[1] < 1:
            raise ValueError("KVPlan: page_table must be (B, P), row_start (B + 1), kv_len (B); got %s, %s, %s"
                             % (tuple(page_table.shape), tuple(row_start.shape), tuple(kv_len.shape)))
        for t in (page_table, row_start, kv_len):
            if t.dtype != torch.int32 or t.stride(-1) != 1:
                raise ValueError("KVPlan: page_table, row_start and kv_len must be int32 with unit stride")
            if t.device != kv_len.device:
                raise ValueError("KVPlan: all three tensors must be on one device")
        if page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]:
            raise ValueError("KVPlan: the rows of page_table overlap")
        if not 0 <= max_rows <= 1 << 30 or not 0 <= max_kv_len <= 1 << 30:
            raise ValueError("KVPlan: max_rows and max_kv_len must lie in [0, 2^30]")
        self.page_table, self.row_start, self.kv_len = page_table, row_start, kv_len
        self.batch, self.table_pages = page_table.shape
        self.max_rows, self.max_kv_len = int(max_rows), int(max_kv_len)
        self.device, self._index = kv_len.device, kv_len.get_device()
        self._c = _lib.KVBatchParams(
            page_table=page_table.data_ptr(), table_sb=max(page_table.stride(0), self.table_pages),
            row_start=row_start.data_ptr(), kv_len=kv_len.data_ptr(), batch=self.batch, table_pages=self.table_pages,
            max_rows=self.max_rows, max_kv_len=self.max_kv_len)
        self._ref = ctypes.byref(self._c)

    def check(self, cache: KVCache, total_rows: int, for_append: bool = True) -> None:
        """Copies the three arrays to the host (which waits for the device) and raises ValueError, naming the first
        sequence, where they break a bound of the plan, of the cache or of ``total_rows`` packed rows; with
        ``for_append`` also where a sequence has more rows than tokens, or a page that is appended to is listed
        twice.  Also where a page that holds tokens (with ``for_append``: tokens before the rows) has a scale whose
        exponent lies outside [-48, 48], which the kernels do not look for (a NaN scale is a value like others)."""
        self._fits(cache)
        table, starts, lens = (t.cpu().contiguous() for t in (self.page_table, self.row_start, self.kv_len))
        host = _lib.KVBatchParams(page_table=table.data_ptr(), table_sb=self.table_pages, row_start=starts.data_ptr(),
                                  kv_len=lens.data_ptr(), batch=self.batch, table_pages=self.table_pages,
                                  max_rows=self.max_rows, max_kv_len=self.max_kv_len)
        bad = ctypes.c_int32(-1)
        rc = _lib.load().dsx_kv_plan_check(ctypes.byref(host), cache.pages, cache.page_size, total_rows,
                                           int(for_append), ctypes.byref(bad))
        if rc != _lib.DSX_OK:
            b = bad.value
            raise ValueError("KVPlan: sequence %d (rows [%d, %d), %d tokens) breaks a bound"
                             % (b, starts[b], starts[b + 1], lens[b]) if b >= 0 else _lib.strerror(rc))
        held = lens - starts.diff() if for_append else lens
        listed = torch.arange(self.table_pages) * cache.page_size < held[:, None]
        ids = torch.where(listed, table, 0).to(cache.device).long()
        for scale in (cache.k_scale, cache.v_scale):
            at = scale.view(torch.uint8)[ids]
            out = ((at < 127 + EXPONENTS[0]) | (at > 127 + EXPONENTS[1])) & (at != 255)
            out = out.any(-1).cpu() & listed
            if out.any():
                b, t = out.nonzero()[0].tolist()
                raise ValueError("KVPlan: sequence %d (page %d) sees a scale outside 2^%d .. 2^%d"
                                 % (b, table[b, t], *EXPONENTS))

    def _fits(self, cache: KVCache):
        if cache._index != self._index:
            raise ValueError("the rows, the cache and the plan must be on one device")
        if self.max_kv_len > self.table_pages * cache.page_size:
            raise ValueError("KVPlan: %d pages of %d tokens cannot hold max_kv_len = %d"
                             % (self.table_pages, cache.page_size, self.max_kv_len))
