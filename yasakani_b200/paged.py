"""A paged cache of 16-bit rows: many sequences in one pool of pages, for servers that do not know a sequence's length ahead.

The packed caches (kv4.py, kvx.py) keep a sequence in one run of `max_ctx` rows of their own.  Here a layer's rows lie in pages of 16 to 128 tokens that a
table hands to sequences; several sequences may name the same page (a common prompt).  Rules as there: tensors are device memory, every call is
enqueue-only on the current stream of the cache's device (or `stream`), all arithmetic happens in libyskn_kv4.so, no fallback.

Rows of a pass: `seq` and `pos` int32 [rows], the sequence and position of each row; `table` int32 [sequences][blocks], the page of each block of `page`
tokens, anything outside the pool where there is none.  A row whose `seq` is outside the table is padding (of a captured graph's batch, say): nothing is read or
written for it.  A pass of a layer is append, (select,) attention:

    cache = paged.PagedCache(pages, hkv, hd, page=64, dtype=torch.bfloat16)
    ws = paged.workspace(cache, rows, nh, table.shape[1])
    paged.launch_append(cache, table, k, v, seq, pos, rope, rd, q=q, q_out=q16)
    paged.launch_attention(q16, cache, table, seq, pos, qscale, o16, ws)
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import PagedCacheC, check, host
from .kv4 import _dtype_code


class PagedCache:
    """One layer's pages: k, v [pages][hkv][page][hd], and with `means` kmean [pages][hkv][hd], the mean key of every page that has been filled.
    What the tensors hold may be written by anyone; the tensors themselves stay those of the start, whose addresses the tensor maps hold (`of` makes a cache over others)."""

    k = property(lambda self: self._k)
    v = property(lambda self: self._v)
    kmean = property(lambda self: self._kmean)

    def __init__(self, pages: int, hkv: int, hd: int, page: int = 64, dtype=torch.bfloat16, means: bool = False, device="cuda"):
        z = lambda *shape: torch.zeros(shape, dtype=dtype, device=device)
        self._bind(z(pages, hkv, page, hd), z(pages, hkv, page, hd), z(pages, hkv, hd) if means else None)

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor, kmean: torch.Tensor | None = None) -> "PagedCache":
        """A cache over tensors that are there already."""
        self = cls.__new__(cls)
        self._bind(k, v, kmean)
        return self

    def _bind(self, k, v, kmean):
        if k.dim() != 4 or k.shape != v.shape or (kmean is not None and kmean.shape != (k.shape[0], k.shape[1], k.shape[3])):
            raise ValueError("k, v [pages, hkv, page, hd], kmean [pages, hkv, hd]")
        if any(t.dtype != k.dtype or t.device != k.device for t in (v, kmean) if t is not None) or k.dtype not in (torch.float16, torch.bfloat16):
            raise TypeError("k, v and kmean are all fp16 or all bf16, on one device")
        if not all(t.is_cuda and t.is_contiguous() for t in (k, v, kmean) if t is not None):
            raise AssertionError("device buffers must be contiguous CUDA tensors")
        self._k, self._v, self._kmean = k, v, kmean
        self.pages, self.hkv, self.page, self.hd = k.shape
        self.dtype, self.device = k.dtype, k.device
        self.c = PagedCacheC(k.data_ptr(), v.data_ptr(), kmean.data_ptr() if kmean is not None else None, self.pages, self.hkv, self.page, self.hd, _dtype_code(k))
        check(_lib.load().yskn_kv4_paged_init(C.byref(self.c)), "yskn_kv4_paged_init")

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.kmean) if t is not None)


def workspace(cache: PagedCache, rows: int, nh: int, blocks: int, shared: int = 0, select: bool = False) -> torch.Tensor:
    """Scratch for launch_attention over up to `rows` rows with up to `shared` common tokens, and with `select` for launch_select over a table of `blocks`.
    It serves one call at a time: calls that may overlap (two streams, two graphs replayed together) need one each."""
    n = _lib.load().yskn_kv4_paged_workspace_bytes(C.byref(cache.c), rows, nh, shared, blocks if select else 0)
    if n == 0:
        raise ValueError(_lib.load().yskn_kv4_last_error().decode(errors="replace"))
    return torch.empty(n, dtype=torch.uint8, device=cache.device)


def launch_append(cache: PagedCache, table, k, v, seq, pos, rope=None, rd: int = 0, q=None, q_out=None, stream=None) -> None:
    """Rotates keys (and queries, into q_out) at each row's position and writes keys and values into their pages, mean keys of pages that
    are full with these rows too (yskn_kv4_paged_append).  k, v [rows][hkv][hd], q [rows][nh][hd] in the cache's type; rows may be slices of a wider
    tensor (their heads are contiguous).  rope: fp32 [positions][rd / 2][2] as kv4.launch_rope_table_g writes it,
    or the same numbers as [positions][rd] or flat; a table of another rotary width is refused."""
    host.paged_append(cache.c, cache.k, table, k, v, seq, pos, rope, rd, q, q_out, stream)


def launch_select(q, cache: PagedCache, table, seq, pos, ids, ws, stream=None) -> None:
    """The blocks that each row attends to, per kv-head: ids int32 [rows][hkv][take] = the take - 1 blocks with the highest score and the row's last block, in
    rising order, -1 behind them (yskn_kv4_paged_select).  The cache keeps mean keys."""
    host.paged_select(cache.c, cache.k, table, seq, pos, q, ids, ws, stream)


def launch_attention(q, cache: PagedCache, table, seq, pos, qscale: float, o16, ws, shared: int = 0, blocks=None, stream=None) -> None:
    """Attention of every row over tokens 0 .. pos of its sequence into o16 [rows][nh][hd] (yskn_kv4_paged_attention).  shared: so many first tokens lie on the same
    pages for every row, and are read once for all: a common prompt, or what lies in front of a chunk of one sequence whose rows these are.  blocks: int32 [rows][hkv][take], the only blocks that a row sees (launch_select)."""
    host.paged_attention(cache.c, cache.k, table, seq, pos, q, qscale, o16, shared, blocks, ws, stream)
