"""Paged key-value cache over torch tensors (include/bmo_kernels.h, ``bmo_k_paged_*``).

A server of many sessions keeps their keys and values in pages of one pool
instead of one ring each: ``PageBook`` says which session ("request") has
which pages and plans every step on the device, ``PagedKV`` holds the pages of
all layers, appends rows, reads them back and attends over them.  The caller
owns every tensor; calls run on torch's current stream and do not
synchronise.

    book = PageBook.empty(n_req, n_pages, page_size, max_blocks, window=512)
    kv = PagedKV.empty(book, n_layers, n_kv_heads, head_dim)
    book.plan(n_new, slot, pos, req, offsets)  # once a step
    kv.append(layer, k, v, slot, pos=pos, q=q, q_out=q, theta=10000.0)  # each layer
    kv.attention(layer, q, out)
"""
from __future__ import annotations

import ctypes
import importlib.util
from typing import Optional

import torch

from . import build as _build
from .engine import KV_F16, KV_Q4_0, lib

NO_PAGES, TABLE_FULL, NO_ROOM, BAD_INDEX = 1 << 5, 1 << 6, 1 << 7, 1 << 8


def _load():
    """The extension module that checks tensors and calls the library (binding/paged_torch.cpp)."""
    so = _build.build_binding()
    if so is None:
        raise ImportError("the torch binding of the paged cache needs a torch with CUDA, and torch's, Python's and CUDA's headers")
    spec = importlib.util.spec_from_file_location("_paged", so)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    L = lib()
    m.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (L.bmo_k_paged_plan, L.bmo_k_paged_append, L.bmo_k_paged_read,
                                                             L.bmo_k_paged_attention)))
    return m


_ext = _load()


class _Book(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("table", "lens", "free_pages", "state")] + \
               [(n, ctypes.c_int32) for n in ("n_req", "max_blocks", "n_pages", "page_size", "window")] + \
               [("undo", ctypes.c_void_p)]


class _Cache(ctypes.Structure):
    _fields_ = [("book", _Book)] + [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + \
               [(n, ctypes.c_int32) for n in ("n_layers", "n_kv_heads", "head_dim", "kv_type")]


def _ints(t: torch.Tensor, name: str, device, numel: Optional[int] = None) -> int:
    """Address of a dense int32 tensor on `device`."""
    if t.dtype is not torch.int32 or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor on {device}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: {numel} entries, got {t.numel()}")
    return t.data_ptr()


class PageBook:
    """Block table [n_req, max_blocks], lengths [n_req], ring of free pages
    [n_pages] and state [4] (first free entry, free pages, status bits, new
    positions of the last step): int32 tensors on one GPU.  Keep one PageBook
    for them: it also holds what lets its last plan be dropped and made again."""

    def __init__(self, table: torch.Tensor, lens: torch.Tensor, free: torch.Tensor, state: torch.Tensor, *,
                 page_size: int, window: int = 0):
        if table.dim() != 2 or table.device.type != "cuda":
            raise ValueError("table: [n_req, max_blocks] on a GPU")
        self.table, self.lens, self.free, self.state = table, lens, free, state
        self.page_size, self.window, self.device = int(page_size), int(window), table.device
        # the C struct has 32 bits for them
        if not 1 <= self.page_size <= 65536 or not 0 <= self.window < 1 << 31:
            raise ValueError(f"pages of 1 to 65536 positions, a window from 0 on: got {page_size}, {window}")
        n_req, max_blocks = table.shape
        self._c = _Book(_ints(table, "table", self.device), _ints(lens, "lens", self.device, n_req),
                        _ints(free, "free", self.device), _ints(state, "state", self.device, 4), n_req, max_blocks,
                        free.numel(), self.page_size, self.window)
        self._undo = torch.zeros(4 + 2 * free.numel(), dtype=torch.int32, device=self.device)
        torch.cuda.current_stream(self.device).synchronize()  # plans may be on another stream
        self._c.undo = self._undo.data_ptr()
        self._addr, self._dev = ctypes.addressof(self._c), self.device.index

    @classmethod
    def empty(cls, n_req: int, n_pages: int, page_size: int, max_blocks: int, window: int = 0,
              device="cuda") -> "PageBook":
        """A book of no positions, every page free."""
        i32 = {"dtype": torch.int32, "device": device}
        return cls(torch.full((n_req, max_blocks), -1, **i32), torch.zeros(n_req, **i32),
                   torch.arange(n_pages, **i32), torch.tensor([0, n_pages, 0, 0], **i32), page_size=page_size,
                   window=window)

    def plan(self, n_new: torch.Tensor, slot: torch.Tensor, pos: torch.Tensor, req: torch.Tensor,
             offsets: torch.Tensor, lens_out: Optional[torch.Tensor] = None,
             state_out: Optional[torch.Tensor] = None) -> None:
        """Plans a step (bmo_k_paged_plan): n_new[r] > 0 appends positions to
        request r, 0 leaves it, < 0 ends it.  slot, pos, req [max_tokens] and
        offsets [n_req + 1] receive the list of new positions; the new
        lengths and state replace the book's unless lens_out / state_out are
        given.  The table and the ring change in place.  A plan into lens_out
        and state_out may be dropped: the next one from the book's own, of this
        step or another, is as if it had not been made (the last plan alone, by
        this PageBook).  state[2] != 0 after it: the step was refused, nothing
        changed."""
        _ext.plan(self._addr, self._dev, n_new, slot, pos, req, offsets, lens_out, state_out)


class PagedKV:
    """Keys and values of all layers in the pages of `book`: fp16 tensors
    [n_layers, n_pages, n_kv_heads, page_size, head_dim], or Q4_0 as uint8
    nibble planes [..., head_dim / 2] with fp16 scales [..., head_dim / 32].
    Attention calls of one PagedKV share a scratch buffer: keep them on one
    stream or order them."""

    def __init__(self, book: PageBook, k: torch.Tensor, v: torch.Tensor, *, k_scale: Optional[torch.Tensor] = None,
                 v_scale: Optional[torch.Tensor] = None):
        q4 = k.dtype is torch.uint8
        if k.dim() != 5 or k.dtype not in (torch.float16, torch.uint8):
            raise ValueError("k: fp16 or uint8 [n_layers, n_pages, n_kv_heads, page_size, row]")
        n_layers, n_pages, n_kv, page_size, row = k.shape
        if n_pages != book.free.numel() or page_size != book.page_size:
            raise ValueError("k: the book's pages")
        head_dim = 2 * row if q4 else row
        self.book, self.k, self.v, self.k_scale, self.v_scale = book, k, v, k_scale, v_scale
        self.n_layers, self.n_kv_heads, self.head_dim = n_layers, n_kv, head_dim
        self.kv_type = KV_Q4_0 if q4 else KV_F16
        planes = [("k", k, k.shape, k.dtype), ("v", v, k.shape, k.dtype)]
        if q4:
            scales = k.shape[:-1] + (head_dim // 32,)
            planes += [("k_scale", k_scale, scales, torch.float16), ("v_scale", v_scale, scales, torch.float16)]
        for name, t, shape, dtype in planes:
            if t is None or t.shape != shape or t.dtype is not dtype or t.device != book.device or not t.is_contiguous():
                raise ValueError(f"{name}: a contiguous {dtype} tensor of {tuple(shape)} on {book.device}")
        self._c = _Cache(book._c, k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if q4 else None,
                         v_scale.data_ptr() if q4 else None, n_layers, n_kv, head_dim, self.kv_type)
        self._addr, self._dev = ctypes.addressof(self._c), book.device.index
        # for any number of query heads (what is needed grows with the query heads of a key head up to 8)
        self._scratch_bytes = max(lib().bmo_k_paged_attention_scratch_bytes(self._addr, g * n_kv) for g in (1, 8))
        if self._scratch_bytes == 0:
            raise ValueError(f"a cache of {n_kv} heads of {head_dim}, pages of {page_size}")
        self._scratch = torch.zeros(self._scratch_bytes, dtype=torch.uint8, device=book.device)
        torch.cuda.current_stream(book.device).synchronize()  # the calls may be on another stream
        self._scratch_addr = self._scratch.data_ptr()

    @classmethod
    def empty(cls, book: PageBook, n_layers: int, n_kv_heads: int, head_dim: int, kv_type: int = KV_F16) -> "PagedKV":
        shape = (n_layers, book.free.numel(), n_kv_heads, book.page_size)
        if kv_type == KV_F16:
            k, v = (torch.zeros(shape + (head_dim,), dtype=torch.float16, device=book.device) for _ in range(2))
            return cls(book, k, v)
        k, v = (torch.zeros(shape + (head_dim // 2,), dtype=torch.uint8, device=book.device) for _ in range(2))
        ks, vs = (torch.zeros(shape + (head_dim // 32,), dtype=torch.float16, device=book.device) for _ in range(2))
        return cls(book, k, v, k_scale=ks, v_scale=vs)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, slot: torch.Tensor, *,
               pos: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None,
               q_out: Optional[torch.Tensor] = None, theta: float = 0.0,
               status: Optional[torch.Tensor] = None) -> None:
        """Stores k, v [n, n_kv_heads, head_dim] at slot[n] (bmo_k_paged_append);
        theta > 0 rotates k, and q into q_out, by the positions pos[n]; with
        theta 0 nothing is rotated, pos is not read and q is refused."""
        _ext.append(self._addr, self._dev, layer, k, v, slot, pos, q, q_out, theta, status)

    def read(self, layer: int, slot: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor,
             status: Optional[torch.Tensor] = None) -> None:
        """Rows at slot[n] as k_out, v_out [n, n_kv_heads, head_dim] (bmo_k_paged_read)."""
        _ext.read(self._addr, self._dev, layer, slot, k_out, v_out, status)

    def attention(self, layer: int, q: torch.Tensor, out: torch.Tensor, *, rows: Optional[torch.Tensor] = None,
                  row_lens: Optional[torch.Tensor] = None, scale: float = 0.0, lse: Optional[torch.Tensor] = None,
                  status: Optional[torch.Tensor] = None) -> None:
        """Attention of q [n, n_heads, head_dim] into out (bmo_k_paged_attention).
        Row i is a token of request rows[i] (default i) that attends to the first
        row_lens[i] positions (default, and at most, the book's length); lse [n,
        n_heads] fp32.  With a window, row_lens below the length before the last
        plan can reach pages that were given back."""
        _ext.attention(self._addr, self._dev, layer, q, out, rows, row_lens, scale, lse, status, self._scratch_addr,
                       self._scratch_bytes)
