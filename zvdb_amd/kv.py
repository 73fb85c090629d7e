"""`KVLayout` -- the 4-bit key/value cache of include/zvdb_hip.h: pages and slots from request lengths, rows in and out, attention over
whole requests or over the rows that a search returned.  Like the `_dev` calls of `Index`, its calls take raw device pointers (e.g.
``torch.Tensor.data_ptr()``) plus a stream handle, only enqueue work and keep nothing: cache, tables and lengths are the caller's."""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import KvLayoutStruct, check


class KVLayout:
    """Sizes of a cache: `pages` pages of `page_size` tokens (16 .. 256, a power of two), `kv_heads` heads of `head_dim` elements
    (a multiple of 8 up to 256).  The cache itself is `pages * page_bytes` bytes of device memory."""

    def __init__(self, head_dim: int, kv_heads: int, page_size: int, pages: int):
        self._L = _lib.hip()
        self._s = KvLayoutStruct(_lib.ABI_VERSION, head_dim, kv_heads, page_size, pages)
        self._p = C.byref(self._s)
        b = C.c_uint64(0)
        check(self._L.zvdb_hip_kv_page_bytes(self._p, C.byref(b)))
        self.page_bytes = b.value

    head_dim = property(lambda self: self._s.head_dim)
    kv_heads = property(lambda self: self._s.kv_heads)
    page_size = property(lambda self: self._s.page_size)
    pages = property(lambda self: self._s.pages)

    def plan_dev(self, lengths_ptr: int, new_ptr: int, n: int, ring_ptr: int, ring_size: int, cursor_ptr: int, tables_ptr: int,
                 table_stride: int, starts_ptr: int, slots_ptr: int, slot_cap: int, out_lengths_ptr: int, out_cursor_ptr: int,
                 status_ptr: int, stream: int = 0) -> None:
        """Pages and slots for the new tokens of n requests (zvdb_hip_kv_plan_dev)."""
        check(self._L.zvdb_hip_kv_plan_dev(self._p, lengths_ptr, new_ptr, n, ring_ptr, ring_size, cursor_ptr, tables_ptr, table_stride,
                                           starts_ptr, slots_ptr, slot_cap, out_lengths_ptr, out_cursor_ptr, status_ptr, stream))

    def append_dev(self, cache_ptr: int, k_ptr: int, k_stride: int, v_ptr: int, v_stride: int, type: int, n: int, slots_ptr: int,
                   stream: int = 0) -> None:
        """Keys and values of n tokens, quantised into their slots."""
        check(self._L.zvdb_hip_kv_append_dev(self._p, cache_ptr, k_ptr, k_stride, v_ptr, v_stride, type, n, slots_ptr, stream))

    def read_dev(self, cache_ptr: int, slots_ptr: int, n: int, k_ptr: int, v_ptr: int, type: int, stream: int = 0) -> None:
        """Rows of n slots, widened; k_ptr or v_ptr may be 0."""
        check(self._L.zvdb_hip_kv_read_dev(self._p, cache_ptr, slots_ptr, n, k_ptr, v_ptr, type, stream))

    def attend_workspace(self, type: int, q_heads: int, n: int, rows: int, max_new: int, max_length: int) -> int:
        """Bytes of workspace of attend_dev with these sizes.  Fewer requests or rows may need more: a buffer for calls of several sizes
        takes the largest of their answers."""
        b = C.c_uint64(0)
        check(self._L.zvdb_hip_kv_attend_workspace(self._p, type, q_heads, n, rows, max_new, max_length, C.byref(b)))
        return b.value

    def attend_dev(self, cache_ptr: int, q_ptr: int, q_stride: int, type: int, q_heads: int, n: int, starts_ptr: int, rows: int, max_new: int,
                   lengths_ptr: int, tables_ptr: int, table_stride: int, max_length: int, scale: float, causal: bool, ws_ptr: int,
                   ws_bytes: int, out_ptr: int, lse_ptr: int = 0, stream: int = 0) -> None:
        """Attention of each request's new tokens over all of its tokens (zvdb_hip_kv_attend_dev)."""
        check(self._L.zvdb_hip_kv_attend_dev(self._p, cache_ptr, q_ptr, q_stride, type, q_heads, n, starts_ptr, rows, max_new, lengths_ptr,
                                             tables_ptr, table_stride, max_length, scale, 1 if causal else 0, ws_ptr, ws_bytes, out_ptr,
                                             lse_ptr, stream))

    def attend_selected_dev(self, cache_ptr: int, q_ptr: int, q_stride: int, type: int, q_heads: int, n: int, ids_ptr: int, count_ptr: int,
                            k: int, lengths_ptr: int, tables_ptr: int, table_stride: int, scale: float, out_ptr: int, lse_ptr: int = 0,
                            stream: int = 0) -> None:
        """Attention of one row per request over the tokens that a search listed for it (zvdb_hip_kv_attend_selected_dev)."""
        check(self._L.zvdb_hip_kv_attend_selected_dev(self._p, cache_ptr, q_ptr, q_stride, type, q_heads, n, ids_ptr, count_ptr, k, lengths_ptr,
                                                      tables_ptr, table_stride, scale, out_ptr, lse_ptr, stream))
