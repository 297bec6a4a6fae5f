"""The attention half of a block, on device pointers (``rbmoe_attention_*``, ``rbmoe_kv_cache_*``, ``rbmoe_decode_*`` of include/rbmoe.h).

Rows are ``[rows, heads, head_dim]`` with consecutive elements; a stride counts the elements from one row to the next (0: no gap).  Calls are
enqueued on the device's stream (``Device.set_stream``) without synchronisation and allocate nothing.  An argument that is not wanted is passed as
0; ``scale`` 0 stands for ``head_dim ** -0.5``.
"""
from __future__ import annotations

import ctypes as C

from . import _lib as L
from .moe import Device, InvalidConfig, _check
from .operators import _Operator, _dtype, _p


class _Heads(_Operator):
    def _take_heads(self, device: Device, heads: int, kv_heads: int, head_dim: int, dtype: str) -> None:
        self.device, self.heads, self.kv_heads, self.head_dim, self.dtype = device, heads, kv_heads, head_dim, dtype
        self._lib = L.load()

    def _scale(self, scale: float) -> float:
        return scale or self.head_dim ** -0.5


class Attention(_Heads):
    """Attention of whole sequences with grouped heads, packed one behind the other or padded, and its backward pass.

    Sequence ``i`` has the query rows from ``query_begin[i]`` on, ``query_count[i]`` of them, and keys likewise (key arrays 0: the queries');
    all four are i32 on the device.  ``longest_queries`` and ``longest_keys`` size the launches.  ``causal``: a sequence's queries are the last of its
    keys.  Rows that see no key are zeros, rows outside every sequence are left as they are."""

    _destroy = "rbmoe_attention_destroy"

    def __init__(self, device: Device, heads: int, kv_heads: int, head_dim: int, *, dtype: str = "f32", backward_rows: int = 0):
        self._take_heads(device, heads, kv_heads, head_dim, dtype)
        h = C.c_void_p()
        _check(self._lib.rbmoe_attention_create(device.handle, heads, kv_heads, head_dim, _dtype(dtype), backward_rows, C.byref(h)), device.handle)
        self.handle = h

    def forward_device(self, sequences: int, q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, *, query_begin_ptr: int, query_count_ptr: int,
                       key_begin_ptr: int = 0, key_count_ptr: int = 0, query_rows: int, key_rows: int, longest_queries: int,
                       longest_keys: int, q_stride: int = 0, k_stride: int = 0, v_stride: int = 0, causal: bool = True, scale: float = 0.0,
                       lse_ptr: int = 0) -> None:
        """``lse`` (``[heads, query_rows]`` f32) is what the backward pass needs beside ``out``."""
        _check(self._lib.rbmoe_attention_forward(self.handle, sequences, longest_queries, longest_keys, _p(query_begin_ptr), _p(query_count_ptr),
                                                 _p(key_begin_ptr), _p(key_count_ptr), query_rows, key_rows, _p(q_ptr), q_stride, _p(k_ptr), k_stride,
                                                 _p(v_ptr), v_stride, int(causal), self._scale(scale), _p(out_ptr), _p(lse_ptr)),
               self.device.handle)

    def backward_device(self, sequences: int, q_ptr: int, k_ptr: int, v_ptr: int, out_ptr: int, lse_ptr: int, grad_out_ptr: int, grad_q_ptr: int,
                        grad_k_ptr: int, grad_v_ptr: int, *, query_begin_ptr: int, query_count_ptr: int, key_begin_ptr: int = 0,
                        key_count_ptr: int = 0, query_rows: int, key_rows: int, longest_queries: int, longest_keys: int, q_stride: int = 0,
                        k_stride: int = 0, v_stride: int = 0, causal: bool = True, scale: float = 0.0) -> None:
        """Gradients of the three inputs, each with its input's stride."""
        _check(self._lib.rbmoe_attention_backward(self.handle, sequences, longest_queries, longest_keys, _p(query_begin_ptr), _p(query_count_ptr),
                                                  _p(key_begin_ptr), _p(key_count_ptr), query_rows, key_rows, _p(q_ptr), q_stride, _p(k_ptr), k_stride,
                                                  _p(v_ptr), v_stride, int(causal), self._scale(scale), _p(out_ptr), _p(lse_ptr),
                                                  _p(grad_out_ptr), _p(grad_q_ptr), _p(grad_k_ptr), _p(grad_v_ptr)), self.device.handle)


class KvCache(_Heads):
    """Keys and values in pages of ``page_rows`` rows: row ``r`` of page ``p`` is slot ``p * page_rows + r``.  ``cache_dtype`` is the rows' type or
    "int8" (a scale a row and head)."""

    _destroy = "rbmoe_kv_cache_destroy"

    def __init__(self, device: Device, kv_heads: int, head_dim: int, pages: int, *, page_rows: int = 16, dtype: str = "f32",
                 cache_dtype: str = ""):
        if cache_dtype and cache_dtype not in L.DTYPES:
            raise InvalidConfig(f"cache_dtype must be f32, bf16 or int8, got {cache_dtype}")
        self._take_heads(device, kv_heads, kv_heads, head_dim, dtype)
        self.pages, self.page_rows, self.cache_dtype = pages, page_rows, cache_dtype or dtype
        h = C.c_void_p()
        _check(self._lib.rbmoe_kv_cache_create(device.handle, kv_heads, head_dim, _dtype(dtype), L.DTYPES[self.cache_dtype], page_rows, pages,
                                               C.byref(h)), device.handle)
        self.handle = h

    def write_device(self, rows: int, k_ptr: int, v_ptr: int, slots_ptr: int, *, k_stride: int = 0, v_stride: int = 0) -> None:
        """Rows to their slots (i64 on the device, all different); rows without one (negative, behind the last page) are left out."""
        _check(self._lib.rbmoe_kv_cache_write(self.handle, rows, _p(k_ptr), k_stride, _p(v_ptr), v_stride, _p(slots_ptr)), self.device.handle)

    def read_device(self, rows: int, k_ptr: int, v_ptr: int, slots_ptr: int, *, k_stride: int = 0, v_stride: int = 0) -> None:
        """The rows of slots; those without one are zeros."""
        _check(self._lib.rbmoe_kv_cache_read(self.handle, rows, _p(k_ptr), k_stride, _p(v_ptr), v_stride, _p(slots_ptr)), self.device.handle)


class DecodeAttention(_Heads):
    """Attention of one new row a sequence over a ``KvCache`` of the same heads; one object serves the caches of all layers."""

    _destroy = "rbmoe_decode_destroy"

    def __init__(self, device: Device, heads: int, kv_heads: int, head_dim: int, max_sequences: int, *, dtype: str = "f32"):
        self._take_heads(device, heads, kv_heads, head_dim, dtype)
        self.max_sequences = max_sequences
        h = C.c_void_p()
        _check(self._lib.rbmoe_decode_create(device.handle, heads, kv_heads, head_dim, _dtype(dtype), max_sequences, C.byref(h)), device.handle)
        self.handle = h

    def forward_device(self, cache: KvCache, sequences: int, q_ptr: int, out_ptr: int, tables_ptr: int, table_pages: int, lengths_ptr: int, *,
                       longest: int, q_stride: int = 0, scale: float = 0.0) -> None:
        """``tables`` ``[sequences, table_pages]`` and ``lengths`` are i32 on the device; a length counts the new row, whose key and value are in
        the cache already."""
        _check(self._lib.rbmoe_decode_attention(self.handle, cache.handle, sequences, _p(q_ptr), q_stride, _p(tables_ptr), table_pages,
                                                _p(lengths_ptr), longest, self._scale(scale), _p(out_ptr)), self.device.handle)
