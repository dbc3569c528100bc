"""Serving over a paged key-value cache (include/mfh_attention.h).

Block tables and slot maps, rotary positions with the cache's writes, and
attention over pages.  Device buffers are integer pointers and streams
``hipStream_t`` integers, as in ``abi``; the descriptors below hold what a
program keeps from call to call.
"""
from __future__ import annotations

import ctypes

from .abi import F8E4M3, KVCacheStruct, AttentionShape, RotaryShape, check, lib

ROTARY_PLAIN, ROTARY_LINEAR, ROTARY_BASE, ROTARY_BANDS = 0, 1, 2, 3


class KVCache(KVCacheStruct):
    """Layout of the key and the value buffer; [pages, kv_heads, page_size, head_dim] unless strides are given."""

    def __init__(self, dtype: int, page_size: int, kv_heads: int, head_dim: int, pages: int, page_stride: int | None = None,
                 token_stride: int | None = None, head_stride: int | None = None, k_scale: float = 1.0,
                 v_scale: float = 1.0):
        super().__init__()
        self.dtype, self.page_size, self.kv_heads, self.head_dim, self.pages = dtype, page_size, kv_heads, head_dim, pages
        self.token_stride = head_dim if token_stride is None else token_stride
        self.head_stride = page_size * head_dim if head_stride is None else head_stride
        self.page_stride = kv_heads * page_size * head_dim if page_stride is None else page_stride
        self.k_scale, self.v_scale = k_scale, v_scale

    @property
    def element_bytes(self) -> int:
        return 1 if self.dtype == F8E4M3 else 2


def _strides(given, heads: int, dim: int):
    return (heads * dim, dim) if given is None else given


class Rotary(RotaryShape):
    """Shape of a rotary call.  Strides are (token, head) pairs in elements, dense [tokens, heads, head_dim] by default."""

    def __init__(self, dtype: int, q_heads: int, kv_heads: int, head_dim: int, rotary_dim: int | None = None,
                 interleaved: bool = False, inverse: bool = False, factor: float = 1.0, q_strides=None,
                 q_out_strides=None, k_strides=None, k_out_strides=None, v_strides=None):
        super().__init__()
        self.dtype, self.interleaved, self.inverse = dtype, int(interleaved), int(inverse)
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        self.factor = factor
        self.q_token_stride, self.q_head_stride = _strides(q_strides, q_heads, head_dim)
        self.q_out_token_stride, self.q_out_head_stride = _strides(q_out_strides, q_heads, head_dim)
        self.k_token_stride, self.k_head_stride = _strides(k_strides, kv_heads, head_dim)
        self.k_out_token_stride, self.k_out_head_stride = _strides(k_out_strides, kv_heads, head_dim)
        self.v_token_stride, self.v_head_stride = _strides(v_strides, kv_heads, head_dim)


class Attention(AttentionShape):
    """Shape of an attention call.  Strides as in Rotary; without them q and out are dense [tokens, q_heads, head_dim]."""

    def __init__(self, dtype: int, q_heads: int, scale: float, softcap: float = 0.0, window: int = 0,
                 q_strides=None, out_strides=None):
        super().__init__()
        self.dtype, self.q_heads, self.scale, self.softcap, self.window = dtype, q_heads, scale, softcap, window
        self.q_token_stride, self.q_head_stride = (0, 0) if q_strides is None else q_strides
        self.out_token_stride, self.out_head_stride = (0, 0) if out_strides is None else out_strides


def page_plan(before: int, after: int, requests: int, page_size: int, table: int, table_width: int, ring: int,
              ring_size: int, ring_state: int, ring_state_out: int, slots: int, positions: int, tokens: int, starts: int,
              lengths: int, status: int, table_stride: int | None = None, stream: int = 0) -> None:
    """Pages, slots and positions of one step from the requests' lengths before and after it."""
    check(lib().mfh_page_plan(before, after, requests, page_size, table,
                              table_width if table_stride is None else table_stride, table_width, ring, ring_size,
                              ring_state, ring_state_out, slots, positions, tokens, starts, lengths, status, stream))


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: int = ROTARY_PLAIN, factor: float = 1.0,
                       original_length: float = 0.0, low: float = 1.0, high: float = 32.0) -> list:
    """The rotary_dim / 2 frequencies in radians per position, as f64 on the host."""
    out = (ctypes.c_double * max(1, rotary_dim // 2))()
    check(lib().mfh_rotary_frequencies(out, rotary_dim, base, scaling, factor, original_length, low, high))
    return list(out)[: rotary_dim // 2]


def rotary(shape: Rotary, tokens: int, q: int, q_out: int, k: int, k_out: int, positions: int, frequencies: int,
           stream: int = 0) -> None:
    """Turns q and k by their positions (back, with shape.inverse)."""
    check(lib().mfh_rotary(shape, tokens, q, q_out, k, k_out, positions, frequencies, stream))


def rotary_append(shape: Rotary, cache: KVCache, tokens: int, q: int, q_out: int, k: int, v: int, positions: int,
                  slots: int, frequencies: int, k_cache: int, v_cache: int, stream: int = 0) -> None:
    """Turns q and k by their positions and writes k and v to their slots of the cache."""
    check(lib().mfh_rotary_append(shape, cache, tokens, q, q_out, k, v, positions, slots, frequencies, k_cache, v_cache,
                                  stream))


def paged_decode_workspace(shape: Attention, cache: KVCache, requests: int, longest: int) -> int:
    """Bytes of workspace with which paged_decode splits as far as it pays."""
    need = ctypes.c_size_t()
    check(lib().mfh_paged_decode_workspace(shape, cache, requests, longest, ctypes.byref(need)))
    return need.value


def paged_decode(shape: Attention, cache: KVCache, requests: int, q: int, k_cache: int, v_cache: int, table: int,
                 table_width: int, lengths: int, longest: int, slopes: int, out: int, lse: int, workspace: int = 0,
                 workspace_bytes: int = 0, table_stride: int | None = None, stream: int = 0) -> None:
    """Attention of one new token per request over its pages."""
    check(lib().mfh_paged_decode(shape, cache, requests, q, k_cache, v_cache, table,
                                 table_width if table_stride is None else table_stride, table_width, lengths, longest,
                                 slopes, out, lse, workspace, workspace_bytes, stream))


def paged_prefill_workspace(shape: Attention, cache: KVCache, requests: int, tokens: int, most_fresh: int,
                            longest: int) -> int:
    """Bytes of workspace with which paged_prefill splits as far as it pays."""
    need = ctypes.c_size_t()
    check(lib().mfh_paged_prefill_workspace(shape, cache, requests, tokens, most_fresh, longest, ctypes.byref(need)))
    return need.value


def paged_prefill(shape: Attention, cache: KVCache, requests: int, tokens: int, most_fresh: int, q: int, k_cache: int,
                  v_cache: int, table: int, table_width: int, starts: int, lengths: int, longest: int, prefix: int,
                  slopes: int, out: int, lse: int, workspace: int = 0, workspace_bytes: int = 0,
                  table_stride: int | None = None, stream: int = 0) -> None:
    """Attention of each request's new tokens over its pages."""
    check(lib().mfh_paged_prefill(shape, cache, requests, tokens, most_fresh, q, k_cache, v_cache, table,
                                  table_width if table_stride is None else table_stride, table_width, starts, lengths,
                                  longest, prefix, slopes, out, lse, workspace, workspace_bytes, stream))
