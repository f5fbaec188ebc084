"""Batched serving over a paged key/value cache that is quantised as it is written: a step takes some new tokens of each of
several sequences (a decode step, drafted tokens, pieces of prompts, or a mix of them). No counterpart in the reference, which
keeps one float32 cache per sequence (layers/mha/cpu.go:184-207) and walks a prompt token by token.

The layout of a page and the arithmetic are in include/welvet_cuda.h (WvKvPages, WvKvBatch). All pointers are device addresses
(ints); the caller owns the buffers."""
from __future__ import annotations

import ctypes as C

from ._lib import WvKvBatch, WvKvPages, check, lib


def KVBlockBytes(bits: int, page_size: int, head_dim: int) -> int:
    """Bytes of one page of one kv head (K and V); a pool takes num_pages * num_kv_heads of them."""
    n = C.c_uint64()
    check(lib().wv_kv_block_bytes(bits, page_size, head_dim, C.byref(n)))
    return n.value


def KVPages(pool: int, bits: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int) -> WvKvPages:
    """The paged cache of one block: `pool` holds num_pages * num_kv_heads * KVBlockBytes(...) bytes."""
    return WvKvPages(pool, bits, num_pages, page_size, num_kv_heads, head_dim)


def Batch(q_start: int, kv_len: int, pages: int, num_seqs: int, table_stride: int, total_q: int, max_q: int, max_kv: int) -> WvKvBatch:
    """The sequences of a step: device arrays of int32 (q_start[num_seqs + 1], kv_len[num_seqs], pages[num_seqs, table_stride]) and
    the bounds of what they hold."""
    return WvKvBatch(q_start, kv_len, pages, num_seqs, table_stride, total_q, max_q, max_kv)


def KVWriteCUDA(pages: WvKvPages, batch: WvKvBatch, dk: int, dv: int, dq: int = 0, dq_out: int = 0, num_heads: int = 0, theta: float = 0.0,
                ldk: int = 0, ldv: int = 0, ldq: int = 0, ldqo: int = 0, stream: int = 0) -> None:
    """RoPE on the new tokens' Q (dq to dq_out) and K, and K and V into the pages (wv_kv_write_dev)."""
    check(lib().wv_kv_write_dev(C.byref(pages), C.byref(batch), dk, ldk, dv, ldv, dq or None, ldq, dq_out or None, ldqo, num_heads, theta, stream))


def KVReadCUDA(pages: WvKvPages, batch: WvKvBatch, dk: int, dv: int, ldk: int = 0, ldv: int = 0, stream: int = 0) -> None:
    """The new tokens' K and V as the cache holds them, float32 (wv_kv_read_dev)."""
    check(lib().wv_kv_read_dev(C.byref(pages), C.byref(batch), dk, ldk, dv, ldv, stream))


def AttnPagedCUDA(pages: WvKvPages, batch: WvKvBatch, dq: int, dout: int, num_heads: int, scale: float, window: int = 0, ldq: int = 0,
                  ldo: int = 0, stream: int = 0) -> None:
    """Causal attention of the new tokens over their sequence's cache, optionally the last `window` positions of it (wv_attn_paged_dev)."""
    check(lib().wv_attn_paged_dev(C.byref(pages), C.byref(batch), dq, ldq, dout, ldo, num_heads, scale, window, stream))
