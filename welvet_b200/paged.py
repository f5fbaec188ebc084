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


class PagedBlockDecoder:
    """One decoder block for a step of several sequences: decode.BlockDecoder's walk (model/transformer/forward.go:57-76) with all
    new tokens of the batch as rows of one projection each, K and V rounded into the block's pages, and attention over them.

    `cfg` is a decode.BlockConfig (MaxSeqLen is not used: the pages bound the lengths), `keys` maps q, k, v, o, gate, up, down to resident
    blob keys, `bufs` maps the working matrices of up to `max_tokens` rows (norm and proj [DModel], q and attn [NumHeads * HeadDim], k and v
    [NumKVHeads * HeadDim], gate and up [IntermediateDim]) and the weights attn_norm / ffn_norm to device pointers. A block has pages of its
    own; the blocks of a stack share the working matrices and the batch."""

    def __init__(self, cfg, keys: dict, bufs: dict, pages: WvKvPages, max_tokens: int, window: int = 0):
        self.cfg, self.keys, self.bufs, self.pages, self.max_tokens, self.window = cfg, keys, bufs, pages, max_tokens, window
        qd, kd = cfg.NumHeads * cfg.HeadDim, cfg.NumKVHeads * cfg.HeadDim

        def group(names, outs):
            n = len(names)
            return (C.c_uint64 * n)(*[keys[m] for m in names]), (C.c_void_p * n)(*[bufs[m] for m in names]), (C.c_int * n)(*outs)
        self._qkv, self._gu = group(("q", "k", "v"), (qd, kd, kd)), group(("gate", "up"), (cfg.IntermediateDim,) * 2)

    def step(self, dh: int, batch: WvKvBatch, stream: int = 0) -> None:
        """The rows of the hidden state [batch.total_q, DModel] at device address dh are updated in place."""
        c, b, k, n, L = self.cfg, self.bufs, self.keys, batch.total_q, lib()
        if n > self.max_tokens:
            raise ValueError(f"{n} new tokens, but the working matrices have {self.max_tokens} rows")
        if n == 0:
            return
        qd = c.NumHeads * c.HeadDim
        check(L.wv_rmsnorm_dev(dh, b["attn_norm"], b["norm"], n, c.DModel, c.Eps, stream))
        check(L.wv_matvec_dev_multi(self._qkv[0], 3, b["norm"], self._qkv[1], n, c.DModel, self._qkv[2], stream))
        KVWriteCUDA(self.pages, batch, b["k"], b["v"], b["q"], b["q"], c.NumHeads, c.RoPETheta, stream=stream)
        AttnPagedCUDA(self.pages, batch, b["q"], b["attn"], c.NumHeads, 1.0 / (c.HeadDim ** 0.5), window=self.window, stream=stream)
        check(L.wv_matvec_dev(k["o"], b["attn"], b["proj"], n, qd, c.DModel, stream))
        check(L.wv_residual_add_dev(dh, b["proj"], n * c.DModel, stream))
        check(L.wv_rmsnorm_dev(dh, b["ffn_norm"], b["norm"], n, c.DModel, c.Eps, stream))
        check(L.wv_matvec_dev_multi(self._gu[0], 2, b["norm"], self._gu[1], n, c.DModel, self._gu[2], stream))
        check(L.wv_silu_mul_dev(b["gate"], b["up"], b["gate"], n * c.IntermediateDim, stream))
        check(L.wv_matvec_dev(k["down"], b["gate"], b["proj"], n, c.IntermediateDim, c.DModel, stream))
        check(L.wv_residual_add_dev(dh, b["proj"], n * c.DModel, stream))
