"""Batched serving over a paged key/value cache that is quantised as it is written: a step takes some new tokens of each of
several sequences (a decode step, drafted tokens, pieces of prompts, or a mix of them). No counterpart in the reference, which
keeps one float32 cache per sequence (layers/mha/cpu.go:184-207) and walks a prompt token by token.

The layout of a page and the arithmetic are in include/welvet_cuda.h (WvKvPages, WvKvBatch). All pointers are device addresses
(ints); the caller owns the buffers."""
from __future__ import annotations

import ctypes as C

from . import adapters as _adapters
from ._lib import WvKvBatch, WvKvGroups, WvKvPages, WvKvTable, check, lib


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


def Groups(start: int, shared: int, num_groups: int, max_shared: int) -> WvKvGroups:
    """Groups of a batch's sequences that share a prefix: device arrays of int32 (start[num_groups + 1] first sequences, shared[num_groups] tokens in the same
    pages) and the bound of what the second holds."""
    return WvKvGroups(start, shared, num_groups, max_shared)


def AttnSharedCUDA(pages: WvKvPages, batch: WvKvBatch, groups: WvKvGroups, dq: int, dout: int, num_heads: int, scale: float, ldq: int = 0, ldo: int = 0,
                   stream: int = 0) -> None:
    """AttnPagedCUDA without a window, the keys that a group's sequences share read once for all of them (wv_attn_shared_dev)."""
    check(lib().wv_attn_shared_dev(C.byref(pages), C.byref(batch), C.byref(groups), dq, ldq, dout, ldo, num_heads, scale, stream))


def KVTable(refs: int, pages: int, kv_len: int, num_pages: int, page_size: int, num_seqs: int, table_stride: int) -> WvKvTable:
    """The page tables of a cache on the device (WvKvTable): int32 refs[num_pages], pages[num_seqs, table_stride] and kv_len[num_seqs], zeroed for
    an empty cache. pages and kv_len are the ones that a Batch names; all blocks of a stack share one table."""
    return WvKvTable(refs, pages, kv_len, num_pages, page_size, num_seqs, table_stride)


def KVBlocks(pools):
    """The caches of all blocks that use a table, as KVExtendCUDA, KVCompactCUDA and KVCopyCUDA take them: a list of KVPages."""
    return (WvKvPages * len(pools))(*pools)


def KVForkCUDA(table: WvKvTable, dsrc: int, ddst: int, n: int, dkeep: int = 0, stream: int = 0) -> None:
    """The empty sequences ddst[:n] become the first dkeep (0: all) tokens of the sequences dsrc[:n], in the same pages (wv_kv_fork_dev)."""
    check(lib().wv_kv_fork_dev(C.byref(table), dsrc, ddst, dkeep or None, n, stream))


def KVExtendCUDA(table: WvKvTable, dadd: int, dgranted: int = 0, pools=None, stream: int = 0) -> None:
    """Room for dadd[s] more tokens of every sequence, counted in kv_len; shared last pages are copied in all `pools` (KVBlocks). dgranted[s]: 1, or 0
    for a sequence that was refused (wv_kv_extend_dev)."""
    check(lib().wv_kv_extend_dev(C.byref(table), dadd, dgranted or None, pools, len(pools) if pools is not None else 0, stream))


def KVTrimCUDA(table: WvKvTable, n: int, dkeep: int = 0, dseqs: int = 0, stream: int = 0) -> None:
    """The sequences dseqs[:n] (0: the first n) are cut to dkeep[:n] tokens (0: freed) and their pages behind them given back (wv_kv_trim_dev)."""
    check(lib().wv_kv_trim_dev(C.byref(table), dseqs or None, dkeep or None, n, stream))


def KVCompactCUDA(table: WvKvTable, pools, dlive: int, stream: int = 0) -> None:
    """The pages in use move to the front of the pools (KVBlocks, or None); their number goes to dlive (wv_kv_compact_dev)."""
    check(lib().wv_kv_compact_dev(C.byref(table), pools, len(pools) if pools is not None else 0, dlive, stream))


def KVCopyCUDA(pools, dsrc: int, ddst: int, n: int, stream: int = 0) -> None:
    """Pages dsrc[:n] of all `pools` (KVBlocks) copied to pages ddst[:n] (wv_kv_copy_dev)."""
    check(lib().wv_kv_copy_dev(pools, len(pools), dsrc, ddst, n, stream))


class PagedBlockDecoder:
    """One decoder block for a step of several sequences: decode.BlockDecoder's walk (model/transformer/forward.go:57-76) with all
    new tokens of the batch as rows of one projection each, K and V rounded into the block's pages, and attention over them.

    `cfg` is a decode.BlockConfig (MaxSeqLen is not used: the pages bound the lengths), `keys` maps q, k, v, o, gate, up, down to resident
    blob keys, `bufs` maps the working matrices of up to `max_tokens` rows (norm and proj [DModel], q and attn [NumHeads * HeadDim], k and v
    [NumKVHeads * HeadDim], gate and up [IntermediateDim]) and the weights attn_norm / ffn_norm to device pointers. A block has pages of its
    own; the blocks of a stack share the working matrices and the batch. `adapters` maps projections (q, k, v, o, gate, up, down, or some of
    them) to adapters.Adapters of one set of slots and one type."""

    def __init__(self, cfg, keys: dict, bufs: dict, pages: WvKvPages, max_tokens: int, window: int = 0, adapters: dict | None = None):
        self.cfg, self.keys, self.bufs, self.pages, self.max_tokens, self.window = cfg, keys, bufs, pages, max_tokens, window
        self.adapters = adapters or {}
        qd, kd = cfg.NumHeads * cfg.HeadDim, cfg.NumKVHeads * cfg.HeadDim

        def group(names, outs):
            n = len(names)
            return (C.c_uint64 * n)(*[keys[m] for m in names]), (C.c_void_p * n)(*[bufs[m] for m in names]), (C.c_int * n)(*outs)
        self._qkv, self._gu = group(("q", "k", "v"), (qd, kd, kd)), group(("gate", "up"), (cfg.IntermediateDim,) * 2)

    def step(self, dh: int, batch: WvKvBatch, stream: int = 0, groups: WvKvGroups | None = None, plan: int = 0) -> None:
        """The rows of the hidden state [batch.total_q, DModel] at device address dh are updated in place. `groups` says which of the
        batch's sequences share a prefix: attention reads it once for all of them. `plan` (adapters.PlanCUDA over the batch's rows) adds the
        block's adapters to its projections."""
        c, b, k, n, L = self.cfg, self.bufs, self.keys, batch.total_q, lib()
        if n > self.max_tokens:
            raise ValueError(f"{n} new tokens, but the working matrices have {self.max_tokens} rows")
        if groups is not None and self.window:
            raise ValueError("a window and a shared prefix")
        if plan and not self.adapters:
            raise ValueError("a plan of adapters, but the block has none")
        if n == 0:
            return

        def adapt(names, x, outs):
            # the adapters of projections on the same x, added to their outputs in place
            have = [m for m in names if m in self.adapters] if plan else []
            if have:
                _adapters.ApplyCUDA(_adapters.Group([self.adapters[m] for m in have]), plan, n, x, [outs[m] for m in have], stream=stream)
        qd = c.NumHeads * c.HeadDim
        check(L.wv_rmsnorm_dev(dh, b["attn_norm"], b["norm"], n, c.DModel, c.Eps, stream))
        check(L.wv_matvec_dev_multi(self._qkv[0], 3, b["norm"], self._qkv[1], n, c.DModel, self._qkv[2], stream))
        adapt(("q", "k", "v"), b["norm"], b)
        KVWriteCUDA(self.pages, batch, b["k"], b["v"], b["q"], b["q"], c.NumHeads, c.RoPETheta, stream=stream)
        if groups is not None:
            AttnSharedCUDA(self.pages, batch, groups, b["q"], b["attn"], c.NumHeads, 1.0 / (c.HeadDim ** 0.5), stream=stream)
        else:
            AttnPagedCUDA(self.pages, batch, b["q"], b["attn"], c.NumHeads, 1.0 / (c.HeadDim ** 0.5), window=self.window, stream=stream)
        check(L.wv_matvec_dev(k["o"], b["attn"], b["proj"], n, qd, c.DModel, stream))
        adapt(("o",), b["attn"], {"o": b["proj"]})
        check(L.wv_residual_add_dev(dh, b["proj"], n * c.DModel, stream))
        check(L.wv_rmsnorm_dev(dh, b["ffn_norm"], b["norm"], n, c.DModel, c.Eps, stream))
        check(L.wv_matvec_dev_multi(self._gu[0], 2, b["norm"], self._gu[1], n, c.DModel, self._gu[2], stream))
        adapt(("gate", "up"), b["norm"], b)
        check(L.wv_silu_mul_dev(b["gate"], b["up"], b["gate"], n * c.IntermediateDim, stream))
        check(L.wv_matvec_dev(k["down"], b["gate"], b["proj"], n, c.IntermediateDim, c.DModel, stream))
        adapt(("down",), b["gate"], {"down": b["proj"]})
        check(L.wv_residual_add_dev(dh, b["proj"], n * c.DModel, stream))
