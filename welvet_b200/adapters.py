"""Low-rank adapters of many requests beside a shared projection: y_r = base_r + scale_s B_s (A_s x_r) for the adapter s of every row r.
No counterpart in the reference.

The layout and the arithmetic are in include/welvet_cuda.h (WvAdapters). All pointers are device addresses (ints); the caller owns the
buffers."""
from __future__ import annotations

import ctypes as C

from ._lib import WvAdapters, check, lib


def Adapters(a: int, b: int, rank: int, scale: int, slots: int, max_rank: int, in_: int, out: int, dtype: int) -> WvAdapters:
    """The adapters of one projection: a[slots, max_rank, in_] and b[slots, out, max_rank] of `dtype` (a core.DType value: quant.DTypeFloat32, DTypeFloat16 or
    DTypeBFloat16), int32 rank[slots] and float32 scale[slots] (either 0: max_rank, 1)."""
    return WvAdapters(a, b, rank or None, scale or None, slots, max_rank, in_, out, dtype)


def Group(targets):
    """Up to four projections on the same x, as ApplyCUDA takes them: a list of Adapters."""
    return (WvAdapters * len(targets))(*targets)


def PlanBytes(rows: int, slots: int) -> int:
    """Bytes of the plan of a step of `rows` rows."""
    n = C.c_uint64()
    check(lib().wv_adapter_plan_bytes(rows, slots, C.byref(n)))
    return n.value


def PlanCUDA(dslot: int, rows: int, slots: int, dplan: int, stream: int = 0) -> None:
    """The rows of a step sorted by adapter: int32 dslot[rows], -1 for none (wv_adapter_plan_dev)."""
    check(lib().wv_adapter_plan_dev(dslot, rows, slots, dplan, stream))


def ApplyCUDA(group, dplan: int, rows: int, dx: int, dy, dbase=None, ldx: int = 0, ldy=None, ldb=None, stream: int = 0) -> None:
    """dy[i] = dbase[i] (None: dy[i]) + scale B (A x) for the targets of `group` (wv_adapter_apply_dev). ldy and ldb are lists of row strides; ldb None: as ldy."""
    n = len(group)
    y, strides = (C.c_void_p * n)(*dy), (C.c_int * n)(*ldy) if ldy is not None else None
    base = (C.c_void_p * n)(*dbase) if dbase is not None else None
    check(lib().wv_adapter_apply_dev(group, n, dplan, rows, dx, ldx, base, (C.c_int * n)(*ldb) if ldb is not None else strides, y, strides, stream))
