"""Host-side mirror of the reference's token pickers (model/sampling/argmax.go:4-18, topk.go:11-50) on the
device: the LM head's logits stay in HBM and only the index comes back."""
from __future__ import annotations

import ctypes as C
import random

from ._lib import check, lib


def ArgMaxCUDA(d_logits: int, n: int, stream: int = 0) -> int:
    """sampling.ArgMax over n device floats at address d_logits (first strict maximum; NaN never wins)."""
    idx = C.c_int()
    check(lib().wv_argmax(d_logits, n, C.byref(idx), stream))
    return idx.value


def SampleTopKCUDA(d_logits: int, n: int, topK: int, temperature: float, deterministic: bool = False,
                   u: float | None = None, stream: int = 0) -> int:
    """sampling.SampleTopK over n device floats. `u` is the uniform draw the reference takes from math/rand inside
    the call (random.random() when omitted). At most 1024 candidates on the device."""
    idx = C.c_int()
    if u is None:
        u = random.random()
    check(lib().wv_topk_sample(d_logits, n, topK, temperature, 1 if deterministic else 0, u, C.byref(idx), stream))
    return idx.value


def SampleRowsCUDA(d_logits: int, rows: int, n: int, d_temperature: int, d_top_k: int, d_top_p: int, d_min_p: int, d_u: int, d_index: int,
                   d_prob: int = 0, ld: int = 0, stream: int = 0) -> None:
    """The next token of every row: temperature, top-k, top-p and min-p of its own from device arrays (float32, int32, float32,
    float32), the draw from d_u (float64); the index (int32; -1 where nothing can be drawn) and its probability (float32) are left in
    device memory. wv_sample_rows_dev; no counterpart in the reference, which samples one row by top-k on the host."""
    check(lib().wv_sample_rows_dev(d_logits, rows, n, ld, d_temperature, d_top_k, d_top_p, d_min_p, d_u, d_index, d_prob or None, stream))
