"""The operators of batched serving, as cases: a paged key/value cache that is quantised as it is written, the attention of
new tokens over it, and the choice of the next token of many rows.

A case is a dict of plain values; `kind` names the operator:

  cache    the new tokens of a batch of sequences: RoPE on Q and K, K and V rounded to `bits` bits into the pages of their
           sequences, and the same tokens read back as float32 (`paged.KVWriteCUDA`, `paged.KVReadCUDA`)
  attn     attention of those tokens over the cached ones of their sequence (`paged.AttnPagedCUDA`): causal, grouped-query
           heads, optionally a sliding window; q = 1 is a decode step
  sample   temperature, top-k, top-p and min-p over rows of logits, from given random numbers (`sampling.SampleRowsCUDA`)

`seqs` sequences have up to `q` new tokens and up to `kv` cached ones, the new ones among them; `ragged` spreads both over the
sequences and leaves one of them empty. `run` makes the framework's calls where `own` is set; otherwise it computes the same with
elementary torch operations. `exact` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

THETA = 10000.0
PHI, PSI = 0.6180339887498949, 0.7548776662466927


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a token of one sequence joins the cache of an 8B-shaped block: the step of a single user, all latency
        {"name": "cache_one", "kind": "cache", "bits": 8, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "seqs": 1, "q": 1, "kv": 2049, "ragged": False},
        # a server's decode step: a token of each of 200 sequences, 4-bit pages of 16 tokens
        {"name": "cache_batch", "kind": "cache", "bits": 4, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 16, "seqs": 200, "q": 1, "kv": 1500, "ragged": False},
        # prompts of different lengths written at once
        {"name": "cache_prompt", "kind": "cache", "bits": 8, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "seqs": 6, "q": 4096, "kv": 4096, "ragged": True},
        # one token over a chat's cache: the attention of a single user's decode step
        {"name": "attn_one", "kind": "attn", "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "seqs": 1, "q": 1, "kv": 2049, "ragged": False, "window": 0},
        # one token over a long document in 4 bits, 70B-shaped heads
        {"name": "attn_long", "kind": "attn", "bits": 4, "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 64, "seqs": 1, "q": 1, "kv": 131000, "ragged": False, "window": 0},
        # a server's decode step: 64 sequences of different lengths
        {"name": "attn_batch", "kind": "attn", "bits": 8, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "seqs": 64, "q": 1, "kv": 8192, "ragged": True, "window": 0},
        # drafted tokens checked together: five a sequence, small heads, a page size that is no power of two
        {"name": "attn_draft", "kind": "attn", "bits": 16, "heads": 16, "kv_heads": 4, "head_dim": 64, "page": 48, "seqs": 16, "q": 5, "kv": 3000, "ragged": False, "window": 0},
        # a piece of a prompt in 8 bits, as a server mixes it in between decode steps
        {"name": "attn_chunk", "kind": "attn", "bits": 8, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "seqs": 1, "q": 512, "kv": 4608, "ragged": False, "window": 0},
        # whole prompts of different lengths
        {"name": "attn_prompt", "kind": "attn", "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "seqs": 4, "q": 4096, "kv": 4096, "ragged": True, "window": 0},
        # a long prompt's chunk with a sliding window, 70B-shaped heads, 4 bits
        {"name": "attn_window", "kind": "attn", "bits": 4, "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 16, "seqs": 1, "q": 2048, "kv": 10000, "ragged": False, "window": 4000},
        # the next token of one user over an LM head's logits
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": 128256, "mix": False},
        # the next tokens of a batch whose users ask for different cuts
        {"name": "sample_batch", "kind": "sample", "rows": 128, "vocab": 128256, "mix": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["cache", "attn", "attn", "attn", "sample"])
    if kind == "sample":
        vocab = _log(rng, 1000, 160000)
        return {"kind": "sample", "rows": min(_log(rng, 1, 256), 128 * 128256 // vocab), "vocab": vocab, "mix": rng.random() < 0.7}
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"kind": kind, "bits": rng.choice((16, 8, 4)), "heads": kv_heads * rng.choice((1, 2, 3, 4, 8)), "kv_heads": kv_heads,
            "head_dim": rng.choice((64, 64, 80, 128, 128, 128)), "page": rng.choice((16, 32, 48, 64, 128)), "seqs": 1, "q": 1, "kv": 1}
    if kind == "cache":
        case["q"] = _log(rng, 1, 2048)
        case["seqs"] = _log(rng, 1, max(2, 8192 // case["q"]))
        case["kv"] = case["q"] + _log(rng, 1, 3000)
        while case["seqs"] * case["kv"] > 400000 or case["seqs"] * case["q"] * case["heads"] > 300000:
            case["seqs"], case["q"] = max(1, case["seqs"] // 2), max(1, case["q"] * 3 // 4)
        case["ragged"] = rng.random() < 0.5
        return case
    form = rng.choice(("token", "token", "draft", "chunk", "prompt"))
    if form == "token":
        case["seqs"] = _log(rng, 1, 128)
        case["kv"] = _log(rng, 16, 131072)
    elif form == "draft":
        case["q"], case["seqs"], case["kv"] = rng.randint(2, 17), _log(rng, 1, 32), _log(rng, 64, 16384)
    elif form == "chunk":
        case["q"] = _log(rng, 64, 2048)
        case["kv"] = case["q"] + _log(rng, 16, 8192)
    else:
        case["q"] = _log(rng, 64, 4096)
        case["kv"], case["seqs"] = case["q"], rng.randint(1, 4)
    while case["seqs"] > 1 and case["seqs"] * case["kv"] > 500000:
        case["seqs"] //= 2
    case["kv"] = max(case["kv"], case["q"])
    case["ragged"] = case["seqs"] > 1 and rng.random() < 0.6
    case["window"] = _log(rng, 16, case["kv"] + 1) if rng.random() < 0.25 else 0
    while work(case)["flops"] > 2.5e11 or work(case)["bytes"] > 5e8:
        case["heads"] = max(case["kv_heads"], case["heads"] // 2 // case["kv_heads"] * case["kv_heads"])
        case["q"], case["kv"] = max(1, case["q"] * 3 // 4), max(1, case["kv"] * 3 // 4)
    return case


def _lengths(case):
    """(new, cached) tokens of every sequence: plain functions of the case."""
    n, q, kv = case["seqs"], case["q"], case["kv"]
    if not case["ragged"]:
        return [(q, kv)] * n
    got = [(q, kv)]
    for i in range(1, n):
        k = 1 + int((kv - 1) * (i * PHI % 1.0))
        got.append((min(k, 1 + int((q - 1) * (i * PSI % 1.0))), k))
    if q == kv:                                   # whole prompts: everything in the cache is new
        got = [(k, k) for _, k in got]
    if n > 3:
        got[3] = (0, 0)                           # a slot without a sequence
    return got


# ------------------------------------------------------------------ the cache's layout (include/welvet_cuda.h, WvKvPages)
# A page holds, for each kv head, one block of `page` tokens: K codes, V codes, K scales, V scales and, in 4 bits, a byte for each
# 16 values of K, then of V.
def _layout(case):
    page, hd, bits = case["page"], case["head_dim"], case["bits"]
    code = hd * bits // 8
    k, v = 0, page * code
    ks = 2 * page * code
    vs = ks + 4 * page
    kt = vs + 4 * page
    vt = kt + page * (hd // 16)
    return {"code": code, "k": (k, ks, kt), "v": (v, vs, vt), "block": vs + 4 * page + (2 * page * (hd // 16) if bits == 4 else 0)}


def _row_bytes(case):
    return case["head_dim"] * case["bits"] // 8 + 4 + (case["head_dim"] // 16 if case["bits"] == 4 else 0)


FLT_MIN = 2.0 ** -126


def _quantise(x, bits):
    """x [..., head_dim] float32 -> (codes as bytes, scales, bytes of the groups of 16 or None). One scale for each row."""
    a = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    x = torch.where(fine[..., None], x, torch.zeros_like(x))
    a = torch.where(fine, a, torch.zeros_like(a))
    tile = None
    if bits == 16:
        _, e = torch.frexp(a)                     # a = m 2^e, m in [0.5, 1)
        s = (((e - 15).clamp(min=-126) + 127) << 23).view(torch.float32)            # 2^(e - 15), by its bits
        s = torch.where(a > 0, s, torch.full_like(s, FLT_MIN))
        codes = (x / s[..., None]).to(torch.float16).view(torch.uint8)
    elif bits == 8:
        s = (a / 127).clamp(min=FLT_MIN)
        codes = torch.round(x / s[..., None]).to(torch.int8).view(torch.uint8)
    else:
        s = (a / 1785).clamp(min=FLT_MIN)
        g = x.unflatten(-1, (-1, 16))
        t = torch.ceil(g.abs().amax(-1) / 7 / s[..., None]).clamp(1, 255)
        c = torch.round(g / (s[..., None] * t)[..., None]).clamp(-7, 7).to(torch.int32).flatten(-2) + 8
        codes = (c[..., 0::2] + 16 * c[..., 1::2]).to(torch.uint8)
        tile = t.to(torch.uint8)
    return codes, torch.where(fine, s, torch.full_like(s, math.nan)), tile


def _values(block, case, which, dtype=torch.float32):
    """The values of whole blocks [..., block bytes] -> [..., page, head_dim]."""
    lay = _layout(case)
    page, hd, bits = case["page"], case["head_dim"], case["bits"]
    at, scale_at, tile_at = lay[which]
    codes = block[..., at:at + page * lay["code"]].contiguous()
    scale = block[..., scale_at:scale_at + 4 * page].contiguous().view(torch.float32).to(dtype)
    if bits == 16:
        c = codes.view(torch.float16).to(dtype).unflatten(-1, (page, hd))
    elif bits == 8:
        c = codes.view(torch.int8).to(dtype).unflatten(-1, (page, hd))
    else:
        c = (torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(dtype) - 8).unflatten(-1, (page, hd // 16, 16))
        t = block[..., tile_at:tile_at + page * (hd // 16)].to(dtype).unflatten(-1, (page, hd // 16))
        c = (c * t[..., None]).flatten(-2)
    return c * scale[..., None]


# ------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["kind"] == "sample":
        return _prepare_sample(case, gen)
    rand = lambda *n: torch.randn(*n, device="cuda", generator=gen)  # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, page, hd, kvh = _lengths(case), case["page"], case["head_dim"], case["kv_heads"]
    need = [-(-k // page) for _, k in lens]
    width = max(need)
    num_pages = sum(need) + 3
    order = torch.randperm(num_pages, device="cuda", generator=gen).to(torch.int32)
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    starts = [0]
    for q, _ in lens:
        starts.append(starts[-1] + q)
    total = starts[-1]
    s = {"case": case, "table": table, "q_start": ints(starts), "kv_len": ints([k for _, k in lens]), "total": total, "num_pages": num_pages,
         "pool": torch.zeros(num_pages, kvh, _layout(case)["block"], dtype=torch.uint8, device="cuda")}
    s["q"] = rand(total, case["heads"] * hd)
    if case["kind"] == "cache":
        # keys and values out of the projections: a few channels are far larger than the rest, as in trained models
        far = 1 + 9 * (torch.rand(kvh * hd, device="cuda", generator=gen) > 0.97)
        s["k"], s["v"] = rand(total, kvh * hd) * far, rand(total, kvh * hd)
        s["out"] = {n: torch.zeros_like(s[n]) for n in ("q", "k", "v")}
        return s
    # the cache as earlier steps left it, written in pieces of pages
    lay = _layout(case)
    for p in range(0, num_pages, 4096):
        blocks = s["pool"][p:p + 4096]
        for which in ("k", "v"):
            codes, scale, tile = _quantise(rand(blocks.shape[0], kvh, page, hd), case["bits"])
            b, bs, bt = lay[which]
            blocks[:, :, b:b + page * lay["code"]] = codes.flatten(-2)
            blocks[:, :, bs:bs + 4 * page] = scale.view(torch.uint8)
            if tile is not None:
                blocks[:, :, bt:bt + page * (hd // 16)] = tile.flatten(-2)
    s["out"] = torch.zeros(total, case["heads"] * hd, device="cuda")
    return s


def _prepare_sample(case, gen):
    rows, n = case["rows"], case["vocab"]
    rand = lambda *k: torch.rand(*k, device="cuda", generator=gen)  # noqa: E731
    # a head's logits: some rows sure of their token, others open
    logits = torch.randn(rows, n, device="cuda", generator=gen) * (1 + 3 * rand(rows, 1))
    s = {"case": case, "logits": logits, "u": rand(rows).double(), "index": torch.zeros(rows, dtype=torch.int32, device="cuda"),
         "prob": torch.zeros(rows, device="cuda")}
    if case["mix"]:
        pick = lambda v: torch.tensor(v, device="cuda")[(rand(rows) * len(v)).long()]  # noqa: E731
        s["temperature"], s["top_k"] = pick([0.0, 0.6, 0.8, 1.0, 1.3]), pick([0, 0, 1, 20, 50, 1000]).to(torch.int32)
        s["top_p"], s["min_p"] = pick([0.5, 0.9, 0.95, 1.0, 1.0]), pick([0.0, 0.0, 0.02, 0.1])
    else:
        full = lambda v, t: torch.full((rows,), v, dtype=t, device="cuda")  # noqa: E731
        s["temperature"], s["top_k"] = full(0.8, torch.float32), full(40, torch.int32)
        s["top_p"], s["min_p"] = full(0.95, torch.float32), full(0.0, torch.float32)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _OWN[kind](s, s["case"])
    return _PLAIN[kind](s, s["case"])


def _handles(s, case):
    """The descriptors of the cache and of the batch that a program keeps beside their tensors."""
    if "pages" not in s:
        import welvet_b200 as wv
        from welvet_b200 import paged, sampling
        wv.init(0)
        s["api"] = sampling if case["kind"] == "sample" else paged
        s["pages"] = None
        if case["kind"] != "sample":
            s["pages"] = paged.KVPages(s["pool"].data_ptr(), case["bits"], s["num_pages"], case["page"], case["kv_heads"], case["head_dim"])
            s["batch"] = paged.Batch(s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), case["seqs"], s["table"].shape[1],
                                     s["total"], case["q"], case["kv"])
    return s["api"], torch.cuda.current_stream().cuda_stream


def _own_cache(s, case):
    api, st = _handles(s, case)
    out = s["out"]
    api.KVWriteCUDA(s["pages"], s["batch"], s["k"].data_ptr(), s["v"].data_ptr(), s["q"].data_ptr(), out["q"].data_ptr(), case["heads"], THETA, stream=st)
    api.KVReadCUDA(s["pages"], s["batch"], out["k"].data_ptr(), out["v"].data_ptr(), stream=st)
    return out


def _own_attn(s, case):
    api, st = _handles(s, case)
    api.AttnPagedCUDA(s["pages"], s["batch"], s["q"].data_ptr(), s["out"].data_ptr(), case["heads"], case["head_dim"] ** -0.5, window=case["window"], stream=st)
    return s["out"]


def _own_sample(s, case):
    api, st = _handles(s, case)
    api.SampleRowsCUDA(s["logits"].data_ptr(), case["rows"], case["vocab"], s["temperature"].data_ptr(), s["top_k"].data_ptr(), s["top_p"].data_ptr(),
                       s["min_p"].data_ptr(), s["u"].data_ptr(), s["index"].data_ptr(), s["prob"].data_ptr(), stream=st)
    return {"index": s["index"], "prob": s["prob"]}


_OWN = {"cache": _own_cache, "attn": _own_attn, "sample": _own_sample}


def _places(s, case, dtype=torch.long):
    """(sequence, position) of every new token's row."""
    rows = torch.arange(s["total"], device="cuda")
    start, kv = s["q_start"].to(dtype), s["kv_len"].to(dtype)
    seq = torch.searchsorted(start[1:].contiguous(), rows, right=True)
    return seq, kv[seq] - (start[seq + 1] - rows)


def _rope(x, pos, heads, hd):
    """The framework's rotation: angles, their sine and the sums in 64 bits (an angle of a late position has few good digits in 32),
    rounded once."""
    half = hd // 2
    d = torch.arange(half, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] / torch.pow(torch.tensor(THETA, dtype=torch.float64, device="cuda"), 2 * d / hd)
    c, si = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    x = x.double().unflatten(-1, (heads, hd))
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * c - b * si, a * si + b * c), -1)


def _plain_cache(s, case):
    hd, kvh, page, lay = case["head_dim"], case["kv_heads"], case["page"], _layout(case)
    seq, pos = _places(s, case)
    q = _rope(s["q"], pos, case["heads"], hd).float().flatten(-2)
    k = _rope(s["k"], pos, kvh, hd).float()
    at, slot = s["table"][seq, pos // page].long(), pos % page
    pool = s["pool"]
    codes = pool[:, :, :2 * page * lay["code"]].unflatten(-1, (2, page, lay["code"]))
    for n, (which, x) in enumerate((("k", k), ("v", s["v"].unflatten(-1, (kvh, hd))))):
        c, scale, tile = _quantise(x, case["bits"])
        codes[at, :, n, slot] = c
        pool[:, :, lay[which][1]:lay[which][1] + 4 * page].unflatten(-1, (page, 4))[at, :, slot] = scale.contiguous().view(torch.uint8).unflatten(-1, (kvh, 4))
        if tile is not None:
            pool[:, :, lay[which][2]:lay[which][2] + page * (hd // 16)].unflatten(-1, (page, hd // 16))[at, :, slot] = tile
    back = []
    for n, which in enumerate(("k", "v")):
        c = codes[at, :, n, slot].contiguous()
        scale = pool[:, :, lay[which][1]:lay[which][1] + 4 * page].unflatten(-1, (page, 4))[at, :, slot].contiguous().view(torch.float32)
        if case["bits"] == 16:
            c = c.view(torch.float16).float()
        elif case["bits"] == 8:
            c = c.view(torch.int8).float()
        else:
            t = pool[:, :, lay[which][2]:lay[which][2] + page * (hd // 16)].unflatten(-1, (page, hd // 16))[at, :, slot].float()
            c = torch.stack((c & 15, c >> 4), -1).flatten(-2).float() - 8
            c = (c.unflatten(-1, (-1, 16)) * t[..., None]).flatten(-2)
        back.append((c * scale).flatten(-2))
    return {"q": q, "k": back[0], "v": back[1]}


def _plain_attn(s, case):
    hd, kvh, group = case["head_dim"], case["kv_heads"], case["heads"] // case["kv_heads"]
    most = case["q"]
    start, kv = s["q_start"].long(), s["kv_len"].long()
    tok = torch.arange(most, device="cuda")
    live = tok < (start[1:] - start[:-1])[:, None]                                       # [seqs, q]
    row = torch.where(live, start[:-1, None] + tok, torch.full_like(tok, s["total"]))   # rows that are none: one past the end
    pos = kv[:, None] - (start[1:] - start[:-1])[:, None] + tok
    q = torch.cat((s["q"], s["q"].new_zeros(1, s["q"].shape[1])))[row].unflatten(-1, (kvh, group, hd)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    block = s["pool"][s["table"].long().clamp(min=0)]                                    # [seqs, pages, kv heads, bytes]
    k, v = (_values(block, case, which).permute(0, 2, 1, 3, 4).flatten(2, 3) for which in ("k", "v"))
    at = torch.arange(k.shape[2], device="cuda")
    seen = (at <= pos[..., None]) & (at < kv[:, None, None])
    if case["window"]:
        seen &= at > pos[..., None] - case["window"]
    seen = seen[:, None, None]
    x = torch.matmul(q, k.transpose(2, 3)).mul_(hd ** -0.5).unflatten(2, (group, most))   # [seqs, kv heads, group, q, kv]
    x = torch.where(seen, x, torch.full_like(x[:1, :1, :1, :1, :1], -math.inf))
    x = x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    v = torch.where((at < kv[:, None])[:, None, :, None], v, torch.zeros_like(v[:1, :1, :1]))
    o = torch.matmul(x.flatten(2, 3), v).unflatten(2, (group, most)) / torch.where(total > 0, total, torch.ones_like(total))
    out = s["q"].new_zeros(s["total"] + 1, case["heads"] * hd)
    out[row] = o.permute(0, 3, 1, 2, 4).flatten(2)
    return out[:-1]


def _plain_sample(s, case):
    """Weights in 32 bits; their running sums in 64, since the index that comes of them has to be the same."""
    x, n = s["logits"], case["vocab"]
    t = s["temperature"][:, None]
    greedy = (t <= 0) | (s["top_k"][:, None] == 1)
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    y = torch.where(greedy, x, x / torch.where(t > 0, t, torch.ones_like(t)))
    y, order = torch.sort(y, dim=-1, descending=True, stable=True)
    place = torch.arange(n, device="cuda")
    k = s["top_k"][:, None].long()
    k = torch.where(greedy, torch.ones_like(k), torch.where(k <= 0, torch.full_like(k, n), k))
    w = torch.where(y == y[:, :1], torch.ones_like(y), torch.exp(y - y[:, :1]))
    w = torch.where((place < k) & (y > -math.inf), w, torch.zeros_like(w)).double()
    run_ = w.cumsum(-1)
    keep = (run_ - w < s["top_p"][:, None].double() * run_[:, -1:]) & (w >= s["min_p"][:, None].double())
    keep[:, 0] = True
    w = torch.where(keep, w, torch.zeros_like(w))
    run_ = w.cumsum(-1)
    at = (run_ >= s["u"][:, None] * run_[:, -1:]).to(torch.uint8).argmax(-1, keepdim=True)
    some = run_[:, -1:] > 0
    index = torch.where(some, order.gather(1, at), torch.full_like(at, -1)).squeeze(1).to(torch.int32)
    prob = torch.where(some, w.gather(1, at) / run_[:, -1:], torch.zeros_like(run_[:, -1:])).squeeze(1).float()
    return {"index": index, "prob": prob}


_PLAIN = {"cache": _plain_cache, "attn": _plain_attn, "sample": _plain_sample}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 32), "flops": 4 * case["rows"] * case["vocab"]}
    lens, hd, kvh = _lengths(case), case["head_dim"], case["kv_heads"]
    new = sum(q for q, _ in lens)
    row = 2 * kvh * _row_bytes(case)                                                    # a token's K and V in the cache
    if case["kind"] == "cache":
        return {"bytes": new * (2 * 4 * case["heads"] * hd + 4 * 4 * kvh * hd + 2 * row), "flops": 6 * new * (case["heads"] + kvh) * hd}
    pairs = touched = 0
    for q, kv in lens:
        w = case["window"] or kv
        p0 = kv - q                                                                     # the first new token's position
        full = max(0, min(q, kv - max(p0, w - 1)))                                      # tokens that see a whole window
        part = q - full                                                                 # the others see everything before them
        pairs += full * w + part * p0 + part * (part + 1) // 2
        touched += min(kv, q + w - 1) if q else 0
    return {"bytes": 8 * new * case["heads"] * hd + touched * row, "flops": 4 * pairs * case["heads"] * hd}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"cache": _exact_cache, "attn": _exact_attn, "sample": _exact_sample}[case["kind"]](s, case)


def _exact_cache(s, case):
    hd, bits, at = case["head_dim"], case["bits"], 0
    out = {n: torch.empty_like(s[n], dtype=torch.float64) for n in ("q", "k", "v")}
    freq = THETA ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    for q, kv in _lengths(case):
        turn = torch.outer(torch.arange(kv - q, kv, device="cuda", dtype=torch.float64), freq)
        turn = torch.polar(torch.ones_like(turn), turn)[:, None]
        for n in ("q", "k", "v"):
            heads = case["heads"] if n == "q" else case["kv_heads"]
            x = s[n][at:at + q].double().reshape(q, heads, hd)
            if n != "v":
                z = torch.complex(x[..., :hd // 2], x[..., hd // 2:]) * turn
                x = torch.cat((z.real, z.imag), -1)
            if n != "q":
                top = x.abs().amax(-1, keepdim=True)
                if bits == 16:
                    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=1e-300))) - 10)         # 11 significant bits
                    step = torch.maximum(step, torch.exp2(torch.floor(torch.log2(top)) - 14 - 24))     # the smallest steps of the row
                    x = torch.round(x / step) * step
                elif bits == 8:
                    x = torch.round(x * 127 / top) * top / 127
                else:
                    g = x.reshape(q, heads, hd // 16, 16)
                    unit = top[..., None] / 1785
                    step = unit * torch.ceil(g.abs().amax(-1, keepdim=True) / 7 / unit).clamp(1, 255)
                    x = (torch.round(g / step).clamp(-7, 7) * step).reshape(q, heads, hd)
            out[n][at:at + q] = x.reshape(q, heads * hd)
        at += q
    return out


def _exact_attn(s, case):
    hd, kvh, group, page = case["head_dim"], case["kv_heads"], case["heads"] // case["kv_heads"], case["page"]
    out, at = torch.zeros(s["total"], kvh, group, hd, dtype=torch.float64, device="cuda"), 0
    for i, (q, kv) in enumerate(_lengths(case)):
        if not q:
            continue
        blocks = s["pool"][s["table"][i, :-(-kv // page)].long()]
        for h in range(kvh):
            k, v = (_values(blocks[:, h], case, which, torch.float64).reshape(-1, hd)[:kv] for which in ("k", "v"))
            for t in range(0, q, 512):                                                   # 512 tokens at a time
                u = min(q, t + 512)
                last = kv - q + u
                first = max(0, kv - q + t - case["window"] + 1) if case["window"] else 0
                x = s["q"][at + t:at + u].double().reshape(u - t, kvh, group, hd)[:, h]
                x = torch.einsum("tgd,kd->tgk", x, k[first:last]) / math.sqrt(hd)
                far = torch.arange(kv - q + t, last, device="cuda")[:, None] - torch.arange(first, last, device="cuda")
                hidden = far < 0
                if case["window"]:
                    hidden |= far >= case["window"]
                p = torch.softmax(x.masked_fill(hidden[:, None], -math.inf), -1)
                out[at + t:at + u, h] = torch.einsum("tgk,kd->tgd", p, v[first:last])
        at += q
    return out.reshape(s["total"], -1)


def _exact_sample(s, case):
    """The probabilities; whole numbers have no other value in 64 bits."""
    prob = torch.zeros(case["rows"], dtype=torch.float64, device="cuda")
    for r in range(case["rows"]):
        t, k = float(s["temperature"][r]), int(s["top_k"][r])
        if t <= 0 or k == 1:
            prob[r] = 1.0
            continue
        p = torch.softmax(torch.sort(s["logits"][r], descending=True, stable=True).values.double() / t, 0)
        if k > 0:
            p = p[:k] / p[:k].sum()
        c = p.cumsum(0)
        keep = (c - p < float(s["top_p"][r])) & (p >= float(s["min_p"][r]) * p[0])
        keep[0] = True
        p = p[keep] / p[keep].sum()
        at = int(torch.searchsorted(p.cumsum(0), s["u"][r:r + 1]).clamp(max=p.numel() - 1))
        prob[r] = p[at]
    return {"index": None, "prob": prob}
