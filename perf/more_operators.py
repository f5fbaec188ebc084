"""More operators of batched serving, as cases: the pages of a cache (fork, extend, trim, compact), the attention of sequences that
share a long prefix, and the low-rank adapters of many requests beside a shared projection.

A case is a dict of plain values; `kind` names the operator:

  pages     sequences' pages as device-side tables (`paged.KVTable`): form "fork" frees the forks of the last pass, forks `seqs`
            sequences `copies` times and extends the forks by `add` tokens (their last, shared pages are copied); "step" trims what a step took
            and was not kept, and extends every sequence by up to `add` tokens; "compact" moves the pages of a scattered pool to its front
  shared    attention of the new tokens of `groups` groups of `seqs` sequences each, whose first `shared` tokens are the same pages
            (`paged.AttnSharedCUDA`): causal, grouped-query heads
  adapter   y = base + scale B (A x) for rows of different adapters, one to four projections on the same x (`adapters.ApplyCUDA`)

`run` makes the framework's calls where `own` is set; otherwise it computes the same with elementary torch operations. `exact` is
the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

PHI, PSI = 0.6180339887498949, 0.7548776662466927


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one chat forked into four continuations that each get a token: one shared, partly filled page is copied for each of them, in 32 blocks
        {"name": "pages_fork", "kind": "pages", "form": "fork", "seqs": 1, "copies": 4, "add": 1, "kv": 2049, "bits": 8, "kv_heads": 8, "head_dim": 128, "page": 64, "blocks": 32},
        # a server's step of drafted tokens: 200 sequences give back what was not kept and take room for up to five tokens each
        {"name": "pages_step", "kind": "pages", "form": "step", "seqs": 200, "copies": 0, "add": 5, "kv": 1500, "bits": 4, "kv_heads": 8, "head_dim": 128, "page": 16, "blocks": 1},
        # a pool that is half empty after its sequences came and went, moved to the front so that the rest can be given back
        {"name": "pages_compact", "kind": "pages", "form": "compact", "seqs": 24, "copies": 0, "add": 0, "kv": 6000, "bits": 8, "kv_heads": 8, "head_dim": 128, "page": 64, "blocks": 4},
        # eight users of one instruction of 2048 tokens, a token each
        {"name": "shared_chat", "kind": "shared", "groups": 1, "seqs": 8, "q": 1, "shared": 2048, "own": 400, "bits": 16, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "ragged": True},
        # a server's step: 64 questions about one long document
        {"name": "shared_batch", "kind": "shared", "groups": 1, "seqs": 64, "q": 1, "shared": 16384, "own": 1000, "bits": 8, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "ragged": True},
        # two documents of different users, 70B-shaped heads, 4 bits
        {"name": "shared_long", "kind": "shared", "groups": 2, "seqs": 16, "q": 1, "shared": 65000, "own": 300, "bits": 4, "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 16, "ragged": True},
        # drafted tokens of four groups checked together: four a sequence, small heads, a page size that is no power of two
        {"name": "shared_draft", "kind": "shared", "groups": 4, "seqs": 6, "q": 4, "shared": 6000, "own": 700, "bits": 16, "heads": 16, "kv_heads": 4, "head_dim": 64, "page": 48, "ragged": False},
        # one user's token, one adapter of rank 16 beside Q, K and V of an 8B-shaped block
        {"name": "adapter_one", "kind": "adapter", "rows": 1, "slots": 8, "rank": 16, "in": 4096, "outs": "4096,1024,1024", "dtype": "bf16", "mix": "few"},
        # a server's step: 64 tokens of 32 requests' adapters beside Q, K and V
        {"name": "adapter_batch", "kind": "adapter", "rows": 64, "slots": 32, "rank": 16, "in": 4096, "outs": "4096,1024,1024", "dtype": "bf16", "mix": "many"},
        # the same beside gate and up, rank 64 in f16, some of the rows without an adapter
        {"name": "adapter_ffn", "kind": "adapter", "rows": 48, "slots": 16, "rank": 64, "in": 4096, "outs": "14336,14336", "dtype": "f16", "mix": "many"},
        # prompts of a few requests, 2048 tokens in all, beside the O projection
        {"name": "adapter_prompt", "kind": "adapter", "rows": 2048, "slots": 6, "rank": 64, "in": 4096, "outs": "4096", "dtype": "bf16", "mix": "few"},
        # float32 adapters of odd ranks as they come from training, an odd number of rows, beside the down projection
        {"name": "adapter_f32", "kind": "adapter", "rows": 333, "slots": 9, "rank": 24, "in": 14336, "outs": "4096", "dtype": "f32", "mix": "few"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["pages", "shared", "shared", "adapter", "adapter"])
    if kind == "adapter":
        case = {"kind": kind, "rows": _log(rng, 1, 2048), "slots": _log(rng, 1, 64), "rank": 8 * rng.randint(1, 8), "in": 8 * _log(rng, 64, 1792),
                "outs": ",".join(str(_log(rng, 500, 14336)) for _ in range(rng.randint(1, 3))), "dtype": rng.choice(("bf16", "bf16", "f16", "f32")),
                "mix": rng.choice(("few", "many"))}
        while work(case)["flops"] > 2.2e9 or work(case)["bytes"] > 1.2e8:
            case["rows"], case["slots"] = max(1, case["rows"] * 2 // 3), max(1, case["slots"] * 4 // 5)
        return case
    kv_heads = rng.choice((1, 2, 4, 8))
    case = {"kind": kind, "bits": rng.choice((16, 8, 4)), "kv_heads": kv_heads, "head_dim": rng.choice((64, 64, 80, 128, 128, 128)), "page": rng.choice((16, 32, 48, 64, 128))}
    if kind == "pages":
        case["form"] = rng.choice(("fork", "fork", "step", "compact"))
        case |= {"seqs": _log(rng, 1, 24 if case["form"] == "fork" else 250), "copies": rng.randint(1, 8) if case["form"] == "fork" else 0,
                 "add": rng.randint(1, 40) if case["form"] != "compact" else 0, "kv": _log(rng, 20, 6000), "blocks": rng.randint(1, 16)}
        while _page_lens(case)[2] * case["page"] * 2 * case["kv_heads"] * _row_bytes(case) * case["blocks"] > 1.2e9 or work(case)["bytes"] > 6e8:
            case["seqs"], case["kv"], case["blocks"] = max(1, case["seqs"] * 4 // 5), max(20, case["kv"] * 4 // 5), max(1, case["blocks"] * 4 // 5)
        return case
    case |= {"groups": rng.randint(1, 4), "seqs": _log(rng, 2, 64), "q": rng.choice((1, 1, 1, 2, 4, 7)), "shared": _log(rng, 200, 66000), "own": _log(rng, 8, 1200),
             "heads": kv_heads * rng.choice((1, 2, 3, 4, 8)), "ragged": rng.random() < 0.6}
    while work(case)["flops"] > 6.5e10 or work(case)["bytes"] > 1.6e8:
        case["shared"], case["own"], case["seqs"] = max(200, case["shared"] * 3 // 4), max(8, case["own"] * 3 // 4), max(2, case["seqs"] * 3 // 4)
    return case


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


def _spread(n, most, step):
    """n lengths from 1 to `most`, spread evenly but in no order; the first is `most`."""
    return [most if i == 0 else 1 + int((most - 1) * (i * step % 1.0)) for i in range(n)]


# ------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"pages": _prepare_pages, "shared": _prepare_shared, "adapter": _prepare_adapter}[case["kind"]](case, gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _page_lens(case):
    """(cached tokens of every sequence, slots of the table, pages of the pool)."""
    lens = _spread(case["seqs"], case["kv"], PHI)
    page, form = case["page"], case["form"]
    held = sum(-(-n // page) for n in lens)
    if form == "fork":
        return lens, case["seqs"] * (1 + case["copies"]), held + case["seqs"] * case["copies"] * (1 + -(-case["add"] // page)) + 5
    if form == "step":
        return lens, case["seqs"], held + case["seqs"] * (1 + -(-case["add"] // page)) + 5
    return lens, case["seqs"], 2 * held + 7


def _prepare_pages(case, gen):
    lens, slots, num_pages = _page_lens(case)
    page = case["page"]
    width = -(-(case["kv"] + case["add"]) // page)
    order = torch.randperm(num_pages, device="cuda", generator=gen).to(torch.int32)      # a pool after some time: pages in no order
    pages, refs, at = torch.full((slots, width), -1, dtype=torch.int32, device="cuda"), torch.zeros(num_pages, dtype=torch.int32, device="cuda"), 0
    for i, n in enumerate(lens):
        k = -(-n // page)
        pages[i, :k] = order[at:at + k]
        at += k
    refs[order[:at].long()] = 1
    size = case["kv_heads"] * _layout(case)["block"]
    pools = [torch.randint(-2 ** 63, 2 ** 63 - 1, (num_pages, size // 8), dtype=torch.int64, device="cuda", generator=gen).view(torch.uint8) for _ in range(case["blocks"])]
    s = {"case": case, "pages": pages, "refs": refs, "kv_len": _ints(lens + [0] * (slots - len(lens))), "pools": pools, "slots": slots, "num_pages": num_pages}
    if case["form"] == "fork":
        n, c = case["seqs"], case["copies"]
        s["src"], s["dst"] = _ints([i // c for i in range(n * c)]), _ints([n + i for i in range(n * c)])
        s["keep"] = _ints([0] * (n * c))
        s["add"] = _ints([0] * n + [case["add"]] * (n * c))
    elif case["form"] == "step":
        s["keep"], s["add"] = s["kv_len"].clone(), _ints(_spread(slots, case["add"], PSI))
    else:
        s["pages0"], s["refs0"], s["live"] = pages.clone(), refs.clone(), _ints([0])
    s["granted"] = torch.zeros(slots, dtype=torch.int32, device="cuda")
    return s


def _shared_lens(case):
    """For every sequence of a group (new tokens, own cached tokens, the new ones among them)."""
    n, q, most = case["seqs"], case["q"], max(case["own"], case["q"])
    if not case["ragged"]:
        return [(q, most)] * n
    got = [(min(q, k), k) for k in _spread(n, most, PHI)]
    if n > 3:
        got[3] = (0, 0)                               # a slot without a sequence
    return got


def _prepare_shared(case, gen):
    rand = lambda *n: torch.randn(*n, device="cuda", generator=gen)  # noqa: E731
    page, hd, kvh, lens = case["page"], case["head_dim"], case["kv_heads"], _shared_lens(case)
    common = case["shared"] // page                   # whole pages; the rest of the prefix is every sequence's own
    kv = [case["shared"] + k if k else 0 for _, k in lens]
    width = -(-max(kv) // page)
    need = case["groups"] * (common + sum(-(-k // page) - common for k in kv if k))
    num_pages = need + 3
    order = torch.randperm(num_pages, device="cuda", generator=gen).to(torch.int32)
    table, at, starts = torch.full((case["groups"] * len(lens), width), -1, dtype=torch.int32, device="cuda"), 0, [0]
    for g in range(case["groups"]):
        front, at = order[at:at + common], at + common
        for i, ((q, _), k) in enumerate(zip(lens, kv)):
            starts.append(starts[-1] + q)
            if k:
                row, n = table[g * len(lens) + i], -(-k // page) - common
                row[:common] = front
                row[common:common + n] = order[at:at + n]
                at += n
    total = starts[-1]
    lay = _layout(case)
    pool = torch.zeros(num_pages, kvh, lay["block"], dtype=torch.uint8, device="cuda")
    for p in range(0, num_pages, 4096):               # the cache as earlier steps left it
        blocks = pool[p:p + 4096]
        for which in ("k", "v"):
            codes, scale, tile = _quantise(rand(blocks.shape[0], kvh, page, hd), case["bits"])
            b, bs, bt = lay[which]
            blocks[:, :, b:b + page * lay["code"]] = codes.flatten(-2)
            blocks[:, :, bs:bs + 4 * page] = scale.view(torch.uint8)
            if tile is not None:
                blocks[:, :, bt:bt + page * (hd // 16)] = tile.flatten(-2)
    return {"case": case, "pool": pool, "table": table, "num_pages": num_pages, "q_start": _ints(starts), "kv_len": _ints(kv * case["groups"]), "total": total,
            "max_kv": max(kv), "start": _ints([g * len(lens) for g in range(case["groups"] + 1)]), "shared": _ints([case["shared"]] * case["groups"]),
            "q": rand(total, case["heads"] * hd), "out": torch.zeros(total, case["heads"] * hd, device="cuda")}


def _quantise(x, bits):
    """x [..., head_dim] float32, finite and not all zero -> (codes as bytes, scales, bytes of the groups of 16 or None)."""
    a, tile = x.abs().amax(-1), None
    if bits == 16:
        s = torch.exp2(torch.frexp(a)[1].float() - 15)
        codes = (x / s[..., None]).to(torch.float16).view(torch.uint8)
    elif bits == 8:
        s = a / 127
        codes = torch.round(x / s[..., None]).to(torch.int8).view(torch.uint8)
    else:
        s = a / 1785
        g = x.unflatten(-1, (-1, 16))
        t = torch.ceil(g.abs().amax(-1) / 7 / s[..., None]).clamp(1, 255)
        c = torch.round(g / (s[..., None] * t)[..., None]).clamp(-7, 7).to(torch.int32).flatten(-2) + 8
        codes = (c[..., 0::2] + 16 * c[..., 1::2]).to(torch.uint8)
        tile = t.to(torch.uint8)
    return codes, s, tile


_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _outs(case):
    return [int(v) for v in case["outs"].split(",")]


def _slots_of(case):
    """The adapter of every row: "many": neighbours differ, and every eleventh row has none; "few": runs of rows, as prompts have."""
    rows, n = case["rows"], case["slots"]
    if case["mix"] == "many":
        return [-1 if i % 11 == 7 else int(n * ((i + 1) * PHI % 1.0)) for i in range(rows)]
    return [int(n * (i / rows)) for i in range(rows)]


def _prepare_adapter(case, gen):
    rand = lambda *n: torch.randn(*n, device="cuda", generator=gen)  # noqa: E731
    t, n, r, k = _TYPES[case["dtype"]], case["slots"], case["rank"], case["in"]
    ranks = [r if i % 3 else max(1, r - 5) for i in range(n)]                  # some adapters have fewer; what is left is zeros
    on = torch.arange(r, device="cuda") < torch.tensor(ranks, device="cuda")[:, None]
    s = {"case": case, "rank": _ints(ranks), "slot": _ints(_slots_of(case)), "x": rand(case["rows"], k), "targets": []}
    for out in _outs(case):
        s["targets"].append({"out": out, "a": (rand(n, r, k) * k ** -0.5 * on[..., None]).to(t), "b": (rand(n, out, r) * 0.3 * on[:, None]).to(t), "scale": 0.5 + torch.rand(n, device="cuda", generator=gen),
                             "base": rand(case["rows"], -(-out // 4) * 4), "y": torch.zeros(case["rows"], -(-out // 4) * 4, device="cuda")})
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        return _OWN[kind](s, s["case"])
    return _PLAIN[kind](s, s["case"])


def _handles(s, case):
    """The descriptors that a program keeps beside their tensors."""
    if "api" not in s:
        import welvet_b200 as wv
        from welvet_b200 import adapters, paged
        wv.init(0)
        if case["kind"] == "adapter":
            code = {"f32": 1, "f16": 2, "bf16": 3}[case["dtype"]]
            s["plan"] = torch.zeros(adapters.PlanBytes(case["rows"], case["slots"]), dtype=torch.uint8, device="cuda")
            s["call"] = adapters.Group([adapters.Adapters(t["a"].data_ptr(), t["b"].data_ptr(), s["rank"].data_ptr(), t["scale"].data_ptr(), case["slots"], case["rank"],
                                                          case["in"], t["out"], code) for t in s["targets"]])
            s["api"] = adapters
            return s["api"], torch.cuda.current_stream().cuda_stream
        if case["kind"] == "pages":
            s["blocks"] = paged.KVBlocks([paged.KVPages(p.data_ptr(), case["bits"], s["num_pages"], case["page"], case["kv_heads"], case["head_dim"]) for p in s["pools"]])
            s["t"] = paged.KVTable(s["refs"].data_ptr(), s["pages"].data_ptr(), s["kv_len"].data_ptr(), s["num_pages"], case["page"], s["slots"], s["pages"].shape[1])
        else:
            s["p"] = paged.KVPages(s["pool"].data_ptr(), case["bits"], s["num_pages"], case["page"], case["kv_heads"], case["head_dim"])
            s["b"] = paged.Batch(s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), case["groups"] * case["seqs"], s["table"].shape[1], s["total"],
                                 case["q"], s["max_kv"])
            s["g"] = paged.Groups(s["start"].data_ptr(), s["shared"].data_ptr(), case["groups"], case["shared"])
        s["api"] = paged
    return s["api"], torch.cuda.current_stream().cuda_stream


def _own_pages(s, case):
    api, st = _handles(s, case)
    if case["form"] == "compact":
        s["pages"].copy_(s["pages0"])                 # the sources of a move are left as they are: the same pool can be compacted again
        s["refs"].copy_(s["refs0"])
        api.KVCompactCUDA(s["t"], s["blocks"], s["live"].data_ptr(), stream=st)
        return {"pages": s["pages"], "refs": s["refs"], "live": s["live"], "pools": s["pools"]}
    if case["form"] == "fork":
        n = s["dst"].numel()
        api.KVTrimCUDA(s["t"], n, s["keep"].data_ptr(), s["dst"].data_ptr(), stream=st)
        api.KVForkCUDA(s["t"], s["src"].data_ptr(), s["dst"].data_ptr(), n, stream=st)
    else:
        api.KVTrimCUDA(s["t"], s["slots"], s["keep"].data_ptr(), stream=st)
    api.KVExtendCUDA(s["t"], s["add"].data_ptr(), s["granted"].data_ptr(), s["blocks"], stream=st)
    return {"pages": s["pages"], "refs": s["refs"], "kv_len": s["kv_len"], "granted": s["granted"], "pools": s["pools"]}


def _own_shared(s, case):
    api, st = _handles(s, case)
    api.AttnSharedCUDA(s["p"], s["b"], s["g"], s["q"].data_ptr(), s["out"].data_ptr(), case["heads"], case["head_dim"] ** -0.5, stream=st)
    return s["out"]


def _own_adapter(s, case):
    api, st = _handles(s, case)
    api.PlanCUDA(s["slot"].data_ptr(), case["rows"], case["slots"], s["plan"].data_ptr(), stream=st)
    api.ApplyCUDA(s["call"], s["plan"].data_ptr(), case["rows"], s["x"].data_ptr(), [t["y"].data_ptr() for t in s["targets"]], [t["base"].data_ptr() for t in s["targets"]],
                  ldy=[t["y"].shape[1] for t in s["targets"]], stream=st)
    return [t["y"][:, :t["out"]] for t in s["targets"]]


_OWN = {"pages": _own_pages, "shared": _own_shared, "adapter": _own_adapter}


def _trim(s, case, rows, keep):
    pages, refs, kv = s["pages"], s["refs"], s["kv_len"]
    at = torch.arange(pages.shape[1], device="cuda")
    new = torch.minimum(kv[rows], keep)
    held, left = (-(-n // case["page"]) for n in (kv[rows], new))
    gone = (at >= left[:, None]) & (at < held[:, None])
    ids = pages[rows].long()
    refs.scatter_add_(0, torch.where(gone, ids, torch.zeros_like(ids)).flatten(), -gone.flatten().int())
    pages[rows] = torch.where(gone, torch.full_like(pages[:1, :1], -1), pages[rows])
    kv[rows] = new


def _plain_pages(s, case):
    pages, refs, kv, page = s["pages"], s["refs"], s["kv_len"], case["page"]
    at = torch.arange(pages.shape[1], device="cuda")
    if case["form"] == "compact":
        pages.copy_(s["pages0"])
        refs.copy_(s["refs0"])
        live = refs > 0
        count = live.sum()
        front = torch.arange(refs.numel(), device="cuda") < count
        src, dst = (live & ~front).nonzero().squeeze(1), (~live & front).nonzero().squeeze(1)
        to = torch.arange(refs.numel(), device="cuda", dtype=torch.int32)
        to[src] = dst.int()
        pages.copy_(torch.where(at < (-(-kv // page))[:, None], to[pages.clamp(min=0).long()], pages))
        refs[dst], refs[src] = refs[src], 0
        [p.index_copy_(0, dst, p[src]) for p in s["pools"]]
        s["live"].copy_(count)
        return {"pages": pages, "refs": refs, "live": s["live"], "pools": s["pools"]}
    if case["form"] == "fork":
        src, dst = s["src"].long(), s["dst"].long()
        _trim(s, case, dst, s["keep"])
        held = at < (-(-kv[src] // page))[:, None]
        ids = pages[src].long()
        refs.scatter_add_(0, torch.where(held, ids, torch.zeros_like(ids)).flatten(), held.flatten().int())
        pages[dst] = torch.where(held, pages[src], torch.full_like(pages[:1, :1], -1))
        kv[dst] = kv[src]
    else:
        _trim(s, case, torch.arange(s["slots"], device="cuda"), s["keep"])
    add = s["add"]
    held, want = -(-kv // page), -(-(kv + add) // page)
    last = (held - 1).clamp(min=0).long()[:, None]
    old = pages.gather(1, last).squeeze(1).clamp(min=0).long()
    part = (add > 0) & (kv % page != 0) & (refs[old] > 1)                     # a shared page that is partly filled: a copy of it
    need = torch.where(add > 0, want - held, torch.zeros_like(held)) + part.int()
    fits = want <= pages.shape[1]
    ok = ((torch.where(fits, need, torch.zeros_like(need)).cumsum(0) <= (refs == 0).sum()) | (need == 0)) & fits
    part &= ok
    new = ok[:, None] & (((at >= held[:, None]) & (at < want[:, None])) | (part[:, None] & (at == held[:, None] - 1)))
    empty = torch.argsort((refs > 0).to(torch.uint8), stable=True).to(torch.int32)        # the free pages first, in rising order
    fresh = empty[(new.flatten().cumsum(0) - 1).clamp(min=0)].reshape(new.shape)
    refs.scatter_add_(0, torch.where(part, old, torch.zeros_like(old)), -part.int())
    refs.scatter_add_(0, torch.where(new, fresh, torch.zeros_like(fresh)).long().flatten(), new.flatten().int())
    pages.copy_(torch.where(new, fresh, pages))
    kv += torch.where(ok, add, torch.zeros_like(add))
    s["granted"].copy_(ok)
    rows = part.nonzero().squeeze(1)
    frm, to = old[rows], pages.gather(1, last).squeeze(1).long()[rows]
    [p.index_copy_(0, to, p[frm]) for p in s["pools"]]
    return {"pages": pages, "refs": refs, "kv_len": kv, "granted": s["granted"], "pools": s["pools"]}


def _plain_shared(s, case):
    hd, kvh, page, n, groups = case["head_dim"], case["kv_heads"], case["page"], case["seqs"], case["groups"]
    group, most, common = case["heads"] // kvh, case["q"], case["shared"] // page
    start, kv = s["q_start"].long(), s["kv_len"].long()
    tok = torch.arange(most, device="cuda")
    live = tok < (start[1:] - start[:-1])[:, None]                                       # [seqs, q]
    row = torch.where(live, start[:-1, None] + tok, torch.full_like(tok, s["total"]))   # rows that are none: one past the end
    pos = kv[:, None] - (start[1:] - start[:-1])[:, None] + tok
    q = torch.cat((s["q"], s["q"].new_zeros(1, s["q"].shape[1])))[row].unflatten(-1, (kvh, group, hd))      # [seqs, q, kv heads, group, hd]
    # the prefix once for a group's rows
    front = s["pool"][s["table"][::n, :common].long().clamp(min=0)]                      # [groups, pages, kv heads, bytes]
    k, v = (_values(front, case, which).permute(0, 2, 1, 3, 4).flatten(2, 3) for which in ("k", "v"))
    qg = q.unflatten(0, (groups, n)).permute(0, 3, 1, 2, 4, 5).flatten(2, 4)             # [groups, kv heads, rows, hd]
    x0 = torch.matmul(qg, k.transpose(2, 3)).mul_(hd ** -0.5)
    # every sequence's own pages
    own_ = s["pool"][s["table"][:, common:].long().clamp(min=0)]
    ko, vo = (_values(own_, case, which).permute(0, 2, 1, 3, 4).flatten(2, 3) for which in ("k", "v"))      # [seqs, kv heads, own, hd]
    at = torch.arange(ko.shape[2], device="cuda") + common * page
    x1 = torch.matmul(q.permute(0, 2, 1, 3, 4).flatten(2, 3), ko.transpose(2, 3)).mul_(hd ** -0.5)          # [seqs, kv heads, q * group, own]
    seen = (at <= pos[..., None])[:, None, :, None, :]
    x1 = torch.where(seen, x1.unflatten(2, (most, group)), torch.full_like(x1[:1, :1, :1, :1, None], -math.inf))
    x1 = x1.unflatten(0, (groups, n)).permute(0, 2, 1, 3, 4, 5).flatten(2, 4)            # [groups, kv heads, rows, own]
    m = torch.maximum(x0.amax(-1, keepdim=True), x1.amax(-1, keepdim=True)).clamp(min=-3e38)
    x0, x1 = x0.sub_(m).exp_(), x1.sub_(m).exp_()
    total = x0.sum(-1, keepdim=True) + x1.sum(-1, keepdim=True)
    vo = torch.where((at < kv[:, None])[:, None, :, None], vo, torch.zeros_like(vo[:1, :1, :1]))
    x1 = x1.unflatten(2, (n, most * group)).permute(0, 2, 1, 3, 4).flatten(0, 1)
    o = torch.matmul(x1, vo).unflatten(0, (groups, n)).permute(0, 2, 1, 3, 4).flatten(2, 3) + torch.matmul(x0, v)
    o = (o / total).unflatten(2, (n, most, group)).permute(0, 2, 3, 1, 4, 5).flatten(0, 1).flatten(2)       # [seqs, q, heads * hd]
    out = s["q"].new_zeros(s["total"] + 1, case["heads"] * hd)
    out[row] = o
    return out[:-1]


def _plain_adapter(s, case):
    """All adapters on all rows, the others' results struck out: two large products a target."""
    n, r, x = case["slots"], case["rank"], s["x"]
    slot = s["slot"]
    mine = (slot[:, None] == torch.arange(n, device="cuda"))[:, :, None] & (torch.arange(r, device="cuda") < s["rank"][:, None])

    def one(t):
        z = torch.matmul(x, t["a"].float().flatten(0, 1).T).unflatten(1, (n, r))
        z = torch.where(mine, z * t["scale"][:, None], torch.zeros_like(z[:1, :1, :1])).flatten(1)
        return t["base"][:, :t["out"]] + torch.matmul(z, t["b"].float().transpose(1, 2).flatten(0, 1))
    return [one(t) for t in s["targets"]]


_PLAIN = {"pages": _plain_pages, "shared": _plain_shared, "adapter": _plain_adapter}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["kind"] == "adapter":
        rows, n, r, k, outs = case["rows"], case["slots"], case["rank"], case["in"], _outs(case)
        used = [s for s in _slots_of(case) if s >= 0]
        width = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 4 * rows * k + sum(8 * rows * o + width * len(set(used)) * r * (k + o) for o in outs), "flops": sum(2 * len(used) * r * (k + o) for o in outs)}
    row = 2 * case["kv_heads"] * _row_bytes(case)                                       # a token's K and V in the cache
    if case["kind"] == "pages":
        lens, slots, num_pages = _page_lens(case)
        page, size = case["page"], case["page"] * row * case["blocks"]
        tables = 8 * sum(-(-n // page) for n in lens) + 8 * slots
        if case["form"] == "fork":
            copied = sum(case["copies"] for n in lens if n % page)
        elif case["form"] == "step":
            copied = 0
        else:
            copied = sum(-(-n // page) for n in lens) // 2                              # of a pool in no order half of the pages move
        return {"bytes": 8 * num_pages + tables * (1 + case["copies"]) + 2 * copied * size, "flops": num_pages}
    lens, hd, common = _shared_lens(case), case["head_dim"], case["shared"] // case["page"] * case["page"]
    new = pairs = touched = 0
    for q, k in lens:
        kv = case["shared"] + k
        new += q
        pairs += q * (kv - q) + q * (q + 1) // 2
        touched += kv - common if q else 0
    return {"bytes": case["groups"] * (8 * new * case["heads"] * hd + (common + touched) * row), "flops": 4 * case["groups"] * pairs * case["heads"] * hd}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    if case["kind"] == "pages":
        return None                                   # whole numbers alone: they have no other value in 64 bits
    s = prepare(case, seed)
    return _exact_shared(s, case) if case["kind"] == "shared" else _exact_adapter(s, case)


def _exact_shared(s, case):
    hd, kvh, group, page = case["head_dim"], case["kv_heads"], case["heads"] // case["kv_heads"], case["page"]
    starts, kvs = s["q_start"].tolist(), s["kv_len"].tolist()
    out = torch.zeros(s["total"], kvh, group, hd, dtype=torch.float64, device="cuda")
    for i, kv in enumerate(kvs):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        blocks = s["pool"][s["table"][i, :-(-kv // page)].long()]
        for h in range(kvh):
            k, v = (_values(blocks[:, h], case, which, torch.float64).reshape(-1, hd)[:kv] for which in ("k", "v"))
            x = torch.einsum("tgd,kd->tgk", s["q"][a:b].double().reshape(b - a, kvh, group, hd)[:, h], k) / math.sqrt(hd)
            late = torch.arange(kv, device="cuda") > torch.arange(kv - (b - a), kv, device="cuda")[:, None]
            out[a:b, h] = torch.einsum("tgk,kd->tgd", torch.softmax(x.masked_fill(late[:, None], -math.inf), -1), v)
    return out.reshape(s["total"], -1)


def _exact_adapter(s, case):
    slot, x, out = s["slot"].tolist(), s["x"].double(), []
    for t in s["targets"]:
        y = t["base"][:, :t["out"]].double()
        for a in sorted(set(v for v in slot if v >= 0)):
            rows, r = (s["slot"] == a).nonzero().squeeze(1), int(s["rank"][a])
            z = torch.einsum("rk,jk->rj", x[rows], t["a"][a, :r].double())
            y[rows] += float(t["scale"][a]) * torch.einsum("rj,oj->ro", z, t["b"][a, :, :r].double())
        out.append(y)
    return out
