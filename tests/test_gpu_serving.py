"""The operators of batched serving together, as a server would use them: a prompt of one sequence, forks of it on the device, steps of
single tokens with the prefix read once and every request's own adapter, drafted tokens given back, a pool moved to its front in the middle,
against the same tokens walked one by one over a float32 cache with the adapters folded into the weights."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D, HEADS, KVH, HD, FFN, LAYERS, SLOTS, RANK = 256, 8, 2, 64, 512, 2, 3, 16
PROJ = {"q": (HEADS * HD, D), "k": (KVH * HD, D), "v": (KVH * HD, D), "o": (D, HEADS * HD), "gate": (FFN, D), "up": (FFN, D), "down": (D, FFN)}


def rope(x, pos):
    half = HD // 2
    ang = pos / 10000.0 ** (2 * np.arange(half) / HD)
    c, s = np.cos(ang), np.sin(ang)
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


class Model:
    """Weights in float64 on the host and resident on the device, adapters of both."""

    def __init__(self, wv):
        rng = np.random.default_rng(21)
        self.keep, self.w, self.keys, self.norms, self.ad, self.host = [], [], [], [], [], []
        for _ in range(LAYERS):
            w, keys, ad, host = {}, {}, {}, {}
            for n, (r, c) in PROJ.items():
                blob = wv.quant.Pack(wv.quant.Format.FormatQ8_0, rng.normal(0, 0.06, r * c).astype(np.float32), r, c)
                self.keep.append(blob)
                w[n], keys[n] = wv.quant.Unpack(blob).reshape(r, c).astype(np.float64), wv.quant.EnsureResident(blob)
                if n in ("k", "up"):
                    continue                             # projections without adapters
                a = torch.from_numpy(rng.normal(0, 0.06, (SLOTS, RANK, c)).astype(np.float32)).cuda().bfloat16()
                b = torch.from_numpy(rng.normal(0, 0.25, (SLOTS, r, RANK)).astype(np.float32)).cuda().bfloat16()
                s = torch.tensor([0.7, 1.3, 1.0], device="cuda")
                self.keep += [a, b, s]
                ad[n] = wv.adapters.Adapters(a.data_ptr(), b.data_ptr(), 0, s.data_ptr(), SLOTS, RANK, c, r, wv.quant.DTypeBFloat16)
                host[n] = [float(s[i]) * b[i].double().cpu().numpy() @ a[i].double().cpu().numpy() for i in range(SLOTS)]
            self.w.append(w), self.keys.append(keys), self.ad.append(ad), self.host.append(host)
            self.norms.append([rng.normal(1, 0.05, D) for _ in range(2)])

    def walk(self, tokens, slots):
        """Hidden states in 64 bits of a sequence's tokens [n, D], token i under adapter slots[i] (-1: none)."""
        cache, out = [([], []) for _ in range(LAYERS)], []
        for pos, (x, slot) in enumerate(zip(tokens.astype(np.float64), slots)):
            h = x.copy()
            for w, host, (g1, g2), (ck, cv) in zip(self.w, self.host, self.norms, cache):
                def mat(n, v, w=w, host=host):
                    y = w[n] @ v
                    return y + host[n][slot] @ v if slot >= 0 and n in host else y
                norm = lambda v, g: v / np.sqrt((v * v).mean() + 1e-5) * g  # noqa: E731
                z = norm(h, g1)
                q, k, v = mat("q", z).reshape(HEADS, HD), mat("k", z).reshape(KVH, HD), mat("v", z).reshape(KVH, HD)
                ck.append(rope(k, pos)), cv.append(v)
                q, K, V = rope(q, pos), np.stack(ck), np.stack(cv)
                o = np.zeros((HEADS, HD))
                for i in range(HEADS):
                    p = K[:, i // (HEADS // KVH)] @ q[i] / np.sqrt(HD)
                    p = np.exp(p - p.max())
                    o[i] = p @ V[:, i // (HEADS // KVH)] / p.sum()
                h = h + mat("o", o.reshape(-1))
                z = norm(h, g2)
                g, u = mat("gate", z), mat("up", z)
                h = h + mat("down", g / (1 + np.exp(-g)) * u)
            out.append(h)
        return np.stack(out)


@pytest.mark.parametrize("bits,tol", [(16, 0.01), (8, 0.04)])
def test_forks_with_adapters_as_one_by_one(wv, bits, tol):
    """Tolerance: as of the decoder block's own test (TF32 products, 2^-10 of sum |w x|, four a block, two blocks; an 8-bit cache adds half a step,
    1 / 254 of a row's largest value, to K and to V); the adapters' products are float32's."""
    p, ad = wv.paged, wv.adapters
    m = Model(wv)
    rng = np.random.default_rng(bits)
    page, slots, num_pages, stride, most = 16, 5, 60, 12, 100
    prompt, steps = 77, 6
    tail = [rng.normal(0, 1, (steps, D)).astype(np.float32) for _ in range(slots)]
    first = rng.normal(0, 1, (prompt, D)).astype(np.float32)
    which = [0, 1, -1, 2, 1]                                              # the adapter of every request; the prompt is walked without one
    z = lambda *n: torch.zeros(*n, device="cuda")  # noqa: E731
    zi = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(list(v), dtype=torch.int32, device="cuda")  # noqa: E731
    work = {"norm": z(most, D), "proj": z(most, D), "q": z(most, HEADS * HD), "attn": z(most, HEADS * HD), "k": z(most, KVH * HD), "v": z(most, KVH * HD),
            "gate": z(most, FFN), "up": z(most, FFN)}
    refs, pages, kv = zi(num_pages), zi(slots, stride) - 1, zi(slots)
    table = p.KVTable(refs.data_ptr(), pages.data_ptr(), kv.data_ptr(), num_pages, page, slots, stride)
    pools = [torch.zeros(num_pages * KVH * p.KVBlockBytes(bits, page, HD), dtype=torch.uint8, device="cuda") for _ in range(LAYERS)]
    caches = [p.KVPages(t.data_ptr(), bits, num_pages, page, KVH, HD) for t in pools]
    blocks, gs = p.KVBlocks(caches), [[torch.from_numpy(g.astype(np.float32)).cuda() for g in n] for n in m.norms]
    decs = [p.PagedBlockDecoder(_cfg(), keys, {**{n: t.data_ptr() for n, t in work.items()}, "attn_norm": g[0].data_ptr(), "ffn_norm": g[1].data_ptr()}, c, most, adapters=a)
            for keys, g, c, a in zip(m.keys, gs, caches, m.ad)]

    def grow(n):
        add, ok = ints(n), zi(slots)
        p.KVExtendCUDA(table, add.data_ptr(), ok.data_ptr(), blocks)
        assert ok.tolist() == [1] * slots

    def step(h, new, groups=None, plan=0):
        start = ints(np.concatenate([[0], np.cumsum(new)]))
        batch = p.Batch(start.data_ptr(), kv.data_ptr(), pages.data_ptr(), slots, stride, sum(new), max(new), int(kv.max()))
        for d in decs:
            d.step(h.data_ptr(), batch, groups=groups, plan=plan)
        torch.cuda.synchronize()
        assert wv._lib.lib().wv_device_status() == 0

    want = [m.walk(np.concatenate([first, t]), [-1] * prompt + [a] * steps) for t, a in zip(tail, which)]
    near = lambda h, ref: float(np.abs(h.double().cpu().numpy() - ref).max()) <= tol * float(np.abs(ref).max())  # noqa: E731
    # the prompt, once
    grow([prompt, 0, 0, 0, 0])
    h = torch.from_numpy(first).cuda()
    step(h, [prompt, 0, 0, 0, 0])
    assert near(h, want[0][:prompt])
    # four forks of it; its last page is copied as soon as somebody writes on
    src, dst = ints([0] * 4), ints([1, 2, 3, 4])
    p.KVForkCUDA(table, src.data_ptr(), dst.data_ptr(), 4)
    start, shared = ints([0, slots]), ints([prompt])
    groups = p.Groups(start.data_ptr(), shared.data_ptr(), 1, prompt)
    plan = torch.zeros(ad.PlanBytes(2 * slots, SLOTS), dtype=torch.uint8, device="cuda")

    def apply(per):
        slot = ints([a for a in which for _ in range(per)])
        ad.PlanCUDA(slot.data_ptr(), per * slots, SLOTS, plan.data_ptr())
        return plan.data_ptr()

    for i in range(2):
        grow([1] * slots)
        h = torch.from_numpy(np.stack([t[i] for t in tail])).cuda()
        step(h, [1] * slots, groups, apply(1))
        assert near(h, np.stack([w[prompt + i] for w in want]))
        if i == 0:
            assert int((refs == slots).sum()) == prompt // page and int(refs.max()) == slots
    # two drafted tokens each, the second one wrong: given back, and the page tables moved to the front of the pools
    grow([2] * slots)
    h = torch.from_numpy(np.concatenate([np.stack([t[2], t[5]]) for t in tail])).cuda()
    step(h, [2] * slots, groups, apply(2))
    assert near(h[::2], np.stack([w[prompt + 2] for w in want]))
    keep, live = ints([prompt + 3] * slots), zi(1)
    p.KVTrimCUDA(table, slots, keep.data_ptr())
    p.KVCompactCUDA(table, blocks, live.data_ptr())
    assert int(live) == prompt // page + slots and not refs[int(live):].any()
    for i in range(3, steps):
        grow([1] * slots)
        h = torch.from_numpy(np.stack([t[i] for t in tail])).cuda()
        step(h, [1] * slots, groups, apply(1))
        assert near(h, np.stack([w[prompt + i] for w in want]))
    p.KVTrimCUDA(table, slots)
    torch.cuda.synchronize()
    assert not refs.any() and not kv.any() and wv._lib.lib().wv_device_status() == 0


def _cfg():
    from welvet_b200.decode import BlockConfig
    return BlockConfig(D, HEADS, KVH, HD, FFN, 256)


def test_step_refuses_what_does_not_fit(wv):
    p = wv.paged
    bufs = {n: 0 for n in ("norm", "proj", "q", "attn", "k", "v", "gate", "up", "attn_norm", "ffn_norm")}
    keys = {n: 0 for n in PROJ}
    batch = p.Batch(0, 0, 0, 1, 1, 1, 1, 1)
    with pytest.raises(ValueError, match="window"):
        p.PagedBlockDecoder(_cfg(), keys, bufs, p.KVPages(0, 8, 1, 16, KVH, HD), 4, window=8).step(0, batch, groups=p.Groups(0, 0, 0, 0))
    with pytest.raises(ValueError, match="adapters"):
        p.PagedBlockDecoder(_cfg(), keys, bufs, p.KVPages(0, 8, 1, 16, KVH, HD), 4).step(0, batch, plan=1)
