"""The paged key/value cache and the attention over it against plain implementations in 64 bits: rounding bit for bit, every width and
head layout, lengths around pages and tiles, rows that see nothing, windows, strides, values that are not finite, and the refusals."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

FLT_MIN = np.float32(2.0 ** -126)


class Cache:
    """A pool with a shuffled page table, filled through wv_kv_write_dev or by hand; `block` is the layout of welvet_cuda.h."""

    def __init__(self, wv, bits, page, kvh, hd, lens, spare=2, seed=0):
        self.wv, self.bits, self.page, self.kvh, self.hd, self.lens = wv, bits, page, kvh, hd, lens
        need = [-(-k // page) for _, k in lens]
        self.num_pages = sum(need) + spare
        self.bytes = wv.paged.KVBlockBytes(bits, page, hd)
        self.pool = torch.zeros(self.num_pages, kvh, self.bytes, dtype=torch.uint8, device="cuda")
        perm = np.random.default_rng(seed).permutation(self.num_pages).astype(np.int32)
        self.table = np.full((len(lens), max(1, max(need))), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = perm[at:at + n]
            at += n
        self.d_table = torch.from_numpy(self.table).cuda()
        self.pages = wv.paged.KVPages(self.pool.data_ptr(), bits, self.num_pages, page, kvh, hd)
        self.batch, self.keep = self.batch_of(lens)

    def batch_of(self, lens, total=None, max_q=None):
        start = np.concatenate([[0], np.cumsum([q for q, _ in lens])]).astype(np.int32)
        ds, dk = torch.from_numpy(start).cuda(), torch.tensor([k for _, k in lens], dtype=torch.int32, device="cuda")
        b = self.wv.paged.Batch(ds.data_ptr(), dk.data_ptr(), self.d_table.data_ptr(), len(lens), self.table.shape[1],
                                int(start[-1]) if total is None else total, max(q for q, _ in lens) if max_q is None else max_q, max(k for _, k in lens))
        return b, (ds, dk)

    def fill(self, k, v):
        """All cached tokens [sum kv, kvh * hd] of the sequences written in one call (theta 0)."""
        b, keep = self.batch_of([(n, n) for _, n in self.lens])
        if k.shape[0]:
            self.wv.paged.KVWriteCUDA(self.pages, b, k.data_ptr(), v.data_ptr())
        torch.cuda.synchronize()

    def rows(self, which):
        """Every cached token's values in 64 bits, from the pool's bytes: [sum kv, kvh, hd]."""
        pool, page, hd, code = self.pool.cpu().numpy(), self.page, self.hd, self.hd * self.bits // 8
        out = []
        for i, (_, kv) in enumerate(self.lens):
            for t in range(kv):
                blk = pool[self.table[i, t // page]]
                s = t % page
                at = (page * code if which == "v" else 0) + s * code
                c = blk[:, at:at + code]
                sa = 2 * page * code + (4 * page if which == "v" else 0) + 4 * s
                scale = np.ascontiguousarray(blk[:, sa:sa + 4]).view(np.float32).astype(np.float64)
                if self.bits == 16:
                    c = np.ascontiguousarray(c).view(np.float16).astype(np.float64)
                elif self.bits == 8:
                    c = c.view(np.int8).astype(np.float64)
                else:
                    c = np.stack([c & 15, c >> 4], -1).reshape(self.kvh, hd).astype(np.float64) - 8
                    ta = 2 * page * code + 8 * page + (page * (hd // 16) if which == "v" else 0) + s * (hd // 16)
                    c *= np.repeat(blk[:, ta:ta + hd // 16].astype(np.float64), 16, -1)
                out.append(c * scale)
        return np.stack(out) if out else np.zeros((0, self.kvh, hd))


def quantise(x, bits):
    """The header's formulas, row by row of the last axis, in the float32 steps that it states -> values in 64 bits."""
    x = np.asarray(x, np.float32)
    fine = np.isfinite(x).all(-1, keepdims=True)
    return np.where(fine, quantise_finite(np.where(fine, x, 0), bits), np.nan)


def quantise_finite(x, bits):
    a = np.abs(x).max(-1, keepdims=True)
    if bits == 16:
        e = np.floor(np.log2(np.maximum(a, FLT_MIN).astype(np.float64)))
        s = np.exp2(np.maximum(e - 14, -126)).astype(np.float32)
        s = np.where(a > 0, s, FLT_MIN)
        return (x / s).astype(np.float16).astype(np.float64) * s
    if bits == 8:
        s = np.maximum(a * (np.float32(1) / np.float32(127)), FLT_MIN)
        return np.rint(x / s).astype(np.float64) * s
    s = np.maximum(a * (np.float32(1) / np.float32(1785)), FLT_MIN)
    g = x.reshape(*x.shape[:-1], -1, 16)
    t = np.clip(np.ceil(np.abs(g).max(-1) * (np.float32(1) / np.float32(7)) / s), 1, 255).astype(np.float32)
    c = np.clip(np.rint(g / (s * t)[..., None]), -7, 7).astype(np.float64)
    return (c * t[..., None]).reshape(x.shape) * s


def rope64(x, pos, theta):
    """mha/rope.go:6-21 in 64 bits: x [tokens, heads, hd]."""
    hd = x.shape[-1]
    x = x.astype(np.float64)
    ang = pos[:, None] / theta ** (2.0 * np.arange(hd // 2) / hd)
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    a, b = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def attn64(q, k, v, scale, window, first):
    """Token i at position first + i; q [n, heads, hd], k and v [kv, kvh, hd]. Also what scales an error bound: for every output
    sum p |v|, and for every row the largest sum |q k| scale."""
    n, heads, hd = q.shape
    g = heads // k.shape[1]
    out, mag, reach = np.zeros((n, heads, hd)), np.zeros((n, heads, hd)), np.zeros((n, heads))
    for i in range(n):
        p = first + i
        lo = max(0, p - window + 1) if window else 0
        if p < 0:
            continue
        for h in range(heads):
            kk, vv = k[lo:p + 1, h // g], v[lo:p + 1, h // g]
            x = kk @ q[i, h].astype(np.float64) * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            out[i, h], mag[i, h] = w @ vv, w @ np.abs(vv)
            reach[i, h] = (np.abs(kk) @ np.abs(q[i, h].astype(np.float64))).max() * abs(scale)
    return out, mag, reach


def bound(mag, reach, hd, kv):
    """float32 arithmetic: a logit's sum of hd products is off by at most hd 2^-23 of the sum of their magnitudes (a tensor core may cut
    instead of rounding: twice 2^-24), a weight by as much relatively, and by 2^-20 for the exponential and the pieces; the sums over
    the keys, block by block, by (kv / 64 + 64) 2^-23. The weights' errors count twice, above and below the fraction."""
    return (2 * hd * 2.0 ** -23 * reach[..., None] + 2.0 ** -19 + (kv / 64 + 64) * 2.0 ** -23) * mag + 1e-30


def run_attn(c, q, heads, scale, window=0, batch=None, ldq=0, ldo=0, out=None, rows=None):
    o = torch.full((rows or q.shape[0], ldo or heads * c.hd), 7.0, device="cuda") if out is None else out
    c.wv.paged.AttnPagedCUDA(c.pages, batch or c.batch, q.data_ptr(), o.data_ptr(), heads, scale, window=window, ldq=ldq, ldo=ldo)
    torch.cuda.synchronize()
    return o.cpu().numpy()


def check_attn(wv, bits, page, heads, kvh, hd, lens, window=0, seed=0, spread=1.0):
    rng = np.random.default_rng(seed)
    c = Cache(wv, bits, page, kvh, hd, lens, seed=seed)
    total_kv, total_q = sum(k for _, k in lens), sum(q for q, _ in lens)
    k = torch.from_numpy((rng.normal(0, spread, (total_kv, kvh * hd))).astype(np.float32)).cuda()
    v = torch.from_numpy((rng.normal(0, 1, (total_kv, kvh * hd)) * np.exp(rng.normal(0, 1, (total_kv, 1)))).astype(np.float32)).cuda()
    c.fill(k, v)
    q = rng.normal(0, 1, (total_q, heads * hd)).astype(np.float32)
    scale = hd ** -0.5
    got = run_attn(c, torch.from_numpy(q).cuda(), heads, scale, window).reshape(total_q, heads, hd)
    kk, vv = c.rows("k"), c.rows("v")
    rq = rk = 0
    for nq, kv in lens:
        want, mag, reach = attn64(q[rq:rq + nq].reshape(nq, heads, hd), kk[rk:rk + kv], vv[rk:rk + kv], scale, window, kv - nq)
        err = np.abs(got[rq:rq + nq] - want)
        tol = bound(mag, reach, hd, kv)
        assert (err <= tol).all(), (nq, kv, float((err / np.maximum(tol, 1e-30)).max()), float(err.max()))
        rq, rk = rq + nq, rk + kv
    assert c.wv._lib.lib().wv_device_status() == 0
    return c


# ------------------------------------------------------------------ the cache
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("hd", [16, 64, 80, 128, 144, 256])
def test_rows_are_rounded_as_stated(wv, bits, hd):
    """Without rotation the codes are those of the header's float32 steps bit for bit, through the pool's bytes and read back."""
    lens = [(5, 37), (1, 1), (0, 20), (33, 33)]
    c = Cache(wv, bits, 16, 2, hd, lens, seed=hd)
    rng = np.random.default_rng(hd + bits)
    n = sum(k for _, k in lens)
    k = (rng.normal(0, 1, (n, 2 * hd)) * np.exp(rng.normal(0, 3, (n, 1)))).astype(np.float32)
    v = rng.normal(0, 1, (n, 2 * hd)).astype(np.float32)
    k[3] = 0.0
    k[4] *= np.float32(1e-40)                     # subnormal
    k[5] *= np.float32(1e37) / np.abs(k[5]).max()
    v[6, ::2] = 0.0
    v[7, :16] *= np.float32(1e6)                  # one group far above the others
    v[8] = 3.0
    c.fill(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    for x, which in ((k, "k"), (v, "v")):
        want = quantise(x.reshape(n, 2, hd), bits)
        assert np.array_equal(c.rows(which), want, equal_nan=True), which
    # read back: the same values, rounded to float32 once
    b, keep = c.batch_of([(m, m) for _, m in lens])
    dk, dv = (torch.full((n, 2 * hd), 9.0, device="cuda") for _ in range(2))
    wv.paged.KVReadCUDA(c.pages, b, dk.data_ptr(), dv.data_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(dk.cpu().numpy().reshape(n, 2, hd), c.rows("k").astype(np.float32), equal_nan=True)
    assert np.array_equal(dv.cpu().numpy().reshape(n, 2, hd), c.rows("v").astype(np.float32))
    # the relative error of a row is what the width allows
    step = {16: 2.0 ** -11, 8: 0.5 / 127 + 1e-6, 4: 0.5 / 7 + 1.0 / 255}[bits]
    err = np.abs(c.rows("v") - v.reshape(n, 2, hd)).max(-1)
    assert (err <= step * np.abs(v.reshape(n, 2, hd)).max(-1)).all()


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("largest", [1e37, 2.0 ** 127, 3.3e38])
def test_rows_of_the_largest_magnitudes(wv, bits, largest):
    """Rows whose largest value is near the end of float32's range, which one that rounds up to the next power of two would pass."""
    c = Cache(wv, bits, 16, 2, 128, [(20, 20)])
    rng = np.random.default_rng(bits)
    k, v = (rng.uniform(-1, 1, (20, 2, 128)) * largest for _ in range(2))
    k[:, :, 5], v[:, :, 100] = largest, -largest
    k, v = k.astype(np.float32), v.astype(np.float32)
    assert np.isfinite(k).all() and np.isfinite(v).all()
    c.fill(torch.from_numpy(k.reshape(20, 256)).cuda(), torch.from_numpy(v.reshape(20, 256)).cuda())
    back = [torch.zeros(20, 256, device="cuda") for _ in range(2)]
    wv.paged.KVReadCUDA(c.pages, c.batch, back[0].data_ptr(), back[1].data_ptr())
    torch.cuda.synchronize()
    for x, which, b in ((k, "k", back[0]), (v, "v", back[1])):
        want = quantise(x, bits)
        assert np.isfinite(want).all() and np.array_equal(c.rows(which), want)
        assert np.array_equal(b.cpu().numpy().reshape(20, 2, 128), want.astype(np.float32))


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("hd,theta", [(64, 10000.0), (128, 500000.0), (80, 10000.0), (256, 10000.0)])
def test_rotation_and_places(wv, bits, hd, theta):
    """Q and K are rotated by their position as wv_rope_cache_dev does, in place or not, with gaps between rows; only the new
    tokens' places change. A rotated value may round the other way where it lies within 2^-22 of a boundary, so codes may be a step
    off in a handful of places."""
    heads, kvh, page = 6, 2, 32
    lens = [(3, 70), (0, 5), (40, 100), (1, 1), (2, 90001)]
    c = Cache(wv, bits, page, kvh, hd, lens, seed=1)
    rng = np.random.default_rng(5)
    n, w, ld = sum(q for q, _ in lens), kvh * hd, kvh * hd + 12
    k, v = (rng.normal(0, 1, (n, ld)).astype(np.float32) for _ in range(2))
    q = rng.normal(0, 1, (n, heads * hd + 4)).astype(np.float32)
    before = c.pool.clone()
    dk, dv, dq = (torch.from_numpy(t).cuda() for t in (k, v, q))
    dqo = torch.zeros(n, heads * hd, device="cuda")
    args = (c.pages, c.batch, dk.data_ptr(), dv.data_ptr())
    wv.paged.KVWriteCUDA(*args, dq.data_ptr(), dqo.data_ptr(), heads, theta, ldk=ld, ldv=ld, ldq=heads * hd + 4)
    torch.cuda.synchronize()
    pos = np.concatenate([np.arange(m - a, m) for a, m in lens]).astype(np.float64)
    want_q = rope64(q[:, :heads * hd].reshape(n, heads, hd), pos, theta)
    got_q = dqo.cpu().numpy().reshape(n, heads, hd)
    assert np.abs(got_q - want_q).max() <= 2.0 ** -22 * np.abs(want_q).max()
    got = {which: c_rows(c, which) for which in "kv"}
    want_k = rope64(k[:, :w].reshape(n, kvh, hd), pos, theta)
    back = quantise(want_k.astype(np.float32), bits)
    step = {16: 2.0 ** -10, 8: 1.0 / 126, 4: 1.0 / 6}[bits]
    off = np.abs(got["k"] - back) / np.abs(want_k).max(-1, keepdims=True)
    assert off.max() <= step and (off > 1e-6).mean() < 1e-3
    assert np.array_equal(got["v"], quantise(v[:, :w].reshape(n, kvh, hd), bits))
    # in place gives the same; nothing but the new tokens' bytes changed
    wv.paged.KVWriteCUDA(*args, dq.data_ptr(), dq.data_ptr(), heads, theta, ldk=ld, ldv=ld, ldq=heads * hd + 4, ldqo=heads * hd + 4)
    torch.cuda.synchronize()
    assert np.array_equal(dq.cpu().numpy()[:, :heads * hd], dqo.cpu().numpy()) and np.array_equal(dq.cpu().numpy()[:, heads * hd:], q[:, heads * hd:])
    used = set(int(c.table[i, t // page]) for i, (a, m) in enumerate(lens) for t in range(m - a, m))
    same = [p for p in range(c.num_pages) if p not in used]
    assert torch.equal(c.pool[same], before[same])
    assert c.wv._lib.lib().wv_device_status() == 0


def c_rows(c, which):
    """The new tokens' rows of c."""
    lens, out = c.lens, []
    keep = c.lens
    for i, (a, m) in enumerate(lens):
        one = Cache.__new__(Cache)
        one.__dict__.update(c.__dict__)
        if not a:
            continue
        first = (m - a) // c.page                 # from the first page that a new token is in
        one.lens, one.table = [(0, m - first * c.page)], c.table[i:i + 1, first:]
        out.append(Cache.rows(one, which)[m - a - first * c.page:])
    c.lens = keep
    return np.concatenate(out)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_rows_that_are_not_finite(wv, bits):
    """NaN scale and zero codes; V and K apart from one another, and only in the row's own head."""
    lens = [(6, 6)]
    c = Cache(wv, bits, 16, 2, 64, lens)
    k, v = torch.randn(6, 128, device="cuda"), torch.randn(6, 128, device="cuda")
    k[1, 3], k[2, 64], v[3, 127], v[4, 0] = math.inf, math.nan, -math.inf, math.nan
    c.fill(k, v)
    rk, rv = c.rows("k"), c.rows("v")
    bad_k, bad_v = np.zeros((6, 2), bool), np.zeros((6, 2), bool)
    bad_k[1, 0] = bad_k[2, 1] = bad_v[3, 1] = bad_v[4, 0] = True
    assert np.array_equal(np.isnan(rk).all(-1), bad_k) and np.array_equal(np.isnan(rk).any(-1), bad_k)
    assert np.array_equal(np.isnan(rv).all(-1), bad_v) and np.array_equal(np.isnan(rv).any(-1), bad_v)


# ------------------------------------------------------------------ attention
LENS = [(1, 1), (1, 2), (0, 0), (1, 15), (1, 16), (1, 17), (0, 9), (3, 33), (1, 129), (5, 64), (1, 300)]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("heads,kvh,hd", [(1, 1, 64), (8, 2, 128), (6, 2, 80), (16, 2, 64), (8, 1, 256), (32, 1, 128), (5, 5, 16), (3, 1, 144)])
def test_attention_small(wv, bits, heads, kvh, hd):
    check_attn(wv, bits, 16, heads, kvh, hd, LENS, seed=heads + hd)


@pytest.mark.parametrize("bits,page", [(16, 16), (8, 48), (4, 64), (16, 128), (8, 16), (4, 80)])
@pytest.mark.parametrize("lens", [[(1, 2049)], [(1, 5000), (1, 3), (1, 1024), (0, 0)], [(17, 500), (1, 700), (130, 130)], [(257, 300)], [(64, 1000), (2, 2), (63, 64)]])
def test_attention_lengths(wv, bits, page, lens):
    check_attn(wv, bits, page, 8, 2, 128, lens, seed=page)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("hd,heads,kvh", [(64, 4, 4), (128, 4, 1), (80, 6, 2), (256, 2, 1)])
def test_attention_of_chunks(wv, bits, hd, heads, kvh):
    check_attn(wv, bits, 32, heads, kvh, hd, [(200, 333), (129, 129), (0, 40), (1, 77), (256, 256)], seed=hd)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 100, 1000])
@pytest.mark.parametrize("lens", [[(1, 400), (1, 5)], [(150, 400), (20, 20)]])
def test_attention_window(wv, window, lens):
    for bits in (16, 4):
        check_attn(wv, bits, 16, 4, 2, 64, lens, window=window, seed=window)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, 301, 300, 299, -5])
@pytest.mark.parametrize("lens", [[(2, 300), (5, 3), (2, 0)], [(310, 300), (70, 64), (1, 90)]])
def test_windows_wider_than_the_cache(wv, window, lens):
    """A window that no sequence fills, up to the largest number, is none, with rows before position 0 as well."""
    for bits in (16, 4):
        check_attn(wv, bits, 16, 4, 1, 64, lens, window=max(window, 0))
        c = Cache(wv, bits, 16, 1, 64, lens)
        n, total = sum(k for _, k in lens), sum(q for q, _ in lens)
        c.fill(torch.randn(n, 64, device="cuda"), torch.randn(n, 64, device="cuda"))
        q = torch.randn(total, 256, device="cuda")
        if window < 0 or window >= 300:
            assert np.array_equal(run_attn(c, q, 4, 0.125, window=window), run_attn(c, q, 4, 0.125))


def test_attention_sharp_and_flat(wv):
    """Weights on a single key, and equal keys: the running maximum has to move and to stay."""
    for spread in (30.0, 0.0, 1e-3):
        check_attn(wv, 16, 16, 4, 2, 128, [(1, 1000), (70, 500)], seed=3, spread=spread)


@pytest.mark.parametrize("nq", [1, 3])
def test_long_sequences_of_a_full_batch(wv, nq):
    """So many sequences that none has to be split to fill the chip: the sums over 12000 positions are as exact as those over a few.
    Bound: at most 40 additions that cut off up to 2^-23 of a sum one after the other, half of that on average, and as much again for
    weights, divisor and the sums of the parts."""
    seqs, kv, heads, hd, dev = 160, 12000, 4, 64, "cuda"
    gen = torch.Generator(device=dev).manual_seed(5)
    rand = lambda *n: torch.randn(*n, device=dev, generator=gen)  # noqa: E731
    c = Cache(wv, 8, 64, 1, hd, [(nq, kv)])
    c.fill(rand(kv, hd), rand(kv, hd))
    k, v = torch.zeros(kv, hd, device=dev), torch.zeros(kv, hd, device=dev)
    whole, keep = c.batch_of([(kv, kv)])
    wv.paged.KVReadCUDA(c.pages, whole, k.data_ptr(), v.data_ptr())
    table = c.d_table.repeat(seqs, 1)                                     # one sequence's pages for all of them
    start, lens = torch.arange(seqs + 1, dtype=torch.int32, device=dev) * nq, torch.full((seqs,), kv, dtype=torch.int32, device=dev)
    b = wv.paged.Batch(start.data_ptr(), lens.data_ptr(), table.data_ptr(), seqs, table.shape[1], seqs * nq, nq, kv)
    q, out = rand(seqs * nq, heads * hd), torch.zeros(seqs * nq, heads * hd, device=dev)
    wv.paged.AttnPagedCUDA(c.pages, b, q.data_ptr(), out.data_ptr(), heads, 0.125)
    torch.cuda.synchronize()
    s = q.double().view(seqs, nq, heads, hd) @ k.double().T * 0.125
    last = kv - nq + torch.arange(nq, device=dev)
    s = s.masked_fill(torch.arange(kv, device=dev) > last[:, None, None], -math.inf)
    want = (torch.softmax(s, -1) @ v.double()).view(seqs * nq, heads * hd)
    assert ((out.double() - want).norm() / want.norm()).item() <= 2 * 40 * 2.0 ** -24


def test_rows_that_see_nothing(wv):
    """More new tokens than the cache holds: positions before 0 give zeros."""
    lens = [(5, 3), (70, 64), (2, 0)]
    for bits in (16, 8, 4):
        check_attn(wv, bits, 16, 4, 1, 64, lens)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("nq", [1, 9, 140])
def test_what_is_masked_does_not_count(wv, bits, nq):
    """Unused slots and pages are full of garbage, and the newest token's K and V are not finite: only the rows that see it are NaN."""
    lens = [(nq, 200), (nq, 150)]
    heads, kvh, hd, page = 8, 2, 64, 64
    c = Cache(wv, bits, page, kvh, hd, lens, seed=nq)
    c.pool.fill_(255)
    rng = np.random.default_rng(nq)
    k, v = (torch.from_numpy(rng.normal(0, 1, (350, kvh * hd)).astype(np.float32)).cuda() for _ in range(2))
    c.fill(k, v)
    q = torch.from_numpy(rng.normal(0, 1, (2 * nq, heads * hd)).astype(np.float32)).cuda()
    clean = run_attn(c, q, heads, 0.125)
    assert np.isfinite(clean).all()
    for what in (k, v):
        saved = what[199].clone()
        what[199, :hd] = math.nan if what is k else math.inf          # kv head 0 of the first sequence's last token
        c.fill(k, v)
        got = run_attn(c, q, heads, 0.125).reshape(2 * nq, heads, hd)
        bad = np.zeros((2 * nq, heads), bool)
        bad[nq - 1, :heads // kvh] = True
        assert np.array_equal(np.isnan(got).all(-1), bad) and np.array_equal(np.isnan(got).any(-1), bad)
        assert np.array_equal(got[~bad], clean.reshape(2 * nq, heads, hd)[~bad])
        what[199] = saved
    c.fill(k, v)
    # a query that is not finite makes its own head's row NaN and no other
    q2 = q.clone()
    q2[0, 5] = math.inf
    q2[nq, 3 * hd] = math.nan
    got = run_attn(c, q2, heads, 0.125).reshape(2 * nq, heads, hd)
    bad = np.zeros((2 * nq, heads), bool)
    bad[0, 0] = bad[nq, 3] = True
    assert np.array_equal(np.isnan(got).all(-1), bad) and np.array_equal(np.isnan(got).any(-1), bad)
    assert np.array_equal(got[~bad], clean.reshape(2 * nq, heads, hd)[~bad])


def test_large_and_small_values(wv):
    """Queries and values far from 1, in rows beside one another."""
    for bits in (16, 8, 4):
        lens = [(2, 90), (100, 100)]
        c = Cache(wv, bits, 16, 1, 64, lens)
        rng = np.random.default_rng(0)
        k = rng.normal(0, 1, (190, 64)).astype(np.float32)
        v = (rng.normal(0, 1, (190, 64)) * 10.0 ** rng.integers(-20, 20, (190, 1))).astype(np.float32)
        k[:, 7] *= 1e5
        q = (rng.normal(0, 1, (102, 128)) * 10.0 ** rng.integers(-12, 1, (102, 1))).astype(np.float32)
        q[:, [7, 71]] = 0
        c.fill(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
        got = run_attn(c, torch.from_numpy(q).cuda(), 2, 0.125).reshape(102, 2, 64)
        kk, vv = c.rows("k"), c.rows("v")
        a = 0
        for (nq, kv), r in zip(lens, (0, 2)):
            want, mag, reach = attn64(q[r:r + nq].reshape(nq, 2, 64), kk[a:a + kv], vv[a:a + kv], 0.125, 0, kv - nq)
            assert (np.abs(got[r:r + nq] - want) <= bound(mag, reach, 64, kv)).all(), bits
            a += kv


def attn_of(c, q, heads, scale, lens):
    """A call's outputs against 64 bits: error and bound of every value. A weight is a multiple of 2^-24 in the products, where the row's
    largest is 2^4 or more (chunks; 2^6 for few rows): rounding leaves 2^-25 / 2^4 of the largest a key, times value codes that reach
    twice the largest value in units of the largest scale. Where the keys with weight have the code 0, that is all there is."""
    got = run_attn(c, torch.from_numpy(q.reshape(q.shape[0], -1)).cuda(), heads, scale).reshape(q.shape)
    kk, vv = c.rows("k"), c.rows("v")
    err, tol = np.zeros(q.shape), np.zeros(q.shape)
    r = a = 0
    for nq, kv in lens:
        want, mag, reach = attn64(q[r:r + nq], kk[a:a + kv], vv[a:a + kv], scale, 0, kv - nq)
        err[r:r + nq] = np.abs(got[r:r + nq] - want)
        tol[r:r + nq] = bound(mag, reach, c.hd, kv) + kv * 2.0 ** -28 * (np.abs(vv[a:a + kv]).max() if kv else 0)
        r, a = r + nq, a + kv
    return err, tol


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("scale", [-0.125, -2.0, 0.0, -0.0, 1e-20, 3.0])
def test_scales_of_any_sign(wv, bits, scale):
    """A scale below 0 turns the order of the keys, one of 0 gives their mean; few rows and chunks."""
    lens = [(1, 90), (12, 40), (100, 400), (6, 3)]
    c = Cache(wv, bits, 16, 2, 64, lens)
    rng = np.random.default_rng(bits)
    n, total = sum(k for _, k in lens), sum(a for a, _ in lens)
    c.fill(*(torch.from_numpy(rng.normal(0, 1, (n, 128)).astype(np.float32)).cuda() for _ in range(2)))
    q = rng.normal(0, 1, (total, 4, 64)).astype(np.float32)
    err, tol = attn_of(c, q, 4, scale, lens)
    assert (err <= tol).all(), float((err / np.maximum(tol, 1e-30)).max())


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("size", [2.0 ** 90, 1e20, 1e-20, 1e-22])
def test_values_over_the_stated_range(wv, bits, size):
    """V from the smallest scales that count (2^-90) to the largest values (2^90), over enough keys for several tiles and splits."""
    lens = [(1, 2000), (12, 40), (100, 900)]
    c = Cache(wv, bits, 16, 2, 64, lens)
    rng = np.random.default_rng(bits)
    n, total = sum(k for _, k in lens), sum(a for a, _ in lens)
    v = rng.uniform(-1, 1, (n, 2, 64))
    v[:, :, 9] = np.sign(v[:, :, 9])                                      # every row reaches 1
    c.fill(torch.from_numpy(rng.normal(0, 1, (n, 128)).astype(np.float32)).cuda(), torch.from_numpy((v * size).astype(np.float32).reshape(n, 128)).cuda())
    q = rng.normal(0, 1, (total, 4, 64)).astype(np.float32)
    err, tol = attn_of(c, q, 4, 0.125, lens)
    assert (err <= tol - 1e-30).all(), float((err / tol).max())          # without the absolute part


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("large", [3e7, 1e9, 1e12, 1e30])
def test_logits_of_any_size(wv, bits, large):
    """Logits far beyond 2^24, whose float32 steps are wider than a weight's range: few rows and chunks, within a tile and over many. The
    weight is all on the largest logit where the next one lies further below it than both may be off (`bound`'s first term) and 64 more,
    which leaves e^-64 to the others; the output is then that key's value, but for the weight's 2^-19."""
    heads, kvh, hd = 4, 2, 64
    lens = [(3, 90), (100, 700), (70, 70)]
    c = Cache(wv, bits, 16, kvh, hd, lens)
    rng = np.random.default_rng(bits)
    n, total = sum(k for _, k in lens), sum(a for a, _ in lens)
    c.fill(*(torch.from_numpy(rng.normal(0, 1, (n, kvh * hd)).astype(np.float32)).cuda() for _ in range(2)))
    q = rng.normal(0, large, (total, heads, hd)).astype(np.float32)
    got = run_attn(c, torch.from_numpy(q.reshape(total, -1)).cuda(), heads, 0.125).reshape(total, heads, hd)
    assert np.isfinite(got).all()
    kk, vv = c.rows("k"), c.rows("v")
    r = a = clear = 0
    for nq, kv in lens:
        for i in range(nq):
            for h in range(heads):
                seen = slice(a, a + kv - nq + i + 1)
                x = kk[seen, h // 2] @ q[r + i, h].astype(np.float64) * 0.125
                off = 2 * hd * 2.0 ** -23 * (np.abs(kk[seen, h // 2]) @ np.abs(q[r + i, h].astype(np.float64))).max() * 0.125
                o = np.argsort(-x)
                if len(x) > 1 and x[o[0]] - x[o[1]] <= 2 * off + 64:
                    continue
                clear += 1
                v = vv[seen, h // 2]
                assert (np.abs(got[r + i, h] - v[o[0]]) <= 2.0 ** -19 * np.abs(v).max()).all(), (nq, i, h)
        r, a = r + nq, a + kv
    assert clear > total * heads * 0.9


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("far", [1e9, 1e20, 1e36])
def test_queries_far_larger_than_their_neighbours(wv, bits, far):
    """A query row's own magnitude is what its products are exact to: other rows, those of tokens that see nothing among them, do not
    matter, for 1 to 8 rows, up to 16, and chunks."""
    heads, kvh, hd = 4, 2, 64
    lens = [(2, 90), (7, 200), (5, 3), (100, 130), (90, 64)]
    c = Cache(wv, bits, 16, kvh, hd, lens)
    rng = np.random.default_rng(bits)
    n, total = sum(k for _, k in lens), sum(a for a, _ in lens)
    c.fill(*(torch.from_numpy(rng.normal(0, 1, (n, kvh * hd)).astype(np.float32)).cuda() for _ in range(2)))
    q = rng.normal(0, 1, (total, heads, hd)).astype(np.float32)
    r = 0
    for nq, kv in lens:
        q[r, 0], q[r, 3] = q[r, 0] * np.float32(far), q[r, 3] / np.float32(far)   # the first token: before position 0 in the third and fifth
        if nq > 60:
            q[r + 60, 1] *= np.float32(far)
        r += nq
    kk, vv = c.rows("k"), c.rows("v")
    for some in ([0], [1], [2], [3], [4], [0, 1, 2, 3, 4]):
        take = np.concatenate([np.arange(lens[i][0]) + sum(a for a, _ in lens[:i]) for i in some])
        part = [lens[i] for i in some]
        b, keep = c.batch_of(part)
        table = c.d_table[some].contiguous()
        b.pages = table.data_ptr()
        got = run_attn(c, torch.from_numpy(q[take].reshape(len(take), -1)).cuda(), heads, 0.125, batch=b).reshape(len(take), heads, hd)
        r = 0
        for i in some:
            nq, kv = lens[i]
            k0 = sum(k for _, k in lens[:i])
            want, mag, reach = attn64(q[take][r:r + nq], kk[k0:k0 + kv], vv[k0:k0 + kv], 0.125, 0, kv - nq)
            err = np.abs(got[r:r + nq] - want)
            assert (err <= bound(mag, reach, hd, kv)).all(), (some, i, float((err / bound(mag, reach, hd, kv)).max()))
            r += nq


def test_strides_and_rows_of_nobody(wv):
    """Gaps between rows stay as they are, and so do rows past the last sequence's."""
    heads, kvh, hd = 4, 2, 64
    for nq in (1, 60):
        lens = [(nq, 100), (nq, 64)]
        c = Cache(wv, 8, 16, kvh, hd, lens)
        c.fill(torch.randn(164, kvh * hd, device="cuda"), torch.randn(164, kvh * hd, device="cuda"))
        q = torch.randn(2 * nq + 3, heads * hd + 8, device="cuda")
        batch, keep = c.batch_of(lens, total=2 * nq + 3)
        got = run_attn(c, q, heads, 0.1, batch=batch, ldq=heads * hd + 8, ldo=heads * hd + 20)
        want = run_attn(c, q[:2 * nq, :heads * hd].contiguous(), heads, 0.1)
        assert np.array_equal(got[:2 * nq, :heads * hd], want)
        assert (got[:, heads * hd:] == 7.0).all() and (got[2 * nq:] == 7.0).all()


@pytest.mark.parametrize("bits", [16, 4])
def test_a_pool_beyond_4_gb(wv, bits):
    """Pages whose bytes start past 2^32: written, read back, and attended over by few rows and chunks as from a small pool."""
    lens, kvh, hd, page = [(1, 200), (60, 130)], 8, 128, 16
    n = sum(k for _, k in lens)
    gen = torch.Generator(device="cuda").manual_seed(bits)
    k, v, q = (torch.randn(r, w, device="cuda", generator=gen) for r, w in ((n, kvh * hd), (n, kvh * hd), (61, 16 * hd)))
    small = Cache(wv, bits, page, kvh, hd, lens)
    big = Cache(wv, bits, page, kvh, hd, lens)
    pages = 2 ** 32 // (kvh * big.bytes) + big.num_pages
    first = pages - big.num_pages
    big.pool = torch.zeros(pages, kvh, big.bytes, dtype=torch.uint8, device="cuda")
    big.table = np.where(big.table < 0, -1, big.table + first).astype(np.int32)
    big.d_table = torch.from_numpy(big.table).cuda()
    big.pages = wv.paged.KVPages(big.pool.data_ptr(), bits, pages, page, kvh, hd)
    big.batch, big.keep = big.batch_of(lens)
    back = []
    for c in (small, big):
        c.fill(k, v)
        b, keep = c.batch_of([(m, m) for _, m in lens])
        kv = [torch.zeros(n, kvh * hd, device="cuda") for _ in range(2)]
        wv.paged.KVReadCUDA(c.pages, b, kv[0].data_ptr(), kv[1].data_ptr())
        first_only, keep2 = c.batch_of([lens[0]])
        one, all_ = run_attn(c, q[:1], 16, 0.09, batch=first_only), run_attn(c, q, 16, 0.09)
        back.append([t.cpu().numpy() for t in kv] + [one, all_])
    assert not big.pool[:first].any() and torch.equal(big.pool[first:], small.pool)
    for a, b in zip(*back):
        assert np.array_equal(a, b) and np.isfinite(a).all() and a.any()
    assert wv._lib.lib().wv_device_status() == 0


def test_results_do_not_change_from_run_to_run(wv):
    for lens in ([(1, 3000), (1, 40)], [(300, 900)]):
        c = Cache(wv, 8, 16, 2, 128, lens)
        n = sum(k for _, k in lens)
        c.fill(torch.randn(n, 256, device="cuda"), torch.randn(n, 256, device="cuda"))
        q = torch.randn(sum(a for a, _ in lens), 1024, device="cuda")
        first = run_attn(c, q, 8, 0.09)
        for _ in range(3):
            assert np.array_equal(first, run_attn(c, q, 8, 0.09))


def test_a_second_stream_and_a_graph(wv):
    """Calls on two streams at once and a captured step whose lengths change between replays."""
    heads, kvh, hd = 8, 2, 128
    lens = [(1, 2000), (1, 500)]
    c = Cache(wv, 8, 16, kvh, hd, [(1, 3000), (1, 700)])
    c.fill(torch.randn(3700, kvh * hd, device="cuda"), torch.randn(3700, kvh * hd, device="cuda"))
    qs = [torch.randn(2, heads * hd, device="cuda") for _ in range(2)]
    want = [run_attn(c, q, heads, 0.09) for q in qs]
    st = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros(2, heads * hd, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, q, o in zip(st, qs, outs):
            wv.paged.AttnPagedCUDA(c.pages, c.batch, q.data_ptr(), o.data_ptr(), heads, 0.09, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(o.cpu().numpy(), w)
    g = torch.cuda.CUDAGraph()
    out = torch.zeros(2, heads * hd, device="cuda")
    with torch.cuda.graph(g, stream=st[0]):
        wv.paged.AttnPagedCUDA(c.pages, c.batch, qs[0].data_ptr(), out.data_ptr(), heads, 0.09, stream=torch.cuda.current_stream().cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want[0])
    c.keep[1].copy_(torch.tensor([k for _, k in lens], dtype=torch.int32))     # shorter now
    g.replay()
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), run_attn(c, qs[0], heads, 0.09))
    assert not np.array_equal(out.cpu().numpy(), want[0])


@pytest.mark.parametrize("nq", [1, 100])
def test_arrays_beyond_their_bounds_are_reported(wv, nq):
    """Page numbers outside the pool and lengths beyond the call's: cut and reported, and the next call is sound."""
    heads, kvh, hd = 4, 2, 64
    lens = [(nq, 200), (nq, 130)]
    c = Cache(wv, 8, 16, kvh, hd, lens)
    c.fill(torch.randn(330, kvh * hd, device="cuda"), torch.randn(330, kvh * hd, device="cuda"))
    q = torch.randn(2 * nq, heads * hd, device="cuda")
    L, check = wv._lib.lib(), wv._lib
    want = run_attn(c, q, heads, 0.1)
    assert L.wv_device_status() == 0
    for bad in (c.num_pages, -5):
        saved = int(c.d_table[0, 2])
        c.d_table[0, 2] = bad
        got = run_attn(c, q, heads, 0.1)
        assert L.wv_device_status() == check.WV_ESHAPE and np.array_equal(got[nq:], want[nq:]) and np.isfinite(got).all()
        b, keep = c.batch_of([(n, n) for _, n in lens])
        k = torch.randn(330, kvh * hd, device="cuda")
        before = c.pool.clone()
        wv.paged.KVWriteCUDA(c.pages, b, k.data_ptr(), k.data_ptr())
        back = torch.full((330, kvh * hd), 5.0, device="cuda")
        wv.paged.KVReadCUDA(c.pages, b, back.data_ptr(), torch.zeros_like(back).data_ptr())
        torch.cuda.synchronize()
        assert L.wv_device_status() == check.WV_ESHAPE
        assert (back[32:48] == 0).all() and (back[:32] != 0).any()
        c.pool.copy_(before)
        c.d_table[0, 2] = saved
    saved = c.keep[1].clone()
    for bad in (10 ** 9, -3):
        c.keep[1][1] = bad
        got = run_attn(c, q, heads, 0.1)
        assert L.wv_device_status() == check.WV_ESHAPE and np.array_equal(got[:nq], want[:nq])
    c.keep[1].copy_(saved)
    c.keep[0][2] = 10 ** 9
    run_attn(c, q, heads, 0.1)
    assert L.wv_device_status() == check.WV_ESHAPE
    c.keep[0][2] = 2 * nq
    assert np.array_equal(run_attn(c, q, heads, 0.1), want) and L.wv_device_status() == 0


def test_refusals(wv):
    P, E = wv.paged, wv.WelvetError
    c = Cache(wv, 8, 16, 2, 64, [(1, 20)])
    x = torch.zeros(4, 256, device="cuda")
    p = x.data_ptr()

    def code(f, *a, **k):
        with pytest.raises(E) as e:
            f(*a, **k)
        return e.value.code

    L = wv._lib
    assert code(P.KVBlockBytes, 5, 16, 64) == L.WV_EFORMAT
    for bad in ((8, 15, 64), (8, 0, 64), (8, 16, 72), (8, 16, 272), (8, 16, 0)):
        assert code(P.KVBlockBytes, *bad) == L.WV_ESHAPE
    assert P.KVBlockBytes(8, 16, 64) == 16 * (2 * 64 + 8) and P.KVBlockBytes(4, 32, 128) == 32 * (2 * 64 + 8 + 16)

    def pages(**k):
        d = dict(pool=c.pool.data_ptr(), bits=8, num_pages=c.num_pages, page_size=16, num_kv_heads=2, head_dim=64)
        d.update(k)
        return P.KVPages(*d.values())

    calls = [lambda pg, b, **k: P.KVWriteCUDA(pg, b, p, p, **k), lambda pg, b, **k: P.KVReadCUDA(pg, b, p, p, **k),
             lambda pg, b, **k: P.AttnPagedCUDA(pg, b, p, p, 4, 0.1, **k)]
    for f in calls:
        assert code(f, pages(bits=3), c.batch) == L.WV_EFORMAT
        for k in (dict(page_size=24), dict(head_dim=20), dict(num_pages=0), dict(num_kv_heads=0), dict(head_dim=512)):
            assert code(f, pages(**k), c.batch) == L.WV_ESHAPE
        assert code(f, pages(pool=0), c.batch) == L.WV_EARG
        assert code(f, pages(pool=c.pool.data_ptr() + 8), c.batch) == L.WV_EARG
        ok = [c.batch.q_start, c.batch.kv_len, c.batch.pages, 1, c.batch.table_stride, 1, 1, 20]
        for i, v, want in ((0, 0, L.WV_EARG), (1, 0, L.WV_EARG), (2, 0, L.WV_EARG), (3, 0, L.WV_EARG), (5, -1, L.WV_EARG), (6, -1, L.WV_EARG), (7, -1, L.WV_EARG),
                           (7, 16 * c.batch.table_stride + 1, L.WV_ESHAPE)):
            a = list(ok)
            a[i] = v
            assert code(f, pages(), P.Batch(*a)) == want
        a = list(ok)
        a[5] = 0
        f(pages(), P.Batch(*a))          # no rows: nothing to do
    assert code(P.KVWriteCUDA, c.pages, c.batch, 0, p) == L.WV_EARG
    assert code(P.KVWriteCUDA, c.pages, c.batch, p + 4, p) == L.WV_EARG
    assert code(P.KVWriteCUDA, c.pages, c.batch, p, p, ldk=64) == L.WV_ESHAPE
    assert code(P.KVWriteCUDA, c.pages, c.batch, p, p, ldk=130) == L.WV_ESHAPE
    assert code(P.KVWriteCUDA, c.pages, c.batch, p, p, p, 0, 4, 1e4) == L.WV_EARG
    assert code(P.KVWriteCUDA, c.pages, c.batch, p, p, p, p, 0, 1e4) == L.WV_ESHAPE
    assert code(P.KVWriteCUDA, c.pages, c.batch, p, p, theta=math.nan) == L.WV_EARG
    assert code(P.AttnPagedCUDA, c.pages, c.batch, p, p, 3, 0.1) == L.WV_ESHAPE
    assert code(P.AttnPagedCUDA, c.pages, c.batch, p, p, 0, 0.1) == L.WV_ESHAPE
    assert code(P.AttnPagedCUDA, c.pages, c.batch, p, p, 4, math.inf) == L.WV_EARG
    assert code(P.AttnPagedCUDA, c.pages, c.batch, p, 0, 4, 0.1) == L.WV_EARG
    assert code(P.AttnPagedCUDA, c.pages, c.batch, p, p, 4, 0.1, ldo=200) == L.WV_ESHAPE
