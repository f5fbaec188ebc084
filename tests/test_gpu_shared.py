"""Attention of sequences that share a prefix against the plain one in 64 bits: every width and head layout, few and many rows for either
part, groups of one and of many, sequences of no group, prefixes that end inside a page, short sequences, values that are not finite,
captured and replayed calls, and the refusals."""
import ctypes as C

import numpy as np
import pytest
import torch
from test_gpu_paged import Cache, attn64, bound

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def always(hooks):
    """The tests' sizes are too small for sharing to pay: take the shared keys apart all the same."""
    hooks.wv_set_attn_sharing(1)
    yield hooks.wv_set_attn_sharing
    hooks.wv_set_attn_sharing(0)


class Shared(Cache):
    """A cache whose sequences start[g] .. start[g + 1] - 1 name the same pages for their first shared[g] tokens."""

    def __init__(self, wv, bits, page, kvh, hd, lens, start, shared, seed=0):
        super().__init__(wv, bits, page, kvh, hd, lens, seed=seed)
        rng = np.random.default_rng(seed + 1)
        n = sum(k for _, k in lens)
        gen = lambda: torch.from_numpy(rng.normal(0, 1, (n, kvh * hd)).astype(np.float32)).cuda()  # noqa: E731
        self.fill(gen(), gen())
        for g, s in enumerate(shared):
            rows = [i for i in range(start[g], start[g + 1]) if lens[i][1]]
            for i in rows[1:]:
                # as far as both have whole pages of it
                common = min(s, lens[i][1], lens[rows[0]][1]) // page
                self.table[i, :common] = self.table[rows[0], :common]
        self.d_table.copy_(torch.from_numpy(self.table))
        self.share(start, shared)

    def share(self, start, shared, most=None):
        self.g = [torch.tensor(start, dtype=torch.int32, device="cuda"), torch.tensor(list(shared) + [0], dtype=torch.int32, device="cuda")]
        self.groups = self.wv.paged.Groups(self.g[0].data_ptr(), self.g[1].data_ptr(), len(shared), max(list(shared) + [0]) if most is None else most)

    def attend(self, q, heads, scale, batch=None, stream=0):
        out = torch.full_like(q, 77.0)
        self.wv.paged.AttnSharedCUDA(self.pages, batch or self.batch, self.groups, q.data_ptr(), out.data_ptr(), heads, scale, stream=stream)
        return out

    def want(self, q, heads, scale):
        k, v = self.rows("k"), self.rows("v")
        at, row, out, tol = 0, 0, [], []
        q = q.cpu().numpy().reshape(-1, heads, self.hd)
        for n, kv in self.lens:
            o, mag, reach = attn64(q[row:row + n], k[at:at + kv], v[at:at + kv], scale, 0, kv - n)
            out.append(o)
            tol.append(bound(mag, reach, self.hd, kv))
            at, row = at + kv, row + n
        return np.concatenate(out).reshape(row, -1), np.concatenate(tol).reshape(row, -1)

    def check(self, heads, seed=5, scale=None, q=None, floor=0.0):
        scale = self.hd ** -0.5 if scale is None else scale
        rows = sum(n for n, _ in self.lens)
        if q is None:
            q = torch.from_numpy(np.random.default_rng(seed).normal(0, 1, (rows, heads * self.hd)).astype(np.float32)).cuda()
        got = self.attend(q, heads, scale)
        torch.cuda.synchronize()
        assert self.wv._lib.lib().wv_device_status() == 0
        want, tol = self.want(q, heads, scale)
        tol = tol + floor
        err = np.abs(got.double().cpu().numpy() - want)
        assert np.array_equal(np.isnan(got.cpu().numpy()), np.isnan(want))
        assert (np.nan_to_num(err) <= np.nan_to_num(tol, nan=1.0)).all(), np.nanmax(err / tol)
        return got, q


# heads, kv heads, head_dim
LAYOUTS = [(8, 2, 64), (4, 4, 128), (12, 1, 80), (16, 2, 128), (6, 2, 48), (3, 1, 256)]


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("heads,kvh,hd", LAYOUTS)
def test_single_tokens(wv, bits, heads, kvh, hd):
    """Two groups, a sequence before, between and behind them, one slot without a sequence in a group."""
    lens = [(1, 50), (1, 400), (1, 333), (0, 0), (1, 321), (1, 20), (1, 700), (1, 690), (1, 1)]
    Shared(wv, bits, 16, kvh, hd, lens, [1, 5, 5, 6, 8], [320, 0, 17, 655]).check(heads)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("hd", [64, 128, 112])
def test_many_rows_share(wv, bits, hd):
    """A group of 40 sequences with two tokens each and eight heads: 640 rows a kv head, tiles that end inside a token, and a group of three."""
    lens = [(2, 600 + 3 * i) for i in range(40)] + [(2, 500), (1, 520), (2, 2)]
    Shared(wv, bits, 48, 1, hd, lens, [0, 40, 42], [576, 490]).check(8)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_chunks_behind_a_prefix(wv, bits):
    """Pieces of prompts behind a prefix: more than 32 rows a sequence, so that both parts go in tiles of 128, beside a single token."""
    lens = [(40, 700), (130, 900), (1, 641), (0, 650), (64, 64)]
    Shared(wv, bits, 32, 2, 128, lens, [0, 4], [640]).check(8)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_long_chunks_behind_a_prefix(wv, bits):
    """Pieces of prompts whose own keys are several tiles a block, the last ones masked, of ten blocks of rows a sequence."""
    Shared(wv, bits, 64, 2, 128, [(300, 2012), (290, 1800), (2, 900)], [0, 3], [512]).check(8)


@pytest.mark.parametrize("bits,spread", [(16, 0), (8, 0), (4, 0), (8, 15), (4, 15)])
def test_many_tiles_a_block(wv, bits, spread):
    """40 sequences of the same 16384 tokens: blocks go through several tiles of keys, the stages of their rings many times around. Three runs. With
    `spread` every fifth tile of 128 value rows has scales up to 2^30 apart, more than float16 pieces of the weights hold, between tiles that have not."""
    kvh, hd, heads, n, rows = 8, 128, 16, 16384, 40
    c = Cache(wv, bits, 64, kvh, hd, [(1, n)])
    rng = np.random.default_rng(bits)
    k, v = (rng.normal(0, 1, (n, kvh * hd)).astype(np.float32) for _ in range(2))
    if spread:
        v *= np.exp2(np.where(np.arange(n) // 128 % 5 == 3, rng.integers(-spread, spread + 1, n), 0)).astype(np.float32)[:, None]
    c.fill(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda())
    table = c.d_table[:1].repeat(rows, 1).contiguous()
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    start, kv, at, shared = ints(*range(rows + 1)), ints(*[n] * rows), ints(0, rows), ints(n, 0)
    batch = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), table.data_ptr(), rows, table.shape[1], rows, 1, n)
    groups = wv.paged.Groups(at.data_ptr(), shared.data_ptr(), 1, n)
    q = torch.from_numpy(rng.normal(0, 1, (rows, heads * hd)).astype(np.float32)).cuda()
    want, mag, reach = attn64(q.cpu().numpy().reshape(rows, heads, hd), c.rows("k"), c.rows("v"), hd ** -0.5, 0, n - 1)
    tol = bound(mag, reach, hd, n)
    first = None
    for _ in range(3):
        out = torch.full_like(q, 77.0)
        wv.paged.AttnSharedCUDA(c.pages, batch, groups, q.data_ptr(), out.data_ptr(), heads, hd ** -0.5)
        torch.cuda.synchronize()
        assert wv._lib.lib().wv_device_status() == 0
        assert (np.abs(out.double().cpu().numpy().reshape(want.shape) - want) <= tol).all()
        first = out if first is None else first
        assert torch.equal(out, first)


def test_chunks_of_wide_heads(wv):
    lens = [(40, 340), (9, 309), (1, 301)]
    Shared(wv, 8, 16, 1, 192, lens, [0, 3], [300]).check(4)


@pytest.mark.parametrize("shared", [0, 1, 15, 16, 31, 32, 33, 160, 10 ** 6])
def test_lengths_of_the_prefix(wv, shared):
    """From nothing to more than the sequences hold: whole pages count, as far as all new tokens see them (max_shared is cut to max_kv)."""
    lens = [(1, 170), (3, 165), (1, 161)]
    c = Shared(wv, 8, 16, 2, 64, lens, [0, 3], [min(shared, 160)])
    c.share([0, 3], [shared])
    if shared > 170:
        # a bound beyond max_kv is cut to it, and so would be its value: report it as any other length
        q = torch.randn(5, 8 * 64, device="cuda")
        c.attend(q, 8, 0.125)
        torch.cuda.synchronize()
        assert wv._lib.lib().wv_device_status() == wv._lib.WV_ESHAPE
        c.share([0, 3], [170])
        c.table[1:, :10] = c.table[0, :10]
    c.check(8)


def test_short_sequences_of_a_group(wv):
    """A sequence shorter than the prefix, and new tokens that lie inside it: what all rows see is less, the result is the same."""
    lens = [(1, 400), (1, 70), (1, 380)]
    Shared(wv, 8, 16, 1, 128, lens, [0, 3], [368]).check(4)
    lens = [(20, 300), (30, 290), (1, 320)]
    Shared(wv, 16, 16, 1, 128, lens, [0, 3], [288]).check(4)


def test_tokens_before_position_0(wv):
    """More new tokens than cached ones: the first stand before position 0 and see nothing."""
    lens = [(6, 4), (1, 200), (2, 199)]
    Shared(wv, 8, 16, 1, 64, lens, [1, 3], [192]).check(4)
    Shared(wv, 8, 16, 1, 64, lens, [0, 3], [192]).check(4)


def test_splits_planned_for_less(wv):
    """max_shared says that nearly all is shared, the device that nothing is: each of the few splits takes what it must. Also many splits of a
    long prefix with little behind it."""
    lens = [(1, 9000), (1, 8800), (2, 8700)]
    c = Shared(wv, 8, 64, 1, 64, lens, [0, 3], [8640])
    c.check(4)
    c.share([0, 3], [0], most=8640)
    c.check(4)
    c.share([0, 0], [8640])
    c.check(4)
    c.share([0], [])
    c.check(4)


def test_groups_of_one(wv):
    lens = [(1, 100 + i) for i in range(37)]
    Shared(wv, 4, 16, 2, 64, lens, list(range(38)), [96] * 37).check(4)


@pytest.mark.parametrize("rows", ["few", "many"])
def test_magnitudes(wv, rows):
    """Keys of one part far larger than the other's: one part's weight vanishes beside the other's, on either side. A weight counts to 2^-28 of its
    row's largest (the entry's stated range), and the divisor is at least the largest: where one key takes all, an output that its value
    leaves at zero may be off by 2^-28 of all values, kv 2^-28 max |v| at most."""
    n = 3 if rows == "few" else 40
    lens = [(1, 300 + i) for i in range(n)]
    for lo, hi in ((0, 240), (240, 10 ** 6)):
        c = Shared(wv, 8, 16, 1, 64, lens, [0, n], [240])
        k = [torch.from_numpy(np.random.default_rng(i).normal(0, 1, (sum(kv for _, kv in lens), 64)).astype(np.float32)).cuda() for i in range(2)]
        at = np.concatenate([np.arange(kv) for _, kv in lens])
        k[0][torch.from_numpy((at >= lo) & (at < hi)).cuda()] *= 30
        c.fill(*k)
        c.check(4, floor=max(kv for _, kv in lens) * 2.0 ** -28 * float(k[1].abs().max()))


def test_values_that_are_not_finite(wv):
    """A token of the prefix that is not finite makes every row of its group NaN and no other; one of a sequence's own keys that sequence's alone."""
    lens = [(1, 120), (1, 115), (1, 118), (1, 130)]
    c = Shared(wv, 8, 16, 1, 64, lens, [0, 3], [112])
    q = torch.randn(4, 4 * 64, device="cuda")
    blk = c.pool[int(c.table[1, 7]), 0]                                   # position 112, the second sequence's own
    blk[2 * 16 * 64:2 * 16 * 64 + 4].copy_(torch.tensor([float("nan")], device="cuda").view(torch.uint8))
    got = c.attend(q, 4, 0.125)
    assert torch.isnan(got).all(1).tolist() == [False, True, False, False] and not torch.isnan(got[[0, 2, 3]]).any()
    blk = c.pool[int(c.table[0, 2]), 0]                                   # a page of the prefix
    blk[2 * 16 * 64 + 64:2 * 16 * 64 + 68].copy_(torch.tensor([float("nan")], device="cuda").view(torch.uint8))
    got = c.attend(q, 4, 0.125)
    assert torch.isnan(got).all(1).tolist() == [True, True, True, False] and not torch.isnan(got[3]).any()
    q[0, 5] = float("inf")
    c = Shared(wv, 8, 16, 1, 64, lens, [0, 3], [112])
    got = c.attend(q, 4, 0.125)
    assert torch.isnan(got[0, :64]).all() and not torch.isnan(got[0, 64:]).any() and not torch.isnan(got[1:]).any()


def test_strides_and_rows_behind_the_last(wv):
    lens, heads, hd = [(1, 200), (2, 210), (1, 207)], 4, 64
    c = Shared(wv, 16, 16, 2, hd, lens, [0, 3], [192])
    w = heads * hd
    q, out = torch.randn(9, w + 20, device="cuda"), torch.full((9, w + 12), 55.0, device="cuda")
    b, keep = c.batch_of(lens, total=7)
    wv.paged.AttnSharedCUDA(c.pages, b, c.groups, q.data_ptr(), out.data_ptr(), heads, 0.125, ldq=w + 20, ldo=w + 12)
    torch.cuda.synchronize()
    want, tol = c.want(q[:4, :w].contiguous(), heads, 0.125)
    assert (np.abs(out[:4, :w].double().cpu().numpy() - want) <= tol).all()
    assert bool((out[4:] == 55).all()) and bool((out[:, w:] == 55).all())


def test_same_as_the_paged_attention_when_rows_are_many(wv):
    """More rows than the scratch holds two results for: the call is wv_attn_paged_dev."""
    lens = [(8192, 8300), (8192, 8310)]
    c = Shared(wv, 8, 64, 1, 128, [(1, 8300), (1, 8310)], [0, 2], [64])
    b, keep = c.batch_of(lens)
    q = torch.randn(16384, 16 * 128, device="cuda")
    got, ref = c.attend(q, 16, 0.09, b), torch.empty_like(q)
    wv.paged.AttnPagedCUDA(c.pages, b, q.data_ptr(), ref.data_ptr(), 16, 0.09)
    torch.cuda.synchronize()
    assert torch.equal(got, ref)


def test_loose_bounds_of_wide_heads(wv):
    """Three sequences of one token under bounds that allow 400 million tiles of sixteen rows: the call is wv_attn_paged_dev."""
    lens = [(1, 200), (1, 190), (1, 195)]
    c = Shared(wv, 8, 16, 1, 256, lens, [0, 3], [176])
    b, keep = c.batch_of(lens, max_q=1 << 28)
    q = torch.randn(3, 8 * 256, device="cuda")
    got, ref = c.attend(q, 8, 0.06, b), torch.empty_like(q)
    wv.paged.AttnPagedCUDA(c.pages, b, q.data_ptr(), ref.data_ptr(), 8, 0.06)
    torch.cuda.synchronize()
    assert torch.equal(got, ref) and wv._lib.lib().wv_device_status() == 0
    want, tol = c.want(q, 8, 0.06)
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("seqs,shared,pays", [(2, 512, False), (8, 512, False), (8, 4480, True)])
def test_shared_where_it_pays(wv, always, seqs, shared, pays):
    """By itself the call takes the shared keys apart for seven passes saved over 4480 keys of eight heads, and is wv_attn_paged_dev below that."""
    c = Shared(wv, 8, 64, 8, 128, [(1, shared + 30 + i) for i in range(seqs)], [0, seqs], [shared])
    q = torch.randn(seqs, 8 * 128, device="cuda")
    apart = c.attend(q, 8, 0.09)
    always(0)
    got, ref = c.attend(q, 8, 0.09), torch.empty_like(q)
    wv.paged.AttnPagedCUDA(c.pages, c.batch, q.data_ptr(), ref.data_ptr(), 8, 0.09)
    torch.cuda.synchronize()
    assert torch.equal(got, apart if pays else ref) and wv._lib.lib().wv_device_status() == 0
    c.share([0, seqs + 1], [shared])                                      # a group out of bounds is met only where groups are looked at
    c.attend(q, 8, 0.09)
    torch.cuda.synchronize()
    assert wv._lib.lib().wv_device_status() == (wv._lib.WV_ESHAPE if pays else 0)


def test_captured_and_replayed(wv):
    """Two graphs of the same call under the same bounds, replayed with other lengths, groups and tables, beside calls on a stream."""
    heads, cases = 8, [([(1, 300), (1, 280), (1, 290), (1, 40)], [0, 3], [272]), ([(1, 30), (1, 290), (1, 299), (1, 260)], [1, 4], [250]), ([(0, 0), (2, 300), (1, 100), (1, 300)], [0, 0], [0])]
    c = Shared(wv, 8, 16, 2, 64, *cases[0])
    start, kv = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    batch = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), c.d_table.data_ptr(), 4, c.table.shape[1], 4, 2, 300)
    c.groups.max_shared = 280
    q = torch.randn(4, heads * 64, device="cuda")
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    st = torch.cuda.Stream()
    for o in outs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st), torch.cuda.graph(g, stream=st):
            wv.paged.AttnSharedCUDA(c.pages, batch, c.groups, q.data_ptr(), o.data_ptr(), heads, 0.125, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    pool, table = c.pool, c.d_table
    for lens, first, shared in cases:
        d = Shared(wv, 8, 16, 2, 64, lens, first, shared, seed=len(lens) + shared[0])
        assert d.table.shape[1] <= table.shape[1] and d.num_pages <= c.num_pages
        pool[:d.num_pages] = d.pool
        table[:, :d.table.shape[1]] = d.d_table
        start.copy_(torch.tensor(np.concatenate([[0], np.cumsum([n for n, _ in lens])])))
        kv.copy_(torch.tensor([k for _, k in lens]))
        c.g[0].copy_(torch.tensor(first)), c.g[1].copy_(torch.tensor(shared + [0]))
        q.normal_()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        side = d.attend(q, heads, 0.125)
        torch.cuda.synchronize()
        assert wv._lib.lib().wv_device_status() == 0
        want, tol = d.want(q, heads, 0.125)
        for o in outs + [side]:
            assert (np.abs(o.double().cpu().numpy() - want) <= tol).all()


def test_bounds_are_cut_and_reported(wv):
    """Groups out of order, beyond the batch, a shared length beyond its bound or negative, a page outside the pool: an error and no fault; the
    sequences of no group keep their results."""
    lens = [(1, 100), (1, 120), (1, 110), (1, 90)]
    c = Shared(wv, 8, 16, 1, 64, lens, [0, 2], [96])
    q = torch.randn(4, 4 * 64, device="cuda")
    want, tol = c.want(q, 4, 0.125)
    for start, shared, most, fine in (([0, 9], [96], 96, []), ([2, 0], [96], 96, [0, 1, 3]), ([-5, 2], [96], 96, [2, 3]), ([0, 2], [97], 96, [2, 3]), ([0, 2], [-1], 96, [2, 3])):
        c.share(start, shared, most)
        got = c.attend(q, 4, 0.125)
        torch.cuda.synchronize()
        assert wv._lib.lib().wv_device_status() == wv._lib.WV_ESHAPE
        for r in fine:
            assert (np.abs(got[r].double().cpu().numpy() - want[r]) <= tol[r]).all()
    c.share([0, 2], [96])
    c.d_table[0, 1] = 10 ** 6
    got = c.attend(q, 4, 0.125)
    torch.cuda.synchronize()
    assert wv._lib.lib().wv_device_status() == wv._lib.WV_ESHAPE
    for r in (2, 3):
        assert (np.abs(got[r].double().cpu().numpy() - want[r]) <= tol[r]).all()


def test_refusals(wv):
    E, L, p = wv._lib, wv._lib.lib(), wv.paged
    c = Shared(wv, 8, 16, 2, 64, [(1, 40), (1, 44)], [0, 2], [32])
    q = torch.zeros(2, 8 * 64, device="cuda")

    def call(code, pages=c.pages, batch=c.batch, groups=c.groups, dq=q.data_ptr(), ldq=0, heads=8, scale=0.1):
        got = L.wv_attn_shared_dev(C.byref(pages), C.byref(batch), C.byref(groups) if groups is not None else None, dq, ldq, q.data_ptr(), 0, heads, scale, None)
        assert got == getattr(E, code)
    a, b = c.g[0].data_ptr(), c.g[1].data_ptr()
    call("WV_EARG", groups=None)
    for g in (p.Groups(0, b, 1, 32), p.Groups(a, 0, 1, 32), p.Groups(a, b, -1, 32), p.Groups(a, b, 3, 32), p.Groups(a, b, 1, -1)):
        call("WV_EARG", groups=g)
    call("WV_ESHAPE", heads=7)
    call("WV_ESHAPE", heads=0)
    call("WV_EARG", scale=float("inf"))
    call("WV_EARG", dq=0)
    call("WV_ESHAPE", ldq=8 * 64 - 4)
    call("WV_EARG", dq=q.data_ptr() + 4)
    call("WV_EFORMAT", pages=p.KVPages(c.pool.data_ptr(), 5, 4, 16, 2, 64))
    call("WV_OK", groups=p.Groups(0, 0, 0, 0))
    call("WV_OK", batch=p.Batch(c.keep[0].data_ptr(), c.keep[1].data_ptr(), c.d_table.data_ptr(), 2, c.table.shape[1], 0, 1, 44))
    torch.cuda.synchronize()
