"""Page tables on the device: fork, extend, trim and compact against the same steps on the host, one sequence after the other, with the
pools' bytes; runs of random steps under pressure, bad entries, captured and replayed calls, and the refusals."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


class Host:
    """The rules of the header, in order, on numpy arrays."""

    def __init__(self, num_pages, page, slots, stride, pools):
        self.refs, self.pages, self.kv = np.zeros(num_pages, np.int64), np.full((slots, stride), -1, np.int64), np.zeros(slots, np.int64)
        self.page, self.pools = page, pools

    def held(self, n):
        return -(-int(n) // self.page)

    def trim(self, seqs, keep):
        for s, k in zip(seqs, keep):
            for j in range(self.held(k), self.held(self.kv[s])):
                self.refs[self.pages[s, j]] -= 1
                self.pages[s, j] = -1
            self.kv[s] = min(self.kv[s], k)

    def fork(self, src, dst, keep=None):
        for i, (a, b) in enumerate(zip(src, dst)):
            n = self.kv[a] if keep is None else min(self.kv[a], keep[i])
            for j in range(self.held(n)):
                self.pages[b, j] = self.pages[a, j]
                self.refs[self.pages[a, j]] += 1
            self.kv[b] = n

    def extend(self, add):
        free = [p for p in range(len(self.refs)) if self.refs[p] == 0]
        refs, asked, at, ok = self.refs.copy(), 0, 0, np.ones(len(add), np.int64)
        for s, n in enumerate(add):
            if n == 0:
                continue
            held, want = self.held(self.kv[s]), self.held(self.kv[s] + n)
            copy = self.kv[s] % self.page != 0 and refs[self.pages[s, held - 1]] > 1
            if want > self.pages.shape[1]:
                ok[s] = 0
                continue
            asked += want - held + copy
            if want - held + copy and asked > len(free):
                ok[s] = 0
                continue
            if copy:
                old, new = self.pages[s, held - 1], free[at]
                at += 1
                self.refs[old] -= 1
                self.refs[new] = 1
                self.pages[s, held - 1] = new
                for p in self.pools:
                    p[new] = p[old]
            for j in range(held, want):
                self.pages[s, j] = free[at]
                self.refs[free[at]] = 1
                at += 1
            self.kv[s] += n
        return ok

    def compact(self):
        live = int((self.refs > 0).sum())
        src = [p for p in range(live, len(self.refs)) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
            for p in self.pools:
                p[b] = p[a]
        for s in range(len(self.kv)):
            for j in range(self.held(self.kv[s])):
                self.pages[s, j] = to.get(self.pages[s, j], self.pages[s, j])
        return live


class Both:
    """A table on the device beside the host's, and pools of several widths."""

    def __init__(self, wv, num_pages, page, slots, stride, shapes=((8, 2, 64), (4, 1, 128), (16, 3, 48)), seed=0):
        self.p, self.slots, self.num_pages = wv.paged, slots, num_pages
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        z = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.refs, self.pages, self.kv = z(num_pages), z(slots, stride) - 1, z(slots)
        self.pools = [torch.randint(0, 256, (num_pages, k * wv.paged.KVBlockBytes(b, page, hd)), dtype=torch.uint8, device="cuda", generator=gen) for b, k, hd in shapes]
        self.blocks = wv.paged.KVBlocks([wv.paged.KVPages(t.data_ptr(), b, num_pages, page, k, hd) for t, (b, k, hd) in zip(self.pools, shapes)])
        self.table = wv.paged.KVTable(self.refs.data_ptr(), self.pages.data_ptr(), self.kv.data_ptr(), num_pages, page, slots, stride)
        self.host = Host(num_pages, page, slots, stride, [t.cpu().numpy() for t in self.pools])
        self.status = wv._lib.lib().wv_device_status

    @staticmethod
    def ints(v):
        return torch.tensor(list(v), dtype=torch.int32, device="cuda")

    def trim(self, seqs, keep):
        a, b = self.ints(seqs), self.ints(keep)
        self.p.KVTrimCUDA(self.table, len(seqs), b.data_ptr(), a.data_ptr())
        torch.cuda.synchronize()
        self.host.trim(seqs, keep)

    def fork(self, src, dst, keep=None):
        a, b, k = self.ints(src), self.ints(dst), None if keep is None else self.ints(keep)
        self.p.KVForkCUDA(self.table, a.data_ptr(), b.data_ptr(), len(src), 0 if k is None else k.data_ptr())
        torch.cuda.synchronize()
        self.host.fork(src, dst, keep)

    def extend(self, add):
        a, ok = self.ints(add), self.ints([7] * self.slots)
        self.p.KVExtendCUDA(self.table, a.data_ptr(), ok.data_ptr(), self.blocks)
        torch.cuda.synchronize()
        want = self.host.extend(add)
        assert ok.tolist() == want.tolist()
        return want

    def compact(self):
        live = self.ints([-1])
        self.p.KVCompactCUDA(self.table, self.blocks, live.data_ptr())
        torch.cuda.synchronize()
        assert int(live) == self.host.compact()

    def same(self, status=0):
        torch.cuda.synchronize()
        assert self.status() == status
        h = self.host
        assert self.refs.tolist() == h.refs.tolist() and self.kv.tolist() == h.kv.tolist()
        assert np.array_equal(self.pages.cpu().numpy(), h.pages)
        # what a call gave up stays in the pools: compare the pages that are held, and that no others changed
        for t, p in zip(self.pools, h.pools):
            assert np.array_equal(t.cpu().numpy(), p)
        held = np.zeros(len(h.refs), np.int64)
        for s in range(self.slots):
            for j in range(h.held(h.kv[s])):
                held[h.pages[s, j]] += 1
        assert np.array_equal(held, h.refs)


@pytest.mark.parametrize("page", [16, 48])
def test_fork_extend_trim(wv, page):
    """A sequence forked three times, at its end, inside its last page and at a page's end; all of them extended, and the forks freed."""
    b = Both(wv, 40, page, 6, 8)
    b.extend([2 * page + 5, 0, 0, 0, 0, 0])
    b.same()
    b.fork([0, 0, 0, 0], [1, 2, 3, 4], [10 ** 6, 2 * page + 1, 2 * page, 0])
    b.same()
    b.extend([1, 1, 1, 1, 1, page])
    b.same()
    b.extend([page - 6, page, 2 * page, 3 * page, 1, 0])
    b.same()
    b.trim([1, 2, 3, 0], [page + 1, 0, 10 ** 6, page])
    b.same()
    b.trim([0, 1, 2, 3, 4, 5], [0] * 6)
    b.same()
    assert int(b.refs.abs().sum()) == 0


def test_all_of_them_freed_without_lists(wv):
    b = Both(wv, 30, 16, 5, 6)
    b.extend([16, 17, 0, 90, 5])
    b.p.KVTrimCUDA(b.table, 5)
    b.host.trim(range(5), [0] * 5)
    b.same()


def test_extend_is_refused_in_order(wv):
    """Rows of the table that are too short refuse their sequence alone; then two pages are free: the third sequence's need passes them, so do those
    behind it that need a page, and ones that need none go on."""
    b = Both(wv, 10, 16, 7, 4)
    b.extend([20, 16, 0, 0, 0, 0, 0])
    b.same()
    got = b.extend([45, 60, 16, 33, 1, 0, 65])           # 65, 76 and 65 tokens do not fit four pages
    b.same()
    assert got.tolist() == [0, 0, 1, 1, 1, 1, 0]
    assert b.extend([0, 32, 17, 1, 1, 16, 16]).tolist() == [1, 1, 0, 1, 1, 0, 0]
    b.same()
    assert b.extend([12, 0, 0, 0, 0, 0, 0])[0] == 1      # inside its last page
    b.same()


def test_copies_of_shared_last_pages_that_do_not_fit(wv):
    """Four forks share a partly filled page and two pages are free: two of them get their copy, the others stay where they are."""
    b = Both(wv, 3, 16, 4, 2)
    b.extend([5, 0, 0, 0])
    b.fork([0, 0, 0], [1, 2, 3])
    b.same()
    assert b.extend([1, 1, 1, 1]).tolist() == [1, 1, 0, 0]
    b.same()


@pytest.mark.parametrize("seed", range(6))
def test_random_steps(wv, seed):
    """Steps as a server takes them, on a pool that runs full; pages, counts, lengths and every byte of the pools as on the host."""
    rng = np.random.default_rng(seed)
    page, slots, stride, num_pages = [(16, 33, 9, 150), (32, 700, 3, 900), (48, 5, 40, 61), (16, 64, 5, 129), (64, 20, 7, 4200), (16, 1, 3, 1)][seed]
    b = Both(wv, num_pages, page, slots, stride, shapes=((8, 1, 16), (4, 2, 16)), seed=seed)
    for _ in range(12):
        b.extend([int(v) for v in np.where(rng.random(slots) < 0.6, rng.integers(0, 2 * page, slots), 0)])
        empty = [int(s) for s in rng.permutation(slots) if b.host.kv[s] == 0]
        full = [int(s) for s in rng.permutation(slots) if b.host.kv[s] > 0]
        if full and empty:
            dst = empty[:max(1, len(empty) // 3)]
            src = [int(rng.choice(full)) for _ in dst]
            b.fork(src, dst, [int(rng.integers(0, stride * page)) for _ in dst] if rng.random() < 0.5 else None)
        b.same()
        if full:
            cut = full[:max(1, len(full) // 2)]
            b.trim(cut, [int(rng.integers(0, stride * page)) if rng.random() < 0.5 else 0 for _ in cut])
        if rng.random() < 0.5:
            b.compact()
        b.same()


def test_compact_of_a_large_pool(wv):
    """More pages than the cluster has threads, held ones scattered over the pool and shared by two sequences."""
    b = Both(wv, 70001, 16, 400, 100, shapes=((8, 1, 16),))
    rng = np.random.default_rng(1)
    order = rng.permutation(70001)
    h, at = b.host, 0
    for s in range(0, 400, 2):
        n = int(rng.integers(1, 101))
        for t in (s, s + 1):
            h.pages[t, :n] = order[at:at + n]
            h.kv[t] = 16 * n - 3
        h.refs[order[at:at + n]] = 2
        at += n
    b.refs.copy_(torch.from_numpy(h.refs)), b.pages.copy_(torch.from_numpy(h.pages)), b.kv.copy_(torch.from_numpy(h.kv))
    b.compact()
    b.same()
    assert not b.refs[at:].any() and bool((b.refs[:at] == 2).all())
    b.compact()                                          # nothing to do
    b.same()
    b.extend([1 if s % 2 else 40 for s in range(400)])
    b.same()


def test_compact_without_pools_and_empty(wv):
    b = Both(wv, 50, 16, 3, 9, shapes=())
    b.compact()
    b.extend([16 * 9, 20, 100])
    b.trim([0], [3])
    b.p.KVCompactCUDA(b.table, None, b.ints([0]).data_ptr())
    b.host.compact()
    b.same()


def test_bad_entries_are_left_out(wv):
    """A sequence's number out of range, a target twice, a target that is not empty or is a source, a negative length: each is reported and
    changes nothing; the entries beside it count."""
    b = Both(wv, 40, 16, 8, 4)
    b.extend([20, 33, 0, 0, 0, 0, 7, 0])
    b.same()
    a, d, k = b.ints([0, 0, 1, 9, 0, 3, 0, 7]), b.ints([2, 2, 3, 4, -1, 5, 6, 7]), b.ints([5, 7, 40, 1, 1, 1, 1, 1])
    b.p.KVForkCUDA(b.table, a.data_ptr(), d.data_ptr(), 8, k.data_ptr())
    b.host.fork([0, 1], [2, 3], [5, 40])                 # 3 is a target and so no source; 6 is not empty
    b.same(wv._lib.WV_ESHAPE)
    a, k = b.ints([0, 0, 8, -3, 1]), b.ints([4, 0, 1, 1, -1])
    b.p.KVTrimCUDA(b.table, 5, k.data_ptr(), a.data_ptr())
    b.host.trim([0], [4])
    b.same(wv._lib.WV_ESHAPE)
    add, ok = b.ints([-1, 2, 2 ** 31 - 1, 0, 65, 64, 0, 0]), b.ints([9] * 8)
    b.p.KVExtendCUDA(b.table, add.data_ptr(), ok.data_ptr(), b.blocks)
    torch.cuda.synchronize()
    want = b.host.extend([0, 2, 0, 0, 65, 64, 0, 0])
    want[[0, 2]] = 0
    assert ok.tolist() == want.tolist()
    b.same(wv._lib.WV_ESHAPE)
    # counts and page numbers that do not fit one another: nothing outside the table is touched
    b.refs.zero_()
    b.pages[1, 0] = 4000
    b.p.KVTrimCUDA(b.table, 8)
    torch.cuda.synchronize()
    assert b.status() == wv._lib.WV_ESHAPE
    assert int(b.refs.abs().sum()) == 0 and int(b.kv.abs().sum()) == 0


def test_copy(wv):
    b = Both(wv, 20, 16, 1, 1)
    before = [t.clone() for t in b.pools]
    src, dst = b.ints([3, 3, 19, 7, 5, 25, 1]), b.ints([4, 0, 18, 7, -1, 2, 20])
    b.p.KVCopyCUDA(b.blocks, src.data_ptr(), dst.data_ptr(), 7)
    torch.cuda.synchronize()
    assert b.status() == wv._lib.WV_ESHAPE
    for t, u in zip(b.pools, before):
        u[4], u[0], u[18] = u[3].clone(), u[3].clone(), u[19].clone()
        assert torch.equal(t, u)
    b.p.KVCopyCUDA(b.blocks, 0, 0, 0)


def test_many_pools_and_large_pages(wv):
    """More pools than a launch takes, and pages of more items than one."""
    n, page = 131, 16
    pools = [torch.randint(0, 256, (3, wv.paged.KVBlockBytes(16, page, 256) * (1 + i % 3)), dtype=torch.uint8, device="cuda") for i in range(n)]
    want = [t[0].clone() for t in pools]
    blocks = wv.paged.KVBlocks([wv.paged.KVPages(t.data_ptr(), 16, 3, page, 1 + i % 3, 256) for i, t in enumerate(pools)])
    src, dst = Both.ints([0]), Both.ints([2])
    wv.paged.KVCopyCUDA(blocks, src.data_ptr(), dst.data_ptr(), 1)
    torch.cuda.synchronize()
    assert all(torch.equal(t[2], w) for t, w in zip(pools, want))


def test_captured_and_replayed(wv):
    """Trim, fork and extend in one graph beside a second graph of the same calls on another table: the replays follow the contents."""
    sides = [Both(wv, 60 + i, 16, 6, 6, seed=i) for i in range(2)]
    graphs = []
    for b in sides:
        b.extend([21, 0, 0, 0, 0, 0])
        b.arg = [b.ints([1, 2]), b.ints([0, 0]), b.ints([0, 0]), b.ints([0, 1, 1, 0, 0, 0]), b.ints([0] * 6), b.ints([0])]
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                s = torch.cuda.current_stream().cuda_stream
                dst, keep, src, add, ok, live = (t.data_ptr() for t in b.arg)
                b.p.KVTrimCUDA(b.table, 2, keep, dst, stream=s)
                b.p.KVForkCUDA(b.table, src, dst, 2, stream=s)
                b.p.KVExtendCUDA(b.table, add, ok, b.blocks, stream=s)
                b.p.KVCompactCUDA(b.table, b.blocks, live, stream=s)
        graphs.append(g)
    for turn in range(3):
        for b, g in zip(sides, graphs):
            b.arg[3].copy_(b.ints([turn, 1 + turn, 20, 0, 3, 0]))
            torch.cuda.synchronize()
            g.replay()
        torch.cuda.synchronize()
        for b in sides:
            b.host.trim([1, 2], [0, 0])
            b.host.fork([0, 0], [1, 2])
            assert b.arg[4].tolist() == b.host.extend([turn, 1 + turn, 20, 0, 3, 0]).tolist()
            assert int(b.arg[5]) == b.host.compact()
            b.same()


def test_two_streams_at_once(wv):
    """Two tables on two streams, each with scratch of its own."""
    sides, streams = [Both(wv, 3000, 16, 200, 20, shapes=((8, 1, 16),), seed=i) for i in range(2)], [torch.cuda.Stream() for _ in range(2)]
    adds = [[[int(v) for v in np.random.default_rng(10 * i + k).integers(0, 40, 200)] for k in range(5)] for i in range(2)]
    dev = [[b.ints(a) for a in adds[i]] for i, b in enumerate(sides)]
    torch.cuda.synchronize()
    for k in range(5):
        for i, b in enumerate(sides):
            b.p.KVExtendCUDA(b.table, dev[i][k].data_ptr(), 0, b.blocks, stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i, b in enumerate(sides):
        for a in adds[i]:
            b.host.extend(a)
        b.same()


def test_refusals(wv):
    E, L, p = wv._lib, wv._lib.lib(), wv.paged
    b = Both(wv, 8, 16, 2, 2)
    one, t = b.ints([0, 0]).data_ptr(), C.byref(b.table)
    bad = lambda **k: C.byref(p.KVTable(**{**dict(refs=one, pages=one, kv_len=one, num_pages=8, page_size=16, num_seqs=2, table_stride=2), **k}))  # noqa: E731
    for k in (dict(refs=0), dict(pages=0), dict(kv_len=0)):
        assert L.wv_kv_trim_dev(bad(**k), None, None, 1, None) == E.WV_EARG
        assert L.wv_kv_fork_dev(bad(**k), one, one, None, 1, None) == E.WV_EARG
        assert L.wv_kv_extend_dev(bad(**k), one, None, None, 0, None) == E.WV_EARG
        assert L.wv_kv_compact_dev(bad(**k), None, 0, one, None) == E.WV_EARG
    for k in (dict(num_pages=0), dict(page_size=24), dict(page_size=0), dict(num_seqs=0), dict(table_stride=0)):
        assert L.wv_kv_trim_dev(bad(**k), None, None, 0, None) == E.WV_ESHAPE
        assert L.wv_kv_compact_dev(bad(**k), None, 0, one, None) == E.WV_ESHAPE
    assert L.wv_kv_trim_dev(t, None, None, 3, None) == E.WV_ESHAPE
    assert L.wv_kv_trim_dev(t, None, None, -1, None) == E.WV_ESHAPE
    assert L.wv_kv_fork_dev(t, one, one, None, 3, None) == E.WV_ESHAPE
    assert L.wv_kv_fork_dev(t, None, one, None, 1, None) == E.WV_EARG
    assert L.wv_kv_extend_dev(t, None, None, None, 0, None) == E.WV_EARG
    assert L.wv_kv_extend_dev(t, one, None, None, 1, None) == E.WV_EARG
    assert L.wv_kv_compact_dev(t, None, 0, None, None) == E.WV_EARG
    pool = b.pools[0].data_ptr()
    for args, code in (((pool, 8, 9, 16, 2, 64), "WV_ESHAPE"), ((pool, 8, 8, 32, 2, 64), "WV_ESHAPE"), ((pool, 7, 8, 16, 2, 64), "WV_EFORMAT"), ((0, 8, 8, 16, 2, 64), "WV_EARG"),
                       ((pool + 8, 8, 8, 16, 2, 64), "WV_EARG"), ((pool, 8, 8, 16, 0, 64), "WV_ESHAPE"), ((pool, 8, 8, 16, 2, 60), "WV_ESHAPE")):
        blocks = p.KVBlocks([p.KVPages(*args)])
        assert L.wv_kv_extend_dev(t, one, None, blocks, 1, None) == getattr(E, code)
        assert L.wv_kv_compact_dev(t, blocks, 1, one, None) == getattr(E, code)
    assert L.wv_kv_copy_dev(b.blocks, 0, one, one, 1, None) == E.WV_EARG
    assert L.wv_kv_copy_dev(b.blocks, 3, one, one, -1, None) == E.WV_ESHAPE
    assert L.wv_kv_copy_dev(b.blocks, 3, None, one, 1, None) == E.WV_EARG
    torch.cuda.synchronize()
    b.same()
