"""Low-rank adapters of many requests against 64 bits: every type, ranks from none to 256, tiles of 16 and of 64 rows, odd widths and strides,
rows without an adapter, in place and beside it, captured and replayed calls, and the refusals."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"f32": (1, torch.float32), "f16": (2, torch.float16), "bf16": (3, torch.bfloat16)}


class Set:
    """Adapters of several projections, what stands behind an adapter's rank being NaN."""

    def __init__(self, wv, dtype, slots, max_rank, k, outs, ranks=None, scale=True, seed=0):
        self.ad, self.slots, self.k, self.outs = wv.adapters, slots, k, outs
        code, t = TYPES[dtype]
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)
        rand = lambda *n: torch.randn(*n, device="cuda", generator=gen)  # noqa: E731
        self.ranks = [max_rank] * slots if ranks is None else ranks
        self.rank = None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device="cuda")
        off = torch.arange(max_rank, device="cuda") >= torch.tensor(self.ranks, device="cuda")[:, None]
        self.a = [rand(slots, max_rank, k).masked_fill(off[..., None], float("nan")).to(t) for _ in outs]
        self.b = [rand(slots, o, max_rank).masked_fill(off[:, None], float("nan")).to(t) for o in outs]
        self.scale = [rand(slots) if scale else None for _ in outs]
        p = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
        self.group = wv.adapters.Group([wv.adapters.Adapters(a.data_ptr(), b.data_ptr(), p(self.rank), p(s), slots, max_rank, k, o, code)
                                        for a, b, s, o in zip(self.a, self.b, self.scale, outs)])

    def want(self, x, slot, base):
        """(y, tolerance) in 64 bits. A product is exact to 2^-24; a chain of 64 columns adds 24 times (48 with float32 weights) and cuts, at most 2^-23 of the
        magnitudes each time, the chains of a warp, the warps and CTAs in / 512 + 16 times more; B's ranks add another 3 (6) a 16, 96 at most. All of
        that on the magnitudes |s| |B| (|A| |x|), the last sum on y's."""
        out = []
        for a, b, s, y0 in zip(self.a, self.b, self.scale, base):
            y, mag = y0.double().clone(), torch.zeros_like(y0, dtype=torch.float64)
            for i in sorted(set(v for v in slot if 0 <= v < self.slots)):
                rows, r = [j for j, v in enumerate(slot) if v == i], self.ranks[i]
                A, B, f = a[i, :r].double(), b[i, :, :r].double(), 1.0 if s is None else float(s[i])
                y[rows] += f * (x[rows].double() @ A.T @ B.T)
                mag[rows] += abs(f) * (x[rows].double().abs() @ A.abs().T @ B.abs().T)
            out.append((y, 2.0 ** -23 * ((160 + self.k / 512) * mag + y.abs()) + 1e-30))
        return out

    def plan(self, slot, stream=0):
        d = torch.tensor(list(slot) + [0], dtype=torch.int32, device="cuda")
        p = torch.full((self.ad.PlanBytes(len(slot), self.slots),), 255, dtype=torch.uint8, device="cuda")
        self.ad.PlanCUDA(d.data_ptr(), len(slot), self.slots, p.data_ptr(), stream=stream)
        return p, d


def up4(n):
    return -(-n // 4) * 4


def run(s, slot, inplace=False, seed=3, status=0):
    rows = len(slot)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    x = torch.randn(rows, s.k, device="cuda", generator=gen)
    base = [torch.randn(rows, up4(o), device="cuda", generator=gen) for o in s.outs]
    keep = [b.clone() for b in base]
    y = base if inplace else [torch.full_like(b, 55.0) for b in base]
    plan, _ = s.plan(slot)
    s.ad.ApplyCUDA(s.group, plan.data_ptr(), rows, x.data_ptr(), [v.data_ptr() for v in y], None if inplace else [b.data_ptr() for b in base], ldy=[up4(o) for o in s.outs])
    torch.cuda.synchronize()
    from welvet_b200 import _lib
    assert _lib.lib().wv_device_status() == status
    for (want, tol), got, b, k, o in zip(s.want(x, slot, [k[:, :o] for k, o in zip(keep, s.outs)]), y, base, keep, s.outs):
        err = (got[:, :o].double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())
        assert torch.equal(got[:, o:], k[:, o:]) if inplace else bool((got[:, o:] == 55).all())
        if not inplace:
            assert torch.equal(b, k)
        none = [i for i, v in enumerate(slot) if not 0 <= v < s.slots]
        assert torch.equal(got[none, :o], k[none, :o])
    return y


def mixed(rows, slots, seed=0):
    v = np.random.default_rng(seed).integers(-1, slots, rows)
    return [int(i) for i in v]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,slots,rank,k,outs", [
    (1, 1, 8, 8, [1]), (1, 3, 16, 4096, [512, 128, 128]), (7, 4, 8, 520, [33]), (16, 1, 24, 1000, [100, 7]), (17, 1, 64, 264, [300]),
    (64, 32, 16, 1024, [257, 64]), (40, 3, 72, 640, [96]), (5, 2, 256, 96, [130]), (3, 2, 32, 5000, [16, 15, 14, 13])])
def test_few_rows(wv, dtype, rows, slots, rank, k, outs):
    s = Set(wv, dtype, slots, rank, k, outs)
    run(s, mixed(rows, slots) if rows > 1 else [slots - 1])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,slots,rank,k,outs", [(65, 1, 16, 512, [200]), (333, 5, 24, 1400, [130, 77]), (300, 2, 64, 136, [1000]), (129, 2, 248, 72, [40]), (1000, 40, 8, 320, [64])])
def test_many_rows(wv, dtype, rows, slots, rank, k, outs):
    """Tiles of 64 rows, the last of an adapter's partly filled."""
    s = Set(wv, dtype, slots, rank, k, outs)
    run(s, sorted(mixed(rows, slots)))
    run(s, mixed(rows, slots, seed=1), inplace=True)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_ranks_of_their_own(wv, dtype):
    """Ranks from 0 to the largest; what stands behind an adapter's is NaN here and must not count. A scale of 1 where none is given."""
    ranks = [0, 1, 2, 3, 5, 7, 8, 9, 15, 16, 17, 31, 33, 40]
    for scale in (True, False):
        s = Set(wv, dtype, len(ranks), 40, 200, [50, 70], ranks=ranks, scale=scale)
        run(s, list(range(14)) + [-1, 3, 3], inplace=not scale)
        run(s, [i % 15 - 1 for i in range(600)])


def test_all_rows_without_an_adapter(wv):
    s = Set(wv, "bf16", 2, 8, 64, [40])
    run(s, [-1] * 70)
    run(s, [-1] * 3, inplace=True)


def test_every_run_is_the_same(wv):
    """The places of a plan's rows come from atomics; the results do not depend on them. Nor on the order of the call's rows."""
    s = Set(wv, "f16", 3, 16, 1000, [90])
    slot = mixed(900, 3)
    first = run(s, slot)[0]
    for _ in range(4):
        assert torch.equal(run(s, slot)[0], first)
    for rows in (14, 40):
        x, slot, order = torch.randn(rows, 1000, device="cuda"), mixed(rows, 3), np.random.default_rng(rows).permutation(rows)
        a, b = torch.zeros(rows, 92, device="cuda"), torch.zeros(rows, 92, device="cuda")
        p, _ = s.plan(slot)
        s.ad.ApplyCUDA(s.group, p.data_ptr(), rows, x.data_ptr(), [a.data_ptr()], ldy=[92])
        turned = torch.from_numpy(order).cuda()
        xt = x[turned].contiguous()
        p, _ = s.plan([slot[i] for i in order])
        s.ad.ApplyCUDA(s.group, p.data_ptr(), rows, xt.data_ptr(), [b.data_ptr()], ldy=[92])
        torch.cuda.synchronize()
        assert torch.equal(a[turned], b)


def test_strides(wv):
    s = Set(wv, "bf16", 3, 16, 104, [30, 41])
    rows, slot = 21, mixed(21, 3)
    x, base = torch.randn(rows, 120, device="cuda"), [torch.randn(rows, 36, device="cuda"), torch.randn(rows, 52, device="cuda")]
    y = [torch.full((rows + 1, w), 9.0, device="cuda") for w in (48, 44)]
    p, _ = s.plan(slot)
    s.ad.ApplyCUDA(s.group, p.data_ptr(), rows, x.data_ptr(), [v.data_ptr() for v in y], [b.data_ptr() for b in base], ldx=120, ldy=[48, 44], ldb=[36, 52])
    torch.cuda.synchronize()
    for (want, tol), got, o in zip(s.want(x[:, :104], slot, [b[:, :o] for b, o in zip(base, s.outs)]), y, s.outs):
        assert bool(((got[:rows, :o].double() - want).abs() <= tol).all())
        assert bool((got[:, o:] == 9).all()) and bool((got[rows:] == 9).all())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_magnitudes_and_values_that_are_not_finite(wv, dtype):
    """Rows of very different size keep their accuracy, a row that is not finite is NaN alone, and only where it has an adapter."""
    s = Set(wv, dtype, 2, 8, 64, [24])
    slot = [0, 1, 0, 1, -1, 0, 0, 1]
    x = torch.randn(8, 64, device="cuda")
    x[0] *= 1e-25
    x[1] *= 1e30
    x[2, 3], x[4, 0], x[7, 5] = float("inf"), float("nan"), float("nan")
    y = torch.zeros(8, 24, device="cuda")
    p, _ = s.plan(slot)
    s.ad.ApplyCUDA(s.group, p.data_ptr(), 8, x.data_ptr(), [y.data_ptr()])
    torch.cuda.synchronize()
    fine = [0, 1, 3, 5, 6]
    (want, tol), = s.want(torch.where(torch.isfinite(x), x, torch.zeros_like(x)), slot, [torch.zeros_like(y)])
    assert bool(((y.double() - want).abs() <= tol)[fine].all())
    assert torch.isnan(y[[2, 7]]).all() and not y[4].any()


def test_bounds_are_reported(wv):
    E = wv._lib
    s = Set(wv, "bf16", 3, 16, 64, [20], ranks=[16, 16, 16])
    run(s, [0, 3, 1, -2, 2, 10 ** 6, -2 ** 31], status=E.WV_ESHAPE)
    s.rank.copy_(torch.tensor([17, -1, 16]))             # cut to 16 and 0
    s.ranks = [16, 0, 16]
    run(s, [0, 1, 2], status=E.WV_ESHAPE)
    # a plan of other rows or adapters: nothing is done
    x, y = torch.randn(5, 64, device="cuda"), torch.full((5, 20), 3.0, device="cuda")
    for plan in (s.plan([0] * 4)[0], torch.zeros(4096, dtype=torch.uint8, device="cuda"), Set(wv, "bf16", 4, 16, 64, [20]).plan([0] * 5)[0]):
        s.ad.ApplyCUDA(s.group, plan.data_ptr(), 5, x.data_ptr(), [y.data_ptr()])
        torch.cuda.synchronize()
        assert E.lib().wv_device_status() == E.WV_ESHAPE and bool((y == 3).all())


def test_captured_and_replayed(wv):
    """Plan and apply in a graph, replayed with other rows' adapters and an adapter exchanged, beside the same calls on another stream."""
    s = Set(wv, "f16", 4, 16, 256, [64, 32], ranks=[16, 9, 3, 16])
    rows = 30
    x, slot = torch.randn(rows, 256, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    base = [torch.randn(rows, o, device="cuda") for o in s.outs]
    ys, graphs, plans = [], [], []
    st = torch.cuda.Stream()
    for _ in range(2):
        y, p = [torch.zeros_like(b) for b in base], torch.zeros(s.ad.PlanBytes(rows, 4), dtype=torch.uint8, device="cuda")
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st), torch.cuda.graph(g, stream=st):
            h = torch.cuda.current_stream().cuda_stream
            s.ad.PlanCUDA(slot.data_ptr(), rows, 4, p.data_ptr(), stream=h)
            s.ad.ApplyCUDA(s.group, p.data_ptr(), rows, x.data_ptr(), [v.data_ptr() for v in y], [b.data_ptr() for b in base], stream=h)
        ys.append(y), graphs.append(g), plans.append(p)
    for turn in range(3):
        now = mixed(rows, 4, seed=turn)
        slot.copy_(torch.tensor(now))
        if turn == 2:
            s.ranks[1] = 5
            s.rank[1] = 5
            s.a[0][1, :5].normal_(), s.b[0][1, :, :5].normal_(), s.scale[0][1].fill_(2.5)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        side = [torch.zeros_like(b) for b in base]
        p = torch.zeros(s.ad.PlanBytes(rows, 4), dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        s.ad.PlanCUDA(slot.data_ptr(), rows, 4, p.data_ptr(), stream=st.cuda_stream)
        s.ad.ApplyCUDA(s.group, p.data_ptr(), rows, x.data_ptr(), [v.data_ptr() for v in side], [b.data_ptr() for b in base], stream=st.cuda_stream)
        torch.cuda.synchronize()
        for (want, tol), a, b, c in zip(s.want(x, now, base), ys[0], ys[1], side):
            for got in (a, b, c):
                assert bool(((got.double() - want).abs() <= tol).all())


def test_more_rows_than_a_block_of_the_plan(wv):
    s = Set(wv, "bf16", 1500, 8, 32, [16])
    run(s, mixed(5000, 1500))
    s = Set(wv, "bf16", 2, 8, 32, [16])
    run(s, mixed(20001, 2))


def test_refusals(wv):
    E, L, ad = wv._lib, wv._lib.lib(), wv.adapters
    buf = torch.zeros(4096, device="cuda")
    p = buf.data_ptr()
    dy, ldy = (C.c_void_p * 2)(p, p), (C.c_int * 2)(32, 32)

    def call(code, n=1, plan=p, rows=2, dx=p, ldx=0, base=None, ldb=None, y=dy, strides=None, **k):
        f = {**dict(a=p, b=p, rank=0, scale=0, slots=2, max_rank=8, in_=16, out=32, dtype=3), **k}
        t = ad.Group([ad.Adapters(**f), ad.Adapters(p, p, 0, 0, 2, 8, 16, 32, 3)])
        assert L.wv_adapter_apply_dev(t, n, plan, rows, dx, ldx, base, ldb, y, strides, None) == getattr(E, code), L.wv_last_error()
    call("WV_OK", rows=0)
    for k in (dict(a=0), dict(b=0), dict(plan=None), dict(dx=None), dict(y=(C.c_void_p * 1)(None)), dict(base=(C.c_void_p * 1)(None)), dict(n=0), dict(n=5), dict(a=p + 8), dict(b=p + 4),
              dict(dx=p + 4), dict(plan=p + 8), dict(y=(C.c_void_p * 1)(p + 4)), dict(base=dy, ldb=(C.c_int * 1)(36), strides=ldy)):
        call("WV_EARG", **k)
    for k in (dict(rows=-1), dict(slots=0), dict(slots=8193), dict(in_=12), dict(in_=0), dict(max_rank=4), dict(max_rank=12), dict(max_rank=264), dict(out=0), dict(ldx=12), dict(ldx=18),
              dict(strides=(C.c_int * 1)(28)), dict(strides=(C.c_int * 1)(34)), dict(out=30), dict(n=2, slots=3), dict(n=2, in_=24), dict(n=2, dtype=2)):
        call("WV_ESHAPE", **k)
    call("WV_EFORMAT", dtype=4)
    call("WV_EFORMAT", dtype=0)
    # outputs that another target, or x, stands in: targets run side by side
    call("WV_EARG")
    other = (C.c_void_p * 2)(p + 4096, p + 8192)
    call("WV_EARG", n=2, y=(C.c_void_p * 2)(p + 4096, p + 4096))
    call("WV_EARG", n=2, y=other, base=(C.c_void_p * 2)(p + 8192, p + 8192))
    call("WV_EARG", n=2, y=(C.c_void_p * 2)(p + 4096, p))
    assert L.wv_adapter_plan_dev(None, 2, 2, p, None) == E.WV_EARG
    assert L.wv_adapter_plan_dev(p, 2, 2, None, None) == E.WV_EARG
    assert L.wv_adapter_plan_dev(p, 2, 2, p + 4, None) == E.WV_EARG
    assert L.wv_adapter_plan_dev(p, -1, 2, p, None) == E.WV_ESHAPE
    assert L.wv_adapter_plan_dev(p, 2, 9000, p, None) == E.WV_ESHAPE
    torch.cuda.synchronize()
