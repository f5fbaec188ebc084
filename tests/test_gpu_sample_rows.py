"""Sampling many rows at once against the definition in 64 bits: every cut alone and together, ties, values that are not finite,
rows without a candidate, sizes around the kernel's limits, and the refusals."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def sample64(x, t, k, p, mp, u):
    """Candidates in order, their weights exp((x - max) / t) with the float32 steps that welvet_cuda.h states (logit / T, difference),
    everything else in 64 bits. Returns (index, prob, margin): margin is the distance of the draw and of the top-p line from the
    nearest running sum, relative to the sum."""
    x = np.asarray(x, np.float32)
    cand = np.flatnonzero(~np.isnan(x) & (x > -np.inf))
    if not len(cand):
        return -1, 0.0, 1.0
    greedy = t <= 0 or k == 1
    with np.errstate(over="ignore", invalid="ignore"):
        y = x[cand] if greedy else x[cand] / np.float32(t)
    keep = ~np.isnan(y)
    cand, y = cand[keep], y[keep]
    if not len(cand):
        return -1, 0.0, 1.0
    o = np.argsort(-y, kind="stable")
    cand, y = cand[o], y[o]
    if greedy:
        return int(cand[0]), 1.0, 1.0
    if k > 0:
        cand, y = cand[:k], y[:k]
    with np.errstate(invalid="ignore"):
        w = np.where(y == y[0], 1.0, np.exp((y - y[0]).astype(np.float64)))
    run = np.cumsum(w)
    margin = 1.0
    keep = np.ones(len(w), bool)
    if not p >= 1:
        line = float(np.float32(p)) * run[-1]
        keep = run - w < line
        margin = min(margin, np.abs(run - line).min() / run[-1])
    keep &= w >= float(np.float32(mp))
    keep[0] = True
    margin = min(margin, np.abs(w - float(np.float32(mp))).min() if mp > 0 else 1.0)
    w, cand = w[keep], cand[keep]
    run = np.cumsum(w)
    r = u * run[-1]
    i = int(np.argmax(run >= r)) if (run >= r).any() else len(w) - 1
    margin = min(margin, np.abs(run - r).min() / run[-1])
    return int(cand[i]), w[i] / run[-1], margin


def run_rows(wv, x, t, k, p, mp, u, ld=0, prob=True):
    rows, n = x.shape if not ld else (x.shape[0], None)
    dev = lambda v, ty: torch.tensor(np.asarray(v), dtype=ty, device="cuda")  # noqa: E731
    d = [dev(t, torch.float32), dev(k, torch.int32), dev(p, torch.float32), dev(mp, torch.float32), dev(u, torch.float64)]
    idx, pr = torch.full((rows,), -7, dtype=torch.int32, device="cuda"), torch.full((rows,), -7.0, device="cuda")
    wv.sampling.SampleRowsCUDA(x.data_ptr(), rows, n or ld[0], *[v.data_ptr() for v in d], idx.data_ptr(), pr.data_ptr() if prob else 0, ld=ld[1] if ld else 0)
    torch.cuda.synchronize()
    return idx.cpu().numpy(), pr.cpu().numpy()


def check_rows(wv, x, t, k, p, mp, u):
    got, prob = run_rows(wv, torch.from_numpy(x).cuda(), t, k, p, mp, u)
    n, far = x.shape[1], 0
    for r in range(len(x)):
        want, pw, margin = sample64(x[r], t[r], k[r], p[r], mp[r], u[r])
        # a weight is exp in float32, off by 2 units of 2^-24 at most, and rounded to 2^-(62 - log2 n): where a line is nearer
        # than that to a running sum, either neighbour is right
        if margin < 4 * 2.0 ** -23:
            far += 1
            continue
        assert got[r] == want, (r, got[r], want, t[r], k[r], p[r], mp[r], u[r])
        assert abs(prob[r] - pw) <= 2.0 ** -21 * pw + 1e-30
    assert far <= max(2, len(x) // 4)


@pytest.mark.parametrize("n", [1, 2, 33, 1000, 1024, 1025, 8192, 8193, 50257, 128256])
def test_every_cut(wv, n):
    rng = np.random.default_rng(n)
    rows = 48
    x = (rng.normal(0, 1, (rows, n)) * rng.choice([0.5, 2, 6], (rows, 1))).astype(np.float32)
    t = rng.choice([0.0, 0.3, 0.8, 1.0, 2.0, -1.0], rows)
    k = rng.choice([0, -3, 1, 2, 7, 40, 1024, 5000, n, n + 5], rows)
    p = rng.choice([0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 1.5], rows)
    mp = rng.choice([0.0, 0.0, 0.01, 0.3, 1.0, 1.5], rows)
    check_rows(wv, x, t, k, p, mp, rng.random(rows))


@pytest.mark.parametrize("n", [5, 700, 20000])
@pytest.mark.parametrize("k,p,mp", [(0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.8, 0.0), (0, 1.0, 0.05), (300, 0.9, 0.001)])
def test_draws_follow_the_distribution(wv, n, k, p, mp):
    """A grid of draws over one row: every token comes as often as its weight says, to one draw at each end."""
    rng = np.random.default_rng(n + k)
    row = rng.normal(0, 2, n).astype(np.float32)
    draws = 4000
    x = torch.from_numpy(row).cuda().repeat(draws, 1)
    full = lambda v: np.full(draws, v)  # noqa: E731
    got, _ = run_rows(wv, x, full(1.1), full(k), full(p), full(mp), (np.arange(draws) + 0.5) / draws)
    o = np.argsort(-row, kind="stable")[:k or n]
    w = np.exp(row[o].astype(np.float64) / np.float32(1.1).astype(np.float64))
    w /= w.sum()
    w = w[(np.cumsum(w) - w < p)]
    w = w[w >= mp * w[0]]
    w /= w.sum()
    counts = np.bincount(got, minlength=n)
    assert counts.sum() == counts[o[:len(w)]].sum()
    assert np.abs(counts[o[:len(w)]] - w * draws).max() <= 1.01
    assert (np.diff([int(np.flatnonzero(o == g)[0]) for g in got]) >= 0).all()        # the largest first


def test_ties_go_by_index(wv):
    """Equal logits around every cut; -0 and 0 are equal."""
    n = 3000
    x = np.zeros((6, n), np.float32)
    x[:, ::2] = -0.0
    x[3:, 1000:1500] = 2.0
    u = [0.0, 0.5, 1.0] * 2
    got, prob = run_rows(wv, torch.from_numpy(x).cuda(), [1.0] * 6, [0, 100, 2000, 10, 600, 0], [1.0, 1.0, 1.0, 1.0, 1.0, 0.1], [0.0] * 6, u)
    assert got[0] == 0 and got[1] == 49 and got[2] == 1999 and got[3] == 1000
    e2 = math.exp(2.0)
    assert got[4] == 1000 + math.ceil(0.5 * (500 + 100 / e2)) - 1
    total = 500 + 2500 / e2
    assert got[5] == 1000 + math.ceil(0.1 * total) - 1
    assert abs(prob[3] - 0.1) < 1e-6


@pytest.mark.parametrize("n", [9001, 128256, 360448, 360449])
def test_many_equal_logits(wv, n):
    """More equal candidates than are sorted together, over one and all of the cluster's parts, and a row that is walked in memory."""
    x = np.zeros((5, n), np.float32)
    x[1, 100:n - 100] = -1.0
    x[2, n - 1] = 1.0
    x[3, ::3] = 0.25
    x[4] = np.linspace(0, 1e-4, n, dtype=np.float32)
    t, k, p, mp = [1.0] * 5, [0, 0, 0, 5000, 0], [1.0, 0.9, 1.0, 0.7, 0.5], [0.0, 0.0, 0.0, 0.9, 0.0]
    u = [0.7, 0.5, 0.999, 0.9, 0.25]
    got, prob = run_rows(wv, torch.from_numpy(x).cuda(), t, k, p, mp, u)
    for r in range(5):
        want, pw, margin = sample64(x[r], t[r], k[r], p[r], mp[r], u[r])
        # equal weights: a place is u n of them, rounded up, and the sums are whole numbers; for the slope one place is 1 / n
        assert abs(got[r] - want) <= (0 if r in (0, 2) else 2), (r, got[r], want)
        assert abs(prob[r] - pw) <= 1e-6 * pw


@pytest.mark.parametrize("n", [200000, 400000])
def test_long_rows(wv, n):
    """The token is the definition's for the draw, or for one 2^-20 beside it: with so many candidates the running sums are near one
    another, and a weight's exponential in float32 is off by 2^-23."""
    rng = np.random.default_rng(n)
    x = (rng.normal(0, 1, (10, n)) * 2).astype(np.float32)
    k, p = [0, 40, 0, 30000, 1, 0, 3000, 0, 1500, n], [1.0, 0.9, 0.95, 0.9, 1.0, 0.4, 1.0, 1.0, 1.0, 0.99]
    mp, u = [0.0, 0.0, 0.0, 0.0, 0.0, 0.001, 0.0, 0.05, 0.0, 0.0], rng.random(10)
    got, prob = run_rows(wv, torch.from_numpy(x).cuda(), [0.9] * 10, k, p, mp, u)
    for r in range(10):
        want = [sample64(x[r], 0.9, k[r], p[r], mp[r], min(max(u[r] + d, 0.0), 1.0)) for d in (0.0, -2.0 ** -20, 2.0 ** -20)]
        assert got[r] in [w[0] for w in want], r
        assert abs(prob[r] - want[0][1]) <= 2.0 ** -18 * want[0][1]


def test_ends_of_the_draw(wv):
    """u = 0 takes the first candidate, u = 1 the last one that has weight."""
    rng = np.random.default_rng(0)
    x = rng.normal(0, 1, (2, 5000)).astype(np.float32)
    got, _ = run_rows(wv, torch.from_numpy(x).cuda(), [1.0, 1.0], [0, 0], [1.0, 1.0], [0.0, 0.0], [0.0, 1.0])
    assert got[0] == x[0].argmax() and got[1] == x[1].argmin()


def test_values_that_are_not_finite(wv):
    n = 2000
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (8, n)).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2, 5:] = -np.inf                       # five candidates
    x[3, ::3] = np.nan
    x[4, 700] = np.inf
    x[5, [3, 900]] = np.inf                  # two that share everything
    x[6, :] = -np.inf
    x[6, 1234] = -3e38                       # one candidate, far down
    x[7, 0] = np.nan
    t, k, p, mp = [0.7] * 8, [0, 0, 0, 50, 0, 0, 3, 1], [0.9] * 8, [0.0] * 8
    u = [0.3, 0.3, 0.99, 0.6, 0.9, 0.9, 0.5, 0.5]
    got, prob = run_rows(wv, torch.from_numpy(x).cuda(), t, k, p, mp, u)
    assert got[0] == -1 and got[1] == -1 and prob[0] == 0 and prob[1] == 0
    assert got[2] in range(5) and got[3] % 3 != 0
    assert got[4] == 700 and prob[4] == 1 and got[5] == 900 and prob[5] == 0.5
    assert got[6] == 1234 and prob[6] == 1
    assert got[7] == np.nanargmax(x[7]) and prob[7] == 1
    for r in (2, 3):
        assert got[r] == sample64(x[r], t[r], k[r], p[r], mp[r], u[r])[0]
    # a row of one candidate class, greedy: -1 where there is none
    got, prob = run_rows(wv, torch.from_numpy(x).cuda(), [0.0] * 8, k, p, mp, u)
    assert got[0] == -1 and got[1] == -1 and got[4] == 700 and got[5] == 3 and got[6] == 1234
    # parameters that are not numbers: only the first candidate, and no candidate with T
    nan = math.nan
    got, _ = run_rows(wv, torch.from_numpy(x[3:4]).cuda().repeat(3, 1), [1.0, 1.0, nan], [0, 0, 0], [nan, 1.0, 1.0], [0.0, nan, 0.0], [0.9] * 3)
    assert got[0] == got[1] == np.nanargmax(x[3]) and got[2] == -1


def test_strides_and_no_prob(wv):
    rng = np.random.default_rng(2)
    x = rng.normal(0, 1, (5, 1007)).astype(np.float32)
    d = torch.from_numpy(x).cuda()
    got, prob = run_rows(wv, d, [0.9] * 5, [0] * 5, [0.9] * 5, [0.0] * 5, [0.7] * 5, ld=(1001, 1007), prob=False)
    assert (prob == -7).all()
    for r in range(5):
        want, _, margin = sample64(x[r, :1001], 0.9, 0, 0.9, 0.0, 0.7)
        assert margin < 1e-6 or got[r] == want


def test_refusals_of_rows(wv):
    S, L = wv.sampling.SampleRowsCUDA, wv._lib
    x = torch.zeros(64, device="cuda")
    p = x.data_ptr()
    for i in (0, 3, 4, 5, 6, 7, 8):
        a = [p, 1, 8, p, p, p, p, p, p]
        a[i] = 0
        with pytest.raises(wv.WelvetError) as e:
            S(*a)
        assert e.value.code == L.WV_EARG
    for rows, n, ld in ((-1, 8, 0), (1, 0, 0), (1, 8, 7)):
        with pytest.raises(wv.WelvetError) as e:
            S(p, rows, n, p, p, p, p, p, p, ld=ld)
        assert e.value.code == L.WV_ESHAPE
    S(p, 0, 8, p, p, p, p, p, p)
