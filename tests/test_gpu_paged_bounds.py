"""A step's contents under bounds that are looser than they are, as a captured graph has them: fewer and shorter sequences than total_q,
max_q and max_kv allow, in calls of one kernel and of both."""
import numpy as np
import pytest
import torch

from test_gpu_paged import Cache, attn64, bound

pytestmark = pytest.mark.gpu


def arrays(c, lens):
    """q_start and kv_len of the step, to be refilled between replays."""
    start = np.concatenate([[0], np.cumsum([q for q, _ in lens])]).astype(np.int32)
    return torch.from_numpy(start).cuda(), torch.tensor([k for _, k in lens], dtype=torch.int32, device="cuda")


def want_attn(c, lens, q, heads, scale):
    """Outputs and tolerances of all rows, by sequence; `c` holds each sequence's longest cache."""
    total, hd = q.shape[0], c.hd
    out, tol = np.full((total, heads, hd), 7.0), np.zeros((total, heads, hd))
    kk, vv = c.rows("k"), c.rows("v")
    a = r = 0
    for (nq, kv), (_, full) in zip(lens, c.lens):
        want, mag, reach = attn64(q[r:r + nq].reshape(nq, heads, hd), kk[a:a + kv], vv[a:a + kv], scale, 0, kv - nq)
        out[r:r + nq], tol[r:r + nq] = want, bound(mag, reach, hd, kv)
        r, a = r + nq, a + full
    return out, tol


@pytest.mark.parametrize("bits,hd", [(16, 64), (8, 128), (4, 80), (8, 256)])
@pytest.mark.parametrize("full,contents", [
    ([(96, 200)], [[(1, 150)], [(8, 200)], [(9, 9)], [(0, 77)], [(0, 0)], [(95, 95)], [(96, 200)]]),
    ([(96, 200), (96, 96)], [[(96, 200), (1, 60)], [(1, 30), (1, 96)], [(0, 10), (8, 80)], [(8, 8), (96, 96)], [(0, 0), (0, 0)], [(96, 200), (96, 96)]])])
def test_a_captured_chunk_with_other_lengths(wv, bits, hd, full, contents):
    """num_seqs * max_q == total_q, and a replay's sequences have fewer tokens, one or none: every row that a sequence owns is
    written, with what a direct call gives, and no other."""
    heads, kvh, scale = 8, 2, hd ** -0.5
    c = Cache(wv, bits, 16, kvh, hd, full, seed=hd)
    rng = np.random.default_rng(hd)
    n, total = sum(k for _, k in full), sum(q for q, _ in full)
    c.fill(*(torch.from_numpy(rng.normal(0, 1, (n, kvh * hd)).astype(np.float32)).cuda() for _ in range(2)))
    q = rng.normal(0, 1, (total, heads * hd)).astype(np.float32)
    dq, out, out2 = torch.from_numpy(q).cuda(), torch.zeros(total, heads * hd, device="cuda"), torch.zeros(total, heads * hd, device="cuda")
    start, kv = arrays(c, full)
    batch = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), c.d_table.data_ptr(), len(full), c.table.shape[1], total, 96, 200)

    def call(o):
        wv.paged.AttnPagedCUDA(c.pages, batch, dq.data_ptr(), o.data_ptr(), heads, scale, stream=torch.cuda.current_stream().cuda_stream)
    call(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out)
    for lens in contents:
        for a, b in zip((start, kv), arrays(c, lens)):
            a.copy_(b)
        out.fill_(7.0)
        out2.fill_(7.0)
        g.replay()
        call(out2)
        torch.cuda.synchronize()
        got = out.cpu().numpy().reshape(total, heads, hd)
        want, tol = want_attn(c, lens, q, heads, scale)
        assert (np.abs(got - want) <= tol).all(), (lens, float(np.abs(got - want).max()))
        assert torch.equal(out, out2)
        assert wv._lib.lib().wv_device_status() == 0


def test_few_and_many_tokens_under_loose_bounds(wv):
    """Decode rows beside a piece of a prompt, captured once; the piece wanders from sequence to sequence, and ends."""
    bits, heads, kvh, hd = 8, 8, 2, 64
    full = [(64, 150), (64, 120), (64, 300), (64, 64)]
    c = Cache(wv, bits, 16, kvh, hd, full, seed=2)
    rng = np.random.default_rng(2)
    n, total = sum(k for _, k in full), 80
    c.fill(*(torch.from_numpy(rng.normal(0, 1, (n, kvh * hd)).astype(np.float32)).cuda() for _ in range(2)))
    q = rng.normal(0, 1, (total, heads * hd)).astype(np.float32)
    dq, out = torch.from_numpy(q).cuda(), torch.zeros(total, heads * hd, device="cuda")
    start, kv = arrays(c, [(0, 0)] * 4)
    batch = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), c.d_table.data_ptr(), 4, c.table.shape[1], total, 64, 300)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        wv.paged.AttnPagedCUDA(c.pages, batch, dq.data_ptr(), out.data_ptr(), heads, 0.125, stream=torch.cuda.current_stream().cuda_stream)
    for lens in ([(64, 64), (1, 100), (1, 300), (0, 0)], [(1, 65), (63, 63), (1, 30), (9, 9)], [(1, 1), (1, 2), (0, 3), (1, 64)], [(0, 0), (0, 0), (64, 300), (8, 8)]):
        for a, b in zip((start, kv), arrays(c, lens)):
            a.copy_(b)
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        want, tol = want_attn(c, lens, q, heads, 0.125)
        assert (np.abs(out.cpu().numpy().reshape(total, heads, hd) - want) <= tol).all(), lens
        assert wv._lib.lib().wv_device_status() == 0


@pytest.mark.parametrize("max_q,long", [(4, 7), (4, 60), (64, 67), (64, 150)])
def test_more_tokens_than_max_q(wv, max_q, long):
    """A sequence in the midst of others with more new tokens than max_q: reported, its first max_q ones are taken at the places that
    they have, the others' rows and places are left as they were, and the other sequences do not notice; in all three calls."""
    heads, kvh, hd, scale = 8, 2, 64, 0.125
    lens = [(3, 90), (long, 200), (max_q, 100)]
    c = Cache(wv, 8, 16, kvh, hd, lens, seed=long)
    rng = np.random.default_rng(long)
    n, total = sum(k for _, k in lens), sum(q for q, _ in lens)
    rand = lambda *s: torch.from_numpy(rng.normal(0, 1, s).astype(np.float32)).cuda()  # noqa: E731
    c.fill(rand(n, kvh * hd), rand(n, kvh * hd))
    status = wv._lib.lib().wv_device_status
    batch, keep = c.batch_of(lens, max_q=max_q)
    whole = c.keep, c.batch
    mine = np.ones(total, bool)
    mine[3 + max_q:3 + long] = False                                      # the rows that nobody takes
    q = rng.normal(0, 1, (total, heads * hd)).astype(np.float32)
    out = torch.full((total, heads * hd), 7.0, device="cuda")
    wv.paged.AttnPagedCUDA(c.pages, batch, torch.from_numpy(q).cuda().data_ptr(), out.data_ptr(), heads, scale)
    torch.cuda.synchronize()
    assert status() == wv._lib.WV_ESHAPE
    got = out.cpu().numpy().reshape(total, heads, hd)
    want, tol = want_attn(c, lens, q, heads, scale)
    assert (np.abs(got - want) <= tol)[mine].all() and (got[~mine] == 7.0).all()
    # what the cache holds, read back
    full = [torch.full((total, kvh * hd), 5.0, device="cuda") for _ in range(2)]
    part = [torch.full((total, kvh * hd), 5.0, device="cuda") for _ in range(2)]
    wv.paged.KVReadCUDA(c.pages, whole[1], *[t.data_ptr() for t in full])
    torch.cuda.synchronize()
    assert status() == 0
    wv.paged.KVReadCUDA(c.pages, batch, *[t.data_ptr() for t in part])
    torch.cuda.synchronize()
    assert status() == wv._lib.WV_ESHAPE
    m = torch.from_numpy(mine).cuda()
    for f, p in zip(full, part):
        assert torch.equal(p[m], f[m]) and (p[~m] == 5.0).all()
    # written anew, with the queries turned
    k, v, before = rand(total, kvh * hd), rand(total, kvh * hd), c.pool.clone()
    dq, qo = rand(total, heads * hd), torch.full((total, heads * hd), 5.0, device="cuda")
    qf = torch.zeros_like(qo)
    wv.paged.KVWriteCUDA(c.pages, batch, k.data_ptr(), v.data_ptr(), dq.data_ptr(), qo.data_ptr(), heads, 10000.0)
    torch.cuda.synchronize()
    assert status() == wv._lib.WV_ESHAPE
    some = [torch.zeros_like(t) for t in full]
    wv.paged.KVReadCUDA(c.pages, whole[1], *[t.data_ptr() for t in some])
    c.pool.copy_(before)
    wv.paged.KVWriteCUDA(c.pages, whole[1], k.data_ptr(), v.data_ptr(), dq.data_ptr(), qf.data_ptr(), heads, 10000.0)
    every = [torch.zeros_like(t) for t in full]
    wv.paged.KVReadCUDA(c.pages, whole[1], *[t.data_ptr() for t in every])
    torch.cuda.synchronize()
    assert status() == 0
    assert torch.equal(qo[m], qf[m]) and (qo[~m] == 5.0).all()
    for f, s, e in zip(full, some, every):
        assert torch.equal(s[m], e[m]) and torch.equal(s[~m], f[~m])
