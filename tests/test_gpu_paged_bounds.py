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


SCRATCH = 256 << 20                               # what a call of the attention may keep for the results of its splits


def taken(call):
    """Device memory that a captured call and its replay leave taken (the graph is still there)."""
    call(torch.cuda.current_stream().cuda_stream)                        # kernels loaded, the stream's own scratch allocated
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(g, stream=st):
        call(torch.cuda.current_stream().cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    return free - torch.cuda.mem_get_info()[0], g


def close(got, want):
    """As in a full batch's long sequences: 40 additions that cut off up to 2^-23 of a sum, half of that on average, and as much again."""
    assert ((got.double() - want).norm() / want.norm()).item() <= 2 * 40 * 2.0 ** -24


def test_scratch_of_a_long_prompt_with_wide_heads(wv):
    """Heads beyond 128 go 16 rows at a time, and their keys in splits: a prompt of 8192 tokens (131072 rows, 7 splits of 258 numbers)
    takes its scratch in parts. Tokens from its start, middle and end against 64 bits."""
    n, heads, kvh, hd = 8192, 16, 8, 256
    c = Cache(wv, 8, 64, kvh, hd, [(n, n)])
    gen = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    k, v, q = rand(n, kvh * hd), rand(n, kvh * hd), rand(n, heads * hd)
    c.fill(k, v)
    wv.paged.KVReadCUDA(c.pages, c.batch, k.data_ptr(), v.data_ptr())
    out = torch.zeros(n, heads * hd, device="cuda")
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    took, g = taken(lambda st: wv.paged.AttnPagedCUDA(c.pages, c.batch, q.data_ptr(), out.data_ptr(), heads, 0.0625, stream=st))
    assert took <= SCRATCH + (4 << 20), took
    kd, vd = (t.view(n, kvh, hd).double() for t in (k, v))
    for t0 in (0, 1279, 4090, 8176):
        qs = q[t0:t0 + 16].view(16, kvh, heads // kvh, hd).double()
        s = torch.einsum("tgrd,kgd->tgrk", qs, kd[:t0 + 16]) * 0.0625
        s = s.masked_fill(torch.arange(t0 + 16, device="cuda") > t0 + torch.arange(16, device="cuda")[:, None, None, None], float("-inf"))
        close(out[t0:t0 + 16], torch.einsum("tgrk,kgd->tgrd", torch.softmax(s, -1), vd[:t0 + 16]).reshape(16, -1))


@pytest.mark.parametrize("piece", [1, 64])
def test_scratch_of_many_sequences_under_a_long_bound(wv, piece):
    """256 short sequences, a piece of a prompt among them or not, under the bound of a model with a context of 131072."""
    seqs, heads, kvh, hd, most, page = 256, 32, 8, 128, 131072, 64
    c = Cache(wv, 8, page, kvh, hd, [(1, 400)])
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    k, v = rand(400, kvh * hd), rand(400, kvh * hd)
    c.fill(k, v)
    whole, keep = c.batch_of([(400, 400)])
    wv.paged.KVReadCUDA(c.pages, whole, k.data_ptr(), v.data_ptr())
    table = torch.full((seqs, most // page), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.d_table                               # one sequence's pages for all of them
    new = [1] * seqs
    new[100] = piece
    new[7] = 0
    start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
    kv = torch.randint(64, 401, (seqs,), device="cuda", dtype=torch.int32, generator=gen)
    total = sum(new)
    q, out = rand(total, heads * hd), torch.zeros(total, heads * hd, device="cuda")
    b = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), table.data_ptr(), seqs, table.shape[1], total, piece, most)
    took, g = taken(lambda st: wv.paged.AttnPagedCUDA(c.pages, b, q.data_ptr(), out.data_ptr(), heads, 0.09, stream=st))
    assert took <= SCRATCH + (4 << 20), took
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), torch.tensor(new, device="cuda"))
    pos = kv[seq] - (start[seq + 1] - torch.arange(total, device="cuda"))
    s = torch.einsum("tgrd,kgd->tgrk", q.view(total, kvh, heads // kvh, hd).double(), k.view(400, kvh, hd).double()) * 0.09
    s = s.masked_fill(torch.arange(400, device="cuda") > pos[:, None, None, None], float("-inf"))
    close(out, torch.einsum("tgrk,kgd->tgrd", torch.softmax(s, -1), v.view(400, kvh, hd).double()).reshape(total, -1))
    assert wv._lib.lib().wv_device_status() == 0


@pytest.mark.parametrize("heads,kvh,hd,max_q,most", [(8, 2, 256, 2048, 400), (4, 4, 144, 300, 5000), (16, 1, 192, 131072, 131072)])
def test_wide_heads_under_loose_bounds(wv, heads, kvh, hd, max_q, most):
    """Heads beyond 128: single tokens, a piece of a prompt and empty sequences in a batch whose bounds allow each far more (256 sequences
    of 131072 tokens have more tiles of rows than a grid)."""
    lens = ([(1, 60), (40, 90), (0, 0), (3, 3), (1, 300), (70, 70), (1, 1), (9, 200)] + [(1, 17), (0, 5)] * 16) if max_q < 131072 else [(1, 60), (33, 90)] + [(0, 0)] * 254
    c = Cache(wv, 8, 16, kvh, hd, lens, seed=hd)
    rng = np.random.default_rng(hd)
    n, total = sum(k for _, k in lens), sum(q for q, _ in lens)
    c.fill(*(torch.from_numpy(rng.normal(0, 1, (n, kvh * hd)).astype(np.float32)).cuda() for _ in range(2)))
    q = rng.normal(0, 1, (total, heads * hd)).astype(np.float32)
    dq, out = torch.from_numpy(q).cuda(), torch.full((total + 5, heads * hd), 7.0, device="cuda")
    table = torch.full((len(lens), -(-most // 16)), -1, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.d_table
    start, kv = arrays(c, lens)
    b = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), table.data_ptr(), len(lens), table.shape[1], total + 5, max_q, most)
    scale = hd ** -0.5
    wv.paged.AttnPagedCUDA(c.pages, b, dq.data_ptr(), out.data_ptr(), heads, scale)
    torch.cuda.synchronize()
    assert wv._lib.lib().wv_device_status() == 0
    got = out.cpu().numpy()
    assert (got[total:] == 7.0).all()
    want, tol = want_attn(c, lens, q, heads, scale)
    assert (np.abs(got[:total].reshape(total, heads, hd) - want) <= tol).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -3e38])
def test_queries_before_position_0(wv, hd, what):
    """What the rows of tokens that see nothing hold does not matter: they are zeros, and the others do not notice."""
    lens = [(9, 5), (1, 0), (3, 1), (90, 60), (40, 0)]
    c = Cache(wv, 8, 16, 2, hd, lens)
    rng = np.random.default_rng(hd)
    n, total = sum(k for _, k in lens), sum(q for q, _ in lens)
    c.fill(*(torch.from_numpy(rng.normal(0, 1, (n, 2 * hd)).astype(np.float32)).cuda() for _ in range(2)))
    q = rng.normal(0, 1, (total, 4 * hd)).astype(np.float32)
    want, tol = want_attn(c, lens, q, 4, hd ** -0.5)
    r = 0
    for nq, kv in lens:
        q[r:r + max(0, nq - kv)] = what
        r += nq
    out = torch.full((total, 4 * hd), 7.0, device="cuda")
    wv.paged.AttnPagedCUDA(c.pages, c.batch, torch.from_numpy(q).cuda().data_ptr(), out.data_ptr(), 4, hd ** -0.5)
    torch.cuda.synchronize()
    assert (np.abs(out.cpu().numpy().reshape(total, 4, hd) - want) <= tol).all()


@pytest.mark.parametrize("hd", [64, 256])
@pytest.mark.parametrize("what", ["kv_len", "q_start"])
@pytest.mark.parametrize("total", [96 * 42, 96 * 42 + 200, 130])
def test_lengths_out_of_bounds_behind_the_first_sequence(wv, hd, what, total):
    """A length out of its bounds is reported wherever it stands, with tokens of its own or none, whichever kernels run."""
    lens = [(96, 100)] + [(0, 50)] * 40 + [(30, 50)]
    c = Cache(wv, 8, 16, 2, hd, lens)
    c.fill(torch.randn(2150, 2 * hd, device="cuda"), torch.randn(2150, 2 * hd, device="cuda"))
    q, out = torch.randn(total, 8 * hd, device="cuda"), torch.zeros(total, 8 * hd, device="cuda")
    start, kv = arrays(c, lens)
    status = wv._lib.lib().wv_device_status
    b = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), c.d_table.data_ptr(), 42, c.table.shape[1], total, 96, 100)

    def call():
        wv.paged.AttnPagedCUDA(c.pages, b, q.data_ptr(), out.data_ptr(), 8, 0.1)
        torch.cuda.synchronize()
        return status()
    assert call() == 0
    for i, bad in ((35, 101), (35, -1), (41, 10 ** 9)) if what == "kv_len" else ((36, 90), (42, 96 + 97), (42, total + 1)):
        a = kv if what == "kv_len" else start
        saved = int(a[i])
        a[i] = bad
        assert call() == wv._lib.WV_ESHAPE, (i, bad)
        a[i] = saved
    assert call() == 0


def test_no_more_positions_than_the_attention_counts(wv):
    """A billion cached tokens and more under one table row are refused: keys are counted in 32 bits."""
    c = Cache(wv, 8, 16, 2, 64, [(1, 20)])
    x, o = torch.zeros(1, 256, device="cuda"), torch.zeros(1, 256, device="cuda")
    start, kv = arrays(c, [(1, 20)])
    for most, ok in ((2 ** 30, True), (2 ** 30 + 1, False), (2 ** 31 - 16, False)):
        b = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), c.d_table.data_ptr(), 1, 2 ** 27, 1, 1, most)
        if ok:
            wv.paged.AttnPagedCUDA(c.pages, b, x.data_ptr(), o.data_ptr(), 4, 0.125)
        else:
            with pytest.raises(wv.WelvetError) as e:
                wv.paged.AttnPagedCUDA(c.pages, b, x.data_ptr(), o.data_ptr(), 4, 0.125)
            assert e.value.code == wv._lib.WV_ESHAPE
    torch.cuda.synchronize()
    assert wv._lib.lib().wv_device_status() == 0
