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
