"""Attention over a shared prefix where far less is shared than the bounds say, or the scratch allows few splits: the splits are long, but no chain of
products into one sum is. A query of zeros weighs all keys alike, exactly, and values of one sign make every cut of a sum count the same way, so that what is
left of the error is the sums'."""
import numpy as np
import pytest
import torch
from test_gpu_paged import Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def always(hooks):
    hooks.wv_set_attn_sharing(1)
    yield
    hooks.wv_set_attn_sharing(0)


def values(bits, kvh, hd, n):
    """n tokens' values in (0.5, 1)."""
    return np.random.default_rng(bits + hd).uniform(0.5, 1.0, (n, kvh * hd)).astype(np.float32)


def tolerance(rows, keys):
    """Of a sum of positive terms over the longest split's keys, relative: 40 products one after the other, each cut by 2^-23 at most; after them the four warps,
    the stretches of the split (2560 keys for up to 8 rows, 1280 for 16) and no more than 8 splits are added in float32, two roundings of 2^-24 each; the
    division, its reciprocal and the weights' two pieces are four more."""
    return 2.0 ** -23 * (40 + 4 + -(-keys // (2560 if rows == 8 else 1280)) + 8 + 4)


def call(wv, c, table, lens, start, shared, most_shared, most_kv, heads, max_q):
    ints = lambda v: torch.tensor(list(v), dtype=torch.int32, device="cuda")  # noqa: E731
    n = sum(q for q, _ in lens)
    at, kv, s, m = ints(np.concatenate([[0], np.cumsum([q for q, _ in lens])]).tolist()), ints(k for _, k in lens), ints(start), ints(list(shared) + [0])
    batch = wv.paged.Batch(at.data_ptr(), kv.data_ptr(), table.data_ptr(), len(lens), table.shape[1], n, max_q, most_kv)
    groups = wv.paged.Groups(s.data_ptr(), m.data_ptr(), len(shared), most_shared)
    q = torch.zeros(n, heads * c.hd, device="cuda")
    out = torch.full_like(q, 77.0)
    wv.paged.AttnSharedCUDA(c.pages, batch, groups, q.data_ptr(), out.data_ptr(), heads, 0.125)
    torch.cuda.synchronize()
    assert wv._lib.lib().wv_device_status() == 0
    return out.reshape(len(lens), max_q, heads, c.hd).double()


def means(c, n, tokens):
    """The mean of the values that each of the last `tokens` of n tokens sees, of one kv head: [tokens, 1, hd]."""
    rows = c.rows("v")[:, 0]
    total = rows.sum(0)
    return torch.from_numpy(np.stack([(total - rows[n - tokens + i + 1:].sum(0)) / (n - tokens + i + 1) for i in range(tokens)])[:, None]).cuda()


@pytest.mark.parametrize("bits,hd,heads,tokens", [(8, 64, 8, 1), (8, 64, 8, 2), (16, 128, 8, 1), (4, 128, 16, 1), (4, 48, 8, 1), (8, 80, 4, 4), (16, 256, 4, 1), (8, 192, 8, 2)])
@pytest.mark.parametrize("n,start,shared", [(131072, [0, 1], [0]), (131072, [1, 2], [64]), (65000, [0, 2], [64])])
def test_far_less_shared_than_planned(wv, bits, hd, heads, tokens, n, start, shared):
    """Two sequences of the same n tokens under bounds by which nearly all of them could be shared: nothing is (a group of one whose prefix is
    empty; a sequence of no group), or one page is."""
    c = Cache(wv, bits, 64, 1, hd, [(tokens, n)])
    c.fill(torch.ones(n, hd, device="cuda"), torch.from_numpy(values(bits, 1, hd, n)).cuda())
    got = call(wv, c, c.d_table.repeat(2, 1).contiguous(), [(tokens, n)] * 2, start, shared, n - 100, n, heads, tokens)
    err = float((got / means(c, n, tokens) - 1).abs().max()) / tolerance(8 if tokens * heads <= 8 else 16, n)
    assert err <= 1, err


@pytest.mark.parametrize("heads,tokens", [(8, 1), (8, 2)])
def test_splits_cut_short_by_the_scratch(wv, heads, tokens):
    """So many rows that a call's scratch has room for three results of each: two splits of the prefix, one of a sequence's own keys. Groups of one, so that
    the prefix too goes to the kernel for few rows."""
    hd, seqs, n, shared = 64, 32768 // tokens, 131072, 65536
    c = Cache(wv, 8, 64, 1, hd, [(1, n)])
    c.fill(torch.ones(n, hd, device="cuda"), torch.from_numpy(values(8, 1, hd, n)).cuda())
    got = call(wv, c, c.d_table.repeat(seqs, 1).contiguous(), [(tokens, n)] * seqs, range(seqs + 1), [shared] * seqs, shared, n, heads, tokens)
    err = float((got / means(c, n, tokens) - 1).abs().max()) / tolerance(8 if tokens * heads <= 8 else 16, 65536)
    assert err <= 1, err
