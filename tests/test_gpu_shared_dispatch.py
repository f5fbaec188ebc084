"""Which way attention over a shared prefix takes by itself: apart from the sequences' own keys where that gains, else wv_attn_paged_dev bit by bit."""
import numpy as np
import pytest
import torch
from test_gpu_paged import Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,kvh,heads,hd,bits,shared,own,apart", [
    # single and a few drafted tokens
    ([1] * 48, 8, 32, 128, 8, 4096, 50, True), ([1] * 4, 8, 32, 128, 8, 512, 50, False), ([4] * 24, 4, 32, 64, 16, 8192, 60, True),
    # pieces of prompts: rows that leave most of a tile of their own empty, and rows that fill it
    ([16] * 16, 8, 32, 128, 8, 16384, 116, True), ([16] * 4, 8, 32, 128, 8, 1024, 116, False), ([65] * 8, 8, 32, 128, 8, 16384, 165, True),
    ([64] * 16, 8, 32, 128, 8, 4096, 164, False), ([128] * 16, 8, 32, 128, 8, 1024, 228, False), ([256] * 4, 8, 32, 128, 16, 4096, 356, False),
    ([300, 160, 250, 299], 8, 32, 128, 8, 1024, 400, False), ([64] * 8, 4, 32, 64, 16, 1024, 164, False),
    # a piece of a prompt beside single tokens
    ([128] + [1] * 63, 8, 32, 128, 8, 4096, 228, True), ([1024] * 4 + [1] * 7, 8, 32, 128, 8, 1024, 1124, False),
    # wide heads: tiles of sixteen rows in either way
    ([1] * 64, 4, 16, 256, 8, 8192, 201, True), ([1] * 16, 4, 64, 192, 8, 8192, 201, False), ([4] * 16, 4, 32, 256, 8, 1024, 204, False), ([64] * 4, 4, 16, 192, 8, 4096, 264, False),
])
def test_the_faster_way(wv, hooks, tokens, kvh, heads, hd, bits, shared, own, apart):
    """Shapes whose two times lie apart by 8 % and more, measured."""
    n = shared + own
    c = Cache(wv, bits, 64, kvh, hd, [(1, n)])
    gen = torch.Generator(device="cuda").manual_seed(n)
    c.fill(*[torch.randn(n, kvh * hd, device="cuda", generator=gen) for _ in range(2)])
    ints = lambda v: torch.tensor(list(v), dtype=torch.int32, device="cuda")  # noqa: E731
    start, kv, at, m = ints(np.concatenate([[0], np.cumsum(tokens)]).tolist()), ints(n - max(tokens) + t for t in tokens), ints([0, len(tokens)]), ints([shared, 0])
    table = c.d_table.repeat(len(tokens), 1).contiguous()
    batch = wv.paged.Batch(start.data_ptr(), kv.data_ptr(), table.data_ptr(), len(tokens), table.shape[1], sum(tokens), max(tokens), n)
    groups = wv.paged.Groups(at.data_ptr(), m.data_ptr(), 1, shared)
    q = torch.randn(sum(tokens), heads * hd, device="cuda", generator=gen)

    def attend(call, *more):
        out = torch.full_like(q, 77.0)
        call(c.pages, batch, *more, q.data_ptr(), out.data_ptr(), heads, hd ** -0.5)
        torch.cuda.synchronize()
        return out
    paged, got = attend(wv.paged.AttnPagedCUDA), attend(wv.paged.AttnSharedCUDA, groups)
    hooks.wv_set_attn_sharing(1)
    try:
        forced = attend(wv.paged.AttnSharedCUDA, groups)
    finally:
        hooks.wv_set_attn_sharing(0)
    assert wv._lib.lib().wv_device_status() == 0 and not torch.equal(paged, forced)
    assert torch.equal(got, forced if apart else paged)
