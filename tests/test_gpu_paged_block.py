"""A small stack served in batches: paged.PagedBlockDecoder with prompts of different lengths in one step, then single tokens, then the
next tokens by sampling.SampleRowsCUDA, against decode.BlockDecoder walking the same tokens one by one over a float32 cache."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

D, HEADS, KVH, HD, FFN, VOCAB, LAYERS = 256, 8, 2, 64, 512, 1000, 2


@pytest.fixture(scope="module")
def model(wv):
    from welvet_b200.decode import BlockConfig, projection_shapes
    rng = np.random.default_rng(11)
    cfg = BlockConfig(D, HEADS, KVH, HD, FFN, 256)

    keep = []                                     # a Blob that goes takes its device copy with it

    def resident(r, c):
        keep.append(wv.quant.Pack(wv.quant.Format.FormatQ8_0, rng.normal(0, 0.06, r * c).astype(np.float32), r, c))
        return wv.quant.EnsureResident(keep[-1])
    blocks = [{n: resident(r, c) for n, (r, c) in projection_shapes(cfg).items()} for _ in range(LAYERS)]
    norms = [[torch.from_numpy(rng.normal(1, 0.05, D).astype(np.float32)).cuda() for _ in range(2)] for _ in range(LAYERS)]
    yield cfg, blocks, norms, resident(VOCAB, D)


def one_by_one(wv, model, tokens):
    """The hidden state of every token of a sequence [n, D] after the stack, through the single-token decoder."""
    from welvet_b200.decode import BlockDecoder
    cfg, blocks, norms, _ = model
    z = lambda *n: torch.zeros(*n, device="cuda")  # noqa: E731
    work = {"q": z(HEADS * HD), "k": z(KVH * HD), "v": z(KVH * HD), "attn": z(HEADS * HD), "ffn": z(FFN)}
    caches, decs = [], []
    for keys, (g1, g2) in zip(blocks, norms):
        ck, cv = z(cfg.MaxSeqLen, KVH * HD), z(cfg.MaxSeqLen, KVH * HD)
        caches += [ck, cv]
        decs.append(BlockDecoder(cfg, keys, {**{n: t.data_ptr() for n, t in work.items()}, "attn_norm": g1.data_ptr(), "ffn_norm": g2.data_ptr(),
                                            "cache_k": ck.data_ptr(), "cache_v": cv.data_ptr()}))
    out = []
    for pos, x in enumerate(tokens):
        h = x.clone()
        for d in decs:
            d.step(h.data_ptr(), pos)
        torch.cuda.synchronize()
        out.append(h)
    return torch.stack(out)


@pytest.mark.parametrize("bits,tol", [(16, 0.01), (8, 0.04)])
def test_prompts_and_steps_as_one_by_one(wv, model, bits, tol):
    """Tolerance: a projection's rows are TF32 products (2^-10 of sum |w x|, some 1e-3 of the result), four of them a block, two
    blocks; an 8-bit cache adds half a step, 1 / 254 of a row's largest value, to K and to V."""
    from welvet_b200 import paged, sampling
    cfg, blocks, norms, head = model
    lens, steps, page = [37, 90, 5], 3, 16
    rng = np.random.default_rng(bits)
    seqs = [torch.from_numpy(rng.normal(0, 1, (n + steps, D)).astype(np.float32)).cuda() for n in lens]
    want = [one_by_one(wv, model, s) for s in seqs]
    total = sum(lens)
    z = lambda *n: torch.zeros(*n, device="cuda")  # noqa: E731
    work = {"norm": z(total, D), "proj": z(total, D), "q": z(total, HEADS * HD), "attn": z(total, HEADS * HD), "k": z(total, KVH * HD), "v": z(total, KVH * HD),
            "gate": z(total, FFN), "up": z(total, FFN)}
    per = -(-(max(lens) + steps) // page)
    table = torch.from_numpy(rng.permutation(len(lens) * per).astype(np.int32)).cuda().reshape(len(lens), per)
    pools, decs = [], []
    for keys, (g1, g2) in zip(blocks, norms):
        pool = torch.zeros(len(lens) * per * KVH * paged.KVBlockBytes(bits, page, HD), dtype=torch.uint8, device="cuda")
        pools.append(pool)
        pages = paged.KVPages(pool.data_ptr(), bits, len(lens) * per, page, KVH, HD)
        bufs = {**{n: t.data_ptr() for n, t in work.items()}, "attn_norm": g1.data_ptr(), "ffn_norm": g2.data_ptr()}
        decs.append(paged.PagedBlockDecoder(cfg, keys, bufs, pages, total))

    def step(h, new, kv):
        start = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device="cuda")
        kv = torch.tensor(kv, dtype=torch.int32, device="cuda")
        batch = paged.Batch(start.data_ptr(), kv.data_ptr(), table.data_ptr(), len(lens), per, sum(new), max(new), int(kv.max()))
        for d in decs:
            d.step(h.data_ptr(), batch)
        torch.cuda.synchronize()
        assert wv._lib.lib().wv_device_status() == 0

    h = torch.cat([s[:n] for s, n in zip(seqs, lens)])
    step(h, lens, lens)
    ref = torch.cat([w[:n] for w, n in zip(want, lens)])
    assert float((h - ref).abs().max()) <= tol * float(ref.abs().max())
    for i in range(steps):                        # single tokens of all sequences
        h = torch.stack([s[n + i] for s, n in zip(seqs, lens)]).contiguous()
        step(h, [1] * len(lens), [n + i + 1 for n in lens])
        ref = torch.stack([w[n + i] for w, n in zip(want, lens)])
        assert float((h - ref).abs().max()) <= tol * float(ref.abs().max())
    # the head and the next tokens: greedy for the first, drawn for the others
    logits = z(len(lens), VOCAB)
    wv._lib.check(wv._lib.lib().wv_matvec_dev(head, h.data_ptr(), logits.data_ptr(), len(lens), D, VOCAB, None))
    dev = lambda v, t: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    par = [dev([0.0, 0.8, 1.0], torch.float32), dev([0, 40, 0], torch.int32), dev([1.0, 0.9, 0.5], torch.float32), dev([0.0, 0.0, 0.1], torch.float32),
           dev([0.5, 0.3, 0.99], torch.float64)]
    index, prob = dev([-7] * 3, torch.int32), z(3)
    sampling.SampleRowsCUDA(logits.data_ptr(), 3, VOCAB, *[t.data_ptr() for t in par], index.data_ptr(), prob.data_ptr())
    torch.cuda.synchronize()
    assert int(index[0]) == int(logits[0].argmax()) == sampling.ArgMaxCUDA(logits[0].data_ptr(), VOCAB)
    p = torch.softmax(logits[1].double() / 0.8, 0)
    assert int(index[1]) in torch.topk(p, 40).indices.tolist() and 0 < float(prob[1]) <= 1
    assert float(torch.softmax(logits[2].double(), 0)[int(index[2])]) >= 0.1 * float(torch.softmax(logits[2].double(), 0).max())


def test_too_many_tokens_are_refused(wv, model):
    from welvet_b200 import paged
    cfg, blocks, norms, _ = model
    bufs = {n: 0 for n in ("norm", "proj", "q", "attn", "k", "v", "gate", "up", "attn_norm", "ffn_norm")}
    d = paged.PagedBlockDecoder(cfg, blocks[0], bufs, paged.KVPages(0, 8, 1, 16, KVH, HD), 4)
    with pytest.raises(ValueError):
        d.step(0, paged.Batch(0, 0, 0, 1, 1, 5, 5, 5))
    d.step(0, paged.Batch(0, 0, 0, 1, 1, 0, 0, 0))          # no tokens: nothing to do
