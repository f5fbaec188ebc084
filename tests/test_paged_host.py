"""CPU tests of the paged cache's host side: the size of a block of pages, the refusals that need no device, and the status of the
device entries without one."""
import ctypes as C

import pytest
import torch


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("page,hd", [(16, 16), (16, 128), (48, 64), (64, 256), (208, 80)])
def test_block_bytes(bits, page, hd):
    """Codes of K and V, two float32 scales a token, and in 4 bits two bytes for each 16 values."""
    from welvet_b200 import paged
    want = 2 * page * (hd * bits // 8) + 8 * page + (2 * page * (hd // 16) if bits == 4 else 0)
    assert paged.KVBlockBytes(bits, page, hd) == want
    assert want % 16 == 0


@pytest.mark.parametrize("bits,page,hd,name", [(5, 16, 64, "WV_EFORMAT"), (0, 16, 64, "WV_EFORMAT"), (8, 0, 64, "WV_ESHAPE"), (8, 24, 64, "WV_ESHAPE"),
                                               (8, -16, 64, "WV_ESHAPE"), (8, 16, 0, "WV_ESHAPE"), (16, 16, 72, "WV_ESHAPE"), (4, 16, 272, "WV_ESHAPE")])
def test_block_bytes_refusals(bits, page, hd, name):
    from welvet_b200 import _lib, paged
    with pytest.raises(_lib.WelvetError) as e:
        paged.KVBlockBytes(bits, page, hd)
    assert e.value.code == getattr(_lib, name)
    assert _lib.lib().wv_kv_block_bytes(8, 16, 64, None) == _lib.WV_EARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
def test_no_cpu_fallback():
    from welvet_b200 import _lib, paged
    L = _lib.lib()
    pages, batch = paged.KVPages(0, 8, 1, 16, 1, 16), paged.Batch(0, 0, 0, 1, 1, 1, 1, 1)
    p, b = C.byref(pages), C.byref(batch)
    assert L.wv_kv_write_dev(p, b, None, 0, None, 0, None, 0, None, 0, 0, 0.0, None) == _lib.WV_EINIT
    assert L.wv_kv_read_dev(p, b, None, 0, None, 0, None) == _lib.WV_EINIT
    assert L.wv_attn_paged_dev(p, b, None, 0, None, 0, 1, 1.0, 0, None) == _lib.WV_EINIT
    assert L.wv_sample_rows_dev(None, 1, 8, 0, None, None, None, None, None, None, None, None) == _lib.WV_EINIT


def test_block_decoder_checks_its_rows():
    """More new tokens than the working matrices have rows is refused before anything is launched; none is nothing to do."""
    from welvet_b200 import decode, paged
    cfg = decode.BlockConfig(DModel=64, NumHeads=4, NumKVHeads=2, HeadDim=16, IntermediateDim=128, MaxSeqLen=0)
    bufs = {n: 0 for n in ("norm", "proj", "q", "attn", "k", "v", "gate", "up", "attn_norm", "ffn_norm")}
    keys = {n: 0 for n in ("q", "k", "v", "o", "gate", "up", "down")}
    block = paged.PagedBlockDecoder(cfg, keys, bufs, paged.KVPages(0, 8, 1, 16, 2, 16), max_tokens=4)
    with pytest.raises(ValueError, match="5 new tokens"):
        block.step(0, paged.Batch(0, 0, 0, 1, 1, 5, 5, 5))
    block.step(0, paged.Batch(0, 0, 0, 1, 1, 0, 0, 0))
