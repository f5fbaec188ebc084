"""CPU tests of the host side of page tables, shared prefixes and adapters: sizes, what is refused without a device, and the status of the device
entries without one."""
import ctypes as C

import pytest
import torch


@pytest.mark.parametrize("rows,slots,tiles", [(0, 1, 0), (1, 1, 1), (8, 1, 1 + 2), (9, 1, 2), (64, 32, 8 + 33), (2048, 6, 64 + 7), (100, 8192, 12 + 100)])
def test_plan_bytes(rows, slots, tiles):
    """16 bytes of head, 16 a tile and 4 a row; tiles of 32 rows where an adapter has more than 8 on average, else of 8, and one more for each
    adapter and for none."""
    from welvet_b200 import adapters
    assert adapters.PlanBytes(rows, slots) == 16 + 16 * tiles + 4 * (-(-rows // 4) * 4)


def test_plan_bytes_refusals():
    from welvet_b200 import _lib, adapters
    for rows, slots in ((-1, 1), (1, 0), (1, 8193), (1 << 25, 1)):
        with pytest.raises(_lib.WelvetError) as e:
            adapters.PlanBytes(rows, slots)
        assert e.value.code == _lib.WV_ESHAPE
    assert _lib.lib().wv_adapter_plan_bytes(1, 1, None) == _lib.WV_EARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
def test_no_cpu_fallback():
    from welvet_b200 import _lib, adapters, paged
    L, init = _lib.lib(), _lib.WV_EINIT
    t = C.byref(paged.KVTable(0, 0, 0, 1, 16, 1, 1))
    assert L.wv_kv_fork_dev(t, None, None, None, 0, None) == init
    assert L.wv_kv_extend_dev(t, None, None, None, 0, None) == init
    assert L.wv_kv_trim_dev(t, None, None, 0, None) == init
    assert L.wv_kv_compact_dev(t, None, 0, None, None) == init
    assert L.wv_kv_copy_dev(None, 0, None, None, 0, None) == init
    p, b, g = paged.KVPages(0, 8, 1, 16, 1, 16), paged.Batch(0, 0, 0, 1, 1, 1, 1, 1), paged.Groups(0, 0, 0, 0)
    assert L.wv_attn_shared_dev(C.byref(p), C.byref(b), C.byref(g), None, 0, None, 0, 1, 1.0, None) == init
    assert L.wv_adapter_plan_dev(None, 1, 1, None, None) == init
    a = adapters.Group([adapters.Adapters(0, 0, 0, 0, 1, 8, 8, 1, 1)])
    assert L.wv_adapter_apply_dev(a, 1, None, 1, None, 0, None, None, None, None, None) == init


def test_block_decoder_checks():
    """A window beside a shared prefix, or a plan for a block without adapters, is refused before anything is launched."""
    from welvet_b200 import decode, paged
    cfg = decode.BlockConfig(DModel=64, NumHeads=4, NumKVHeads=2, HeadDim=16, IntermediateDim=128, MaxSeqLen=0)
    bufs = {n: 0 for n in ("norm", "proj", "q", "attn", "k", "v", "gate", "up", "attn_norm", "ffn_norm")}
    keys = {n: 0 for n in ("q", "k", "v", "o", "gate", "up", "down")}
    batch = paged.Batch(0, 0, 0, 1, 1, 1, 1, 1)
    with pytest.raises(ValueError, match="window"):
        paged.PagedBlockDecoder(cfg, keys, bufs, paged.KVPages(0, 8, 1, 16, 2, 16), 4, window=8).step(0, batch, groups=paged.Groups(0, 0, 0, 0))
    with pytest.raises(ValueError, match="adapters"):
        paged.PagedBlockDecoder(cfg, keys, bufs, paged.KVPages(0, 8, 1, 16, 2, 16), 4).step(0, batch, plan=1)
