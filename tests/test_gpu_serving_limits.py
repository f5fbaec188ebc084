"""Page tables of more pages, sequences or places in a row, and adapters of more columns or outputs, than the kernels' 32-bit numbers reach are refused before
anything is launched."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("over", ["num_pages", "num_seqs", "table_stride"])
@pytest.mark.parametrize("by", [1, 2 ** 30 - 1])
def test_tables_beyond_their_limits(wv, over, by):
    E, L = wv._lib, wv._lib.lib()
    buf = torch.zeros(64, dtype=torch.int32, device="cuda")
    p = buf.data_ptr()
    t = wv.paged.KVTable(p, p + 64, p + 128, 4, 16, 2, 2)
    setattr(t, over, 2 ** 30 + by)
    t = C.byref(t)
    for rc in (L.wv_kv_fork_dev(t, p, p + 4, None, 0, None), L.wv_kv_extend_dev(t, p, None, None, 0, None), L.wv_kv_trim_dev(t, None, None, 0, None), L.wv_kv_compact_dev(t, None, 0, p, None)):
        assert rc == E.WV_ESHAPE and str(2 ** 30).encode() in L.wv_last_error()
    torch.cuda.synchronize()
    assert not buf.any() and L.wv_device_status() == 0


@pytest.mark.parametrize("wide", [dict(in_=2 ** 30 + 8), dict(in_=2 ** 31 - 8), dict(out=2 ** 30 + 4), dict(out=2 ** 31 - 1)])
@pytest.mark.parametrize("rows", [0, 1])
def test_adapters_beyond_their_limits(wv, wide, rows):
    """Columns or outputs whose offsets would not fit 32 bits."""
    E, L, ad = wv._lib, wv._lib.lib(), wv.adapters
    buf = torch.zeros(256, device="cuda")
    p = buf.data_ptr()
    g = ad.Group([ad.Adapters(**{**dict(a=p, b=p, rank=0, scale=0, slots=1, max_rank=8, in_=8, out=8, dtype=1), **wide})])
    assert L.wv_adapter_apply_dev(g, 1, p, rows, p, 0, None, None, (C.c_void_p * 1)(p + 512), None, None) == E.WV_ESHAPE
    assert str(2 ** 30).encode() in L.wv_last_error()
    torch.cuda.synchronize()
    assert not buf.any()
