"""Adapters whose targets' matrices meet: a call in which one would write what another one, or the product, reads is refused; columns beside one another
in rows of one stride are not."""
import pytest
import torch
from test_gpu_adapters import Set, mixed

pytestmark = pytest.mark.gpu
K, OUTS, ROWS = 64, [40, 24], 9


def apply(wv, s, plan, x, y, base=None, ldx=0, ldy=None, ldb=None, rows=ROWS):
    s.ad.ApplyCUDA(s.group, plan.data_ptr(), rows, x, y, base, ldx=ldx, ldy=ldy, ldb=ldb)


@pytest.mark.parametrize("name,ok,y,base,ldx,ldy,ldb", [
    # offsets in floats from one buffer, x at 0 (its rows end at 640 with ldx 72, at 1152 with 128)
    ("apart", True, (2000, 3000), None, 72, (40, 24), None),
    ("columns of one matrix", True, (2000, 2040), None, 72, (64, 64), None),
    ("columns of one matrix, the second first", True, (2024, 2000), None, 72, (64, 64), None),
    ("a column range that is wider than its place", False, (2000, 2036), None, 72, (64, 64), None),
    ("a column range that runs into the next row", False, (2000, 2044), None, 72, (64, 64), None),
    ("beside x's columns", True, (64, 104), None, 128, (128, 128), None),
    ("in x's columns", False, (60, 104), None, 128, (128, 128), None),
    ("in x's next row", False, (64, 108), None, 128, (128, 128), None),
    ("behind x's last row", True, (8 * 128 + 64, 3000), None, 128, (40, 24), None),
    ("in x's last row", False, (8 * 128 + 60, 3000), None, 128, (40, 24), None),
    ("beside x's columns, another stride", False, (64, 3000), None, 128, (132, 24), None),
    ("rows of another target's base", False, (2000, 4000), (5000, 2000 + 4 * 40), 72, (40, 24), (40, 24)),
    ("behind another target's base", True, (2000, 4000), (5000, 2000 + 9 * 40), 72, (40, 24), (40, 24)),
    ("rows of its own base", False, (2000, 4000), (2040, 5000), 72, (40, 24), (40, 24)),
    ("columns beside its own base", True, (2000, 4000), (2040, 5000), 72, (80, 24), (80, 24)),
    ("in place", True, (2000, 4000), (2000, 4000), 72, (44, 24), (44, 24)),
    ("one base for both", True, (2000, 4000), (6000, 6000), 72, (40, 24), (40, 40)),
])
def test_targets_that_meet(wv, name, ok, y, base, ldx, ldy, ldb):
    s = Set(wv, "f32", 3, 16, K, OUTS)
    slot = mixed(ROWS, 3)
    plan, _ = s.plan(slot)
    buf = torch.randn(8192, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    view = lambda at, ld, w: buf[at:at + 9 * ld + w].as_strided((ROWS, w), (ld, 1))  # noqa: E731
    x, ys = view(0, ldx, K), [view(a, d, o) for a, d, o in zip(y, ldy, OUTS)]
    bases = ys if base is None else [view(a, d, o) for a, d, o in zip(base, ldb, OUTS)]
    keep = [b.clone() for b in bases]
    before = buf.clone()
    want = s.want(x.clone(), slot, keep)
    call = lambda: apply(wv, s, plan, x.data_ptr(), [v.data_ptr() for v in ys], None if base is None else [b.data_ptr() for b in bases], ldx, list(ldy), None if ldb is None else list(ldb))  # noqa: E731
    if not ok:
        with pytest.raises(wv._lib.WelvetError) as e:
            call()
        torch.cuda.synchronize()
        assert e.value.code == wv._lib.WV_EARG and torch.equal(buf, before)
        return
    call()
    torch.cuda.synchronize()
    mask = torch.zeros_like(buf, dtype=torch.bool)
    for a, d, o, got, (w, tol) in zip(y, ldy, OUTS, ys, want):
        assert bool(((got.double() - w).abs() <= tol).all())
        mask[a:a + 9 * d + o].as_strided((ROWS, o), (d, 1)).fill_(True)
    assert torch.equal(buf[~mask], before[~mask])


def test_one_row_and_none(wv):
    """Of a single row the strides do not matter, and without rows nothing is read or written."""
    s = Set(wv, "bf16", 1, 8, K, OUTS)
    plan, _ = s.plan([0])
    buf = torch.zeros(1024, device="cuda")
    p = buf.data_ptr()
    apply(wv, s, plan, p, [p + 256, p + 416], ldx=64, ldy=[400, 800], rows=1)
    apply(wv, s, plan, p, [p, p], ldx=64, ldy=[400, 800], rows=0)
    with pytest.raises(wv._lib.WelvetError):
        apply(wv, s, plan, p, [p + 256, p + 400], ldx=64, ldy=[400, 800], rows=1)
    torch.cuda.synchronize()
