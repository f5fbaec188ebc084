"""Rows whose values lie far apart, the largest of them beside weights of zero: what is left of the small ones. float32 and bfloat16 weights keep
24 bits of each value, float16 ones up to 2^-32 of the largest of its row."""
import pytest
import torch
from test_gpu_adapters import Set, mixed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,slots,rank", [(1, 1, 16), (7, 3, 40), (90, 3, 16), (90, 3, 72), (5, 2, 136)])
@pytest.mark.parametrize("far", [4, 12, 20])
def test_values_far_below_the_largest(wv, dtype, rows, slots, rank, far):
    """Every 16 columns of x hold one that is 2^far larger, with zeros of A beside it, and every eighth of A's rows is 2^(far / 2) larger, with zeros of B. With float16
    weights x and t enter with three pieces behind a power of two of the row: off by 2^-32 of its largest value at most, on the magnitudes of A and B."""
    k, outs = 528, [200]
    s = Set(wv, dtype, slots, rank, k, outs)
    gen = torch.Generator(device="cuda").manual_seed(far)
    s.a[0][:, ::8] *= 2.0 ** (far // 2)
    s.a[0][:, :, 5::16] = 0
    s.b[0][:, :, ::8] = 0
    x = torch.randn(rows, k, device="cuda", generator=gen)
    x[:, 5::16] *= 2.0 ** far
    base = torch.randn(rows, outs[0], device="cuda", generator=gen)
    y, slot = torch.empty_like(base), mixed(rows, slots) if rows > 1 else [0]
    plan, _ = s.plan(slot)
    s.ad.ApplyCUDA(s.group, plan.data_ptr(), rows, x.data_ptr(), [y.data_ptr()], [base.data_ptr()])
    torch.cuda.synchronize()
    (want, tol), = s.want(x, slot, [base])
    if dtype == "f16":
        for i, v in enumerate(slot):
            if v < 0:
                continue
            A, B, f = s.a[0][v].double().abs(), s.b[0][v].double().abs(), abs(float(s.scale[0][v]))
            t = (s.a[0][v].double() @ x[i].double()).abs().max()
            tol[i] += 2.0 ** -32 * f * (B @ (A.sum(1) * float(x[i].abs().max())) + B.sum(1) * t)
    err = (y.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
