"""Long splits of the shared attention, which a block takes in stretches: keys whose logits rise or fall from one stretch to the next by more than a weight reaches,
drafted tokens that see unlike ends, values that are not finite and pages outside the pool in one stretch alone."""
import numpy as np
import pytest
import torch
from test_gpu_paged import Cache, attn64, bound

pytestmark = pytest.mark.gpu
N = 9000                                                                   # four stretches of 2560 keys, or eight of 1280


@pytest.fixture(autouse=True)
def always(hooks):
    hooks.wv_set_attn_sharing(1)
    yield
    hooks.wv_set_attn_sharing(0)


class Lone(Cache):
    """One sequence under bounds that let all of it be shared, in a group that shares nothing: few splits of its own keys."""

    def __init__(self, wv, bits, hd, tokens, k, v):
        super().__init__(wv, bits, 64, 1, hd, [(tokens, N)])
        self.fill(k, v)
        self.tokens, self.ints = tokens, [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [0, 0])]
        self.groups = wv.paged.Groups(self.ints[0].data_ptr(), self.ints[1].data_ptr(), 1, N)

    def attend(self, q, heads, scale):
        out = torch.full_like(q, 77.0)
        self.wv.paged.AttnSharedCUDA(self.pages, self.batch, self.groups, q.data_ptr(), out.data_ptr(), heads, scale)
        torch.cuda.synchronize()
        return out


def data(hd, heads, tokens, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *n: torch.randn(*n, device="cuda", generator=gen)  # noqa: E731
    return r(N, hd), r(N, hd), r(tokens, heads * hd)


@pytest.mark.parametrize("bits,hd,heads,tokens", [(8, 64, 8, 1), (16, 128, 8, 1), (4, 128, 8, 2), (8, 80, 4, 4), (4, 48, 3, 5), (16, 256, 4, 1), (8, 192, 8, 2)])
@pytest.mark.parametrize("walk", ["even", "rising", "falling", "a peak"])
def test_logits_from_stretch_to_stretch(wv, bits, hd, heads, tokens, walk):
    k, v, q = data(hd, heads, tokens, bits + hd)
    at = torch.arange(N, device="cuda") / N
    k *= {"even": torch.ones_like(at), "rising": 0.1 + 8 * at, "falling": 8.1 - 8 * at, "a peak": torch.where((at > 0.5) & (at < 0.51), 12.0, 0.5)}[walk][:, None]
    c = Lone(wv, bits, hd, tokens, k, v)
    got = c.attend(q, heads, hd ** -0.5)
    assert wv._lib.lib().wv_device_status() == 0
    want, mag, reach = attn64(q.cpu().numpy().reshape(tokens, heads, hd), c.rows("k"), c.rows("v"), hd ** -0.5, 0, N - tokens)
    err = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    # a weight counts to 2^-28 of its row's largest (the entry's stated range)
    tol = bound(mag, reach, hd, N) + N * 2.0 ** -28 * float(v.abs().max())
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("heads,tokens", [(8, 1), (8, 2)])
@pytest.mark.parametrize("key", [5, 4000, 8990])
def test_a_value_that_is_not_finite(wv, heads, tokens, key):
    k, v, q = data(64, heads, tokens, key)
    v[key, 3] = float("nan")
    assert torch.isnan(Lone(wv, 8, 64, tokens, k, v).attend(q, heads, 0.125)).all()
    v[key, 3] = 0
    assert not torch.isnan(Lone(wv, 8, 64, tokens, k, v).attend(q, heads, 0.125)).any()


@pytest.mark.parametrize("heads,tokens", [(8, 1), (8, 2)])
@pytest.mark.parametrize("first,last", [(0, 2560), (2560, 5120), (7680, 9000), (0, 9000)])
def test_pages_outside_the_pool(wv, heads, tokens, first, last):
    """A whole stretch without keys, the first, a middle or the last one, and all of them: the others' keys alone, and zeros where there are none."""
    k, v, q = data(64, heads, tokens, first)
    c = Lone(wv, 8, 64, tokens, k, v)
    kk, vv = c.rows("k"), c.rows("v")
    c.d_table[0, first // 64:-(-last // 64)] = 10 ** 6
    got = c.attend(q, heads, 0.125).double().cpu().numpy().reshape(tokens, heads, 64)
    assert wv._lib.lib().wv_device_status() == wv._lib.WV_ESHAPE
    for i in range(tokens):
        see = np.r_[0:first, last:N - tokens + 1 + i]
        if not len(see):
            assert not got[i].any()
            continue
        want, mag, reach = attn64(q.cpu().numpy().reshape(tokens, heads, 64)[i:i + 1], kk[see], vv[see], 0.125, 0, len(see) - 1)
        assert (np.abs(got[i] - want[0]) <= bound(mag, reach, 64, N)[0]).all()
