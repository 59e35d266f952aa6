"""Paged attention over values that are infinite or NaN at positions that rows
do see. Such a row's element is what the sum of positive weights times values
is: infinite, with the sign of the infinities if they have one sign, NaN
otherwise; its other elements are as without them."""
import pytest
import torch

from test_gpu_paged import attend, make, visible
from test_gpu_paged_nan import SHAPES

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def expected(s, clean, window, sinks):
    """`clean` (the result without them) with the elements that a value which
    is not finite reaches."""
    B, T, nh, nkv, d, ps = (s[x] for x in ("B", "T", "nh", "nkv", "d", "ps"))
    rep, want = nh // nkv, clean.float().view(B, T, nkv, nh // nkv, d).clone()
    for b in range(B):
        for t in range(T):
            j = visible(s, b, t, window, sinks)
            v = s["v"][s["table"][b, j // ps].long(), :, j % ps].float()  # [keys, nkv, d]
            bad = torch.where(torch.isfinite(v), torch.zeros_like(v), v)
            hit = ~torch.isfinite(v).all(0)                               # [nkv, d]
            sums = bad.sum(0)                                             # inf, -inf or NaN where hit
            want[b, t] = torch.where(hit[:, None].expand(nkv, rep, d), sums[:, None], want[b, t])
    return want.view(B * T, nh * d)


def same(out, want):
    out = out.float()
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(torch.isinf(out) * torch.sign(out).nan_to_num(), torch.isinf(want) * torch.sign(want).nan_to_num())
    fine = torch.isfinite(want)
    assert torch.equal(out[fine], want[fine])


@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 3)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_that_are_seen(rb, shape, window, sinks):
    B, T, nh, nkv, d, ps, lens = shape
    s = make(*shape)
    clean, v0 = attend(rb, s, window, sinks), s["v"].clone()
    for value in (INF, -INF, NAN):
        for b in range(B):
            # Early keys, keys about the call's own tokens, the last key; a
            # dimension of its own for each, so that the others stay clean.
            places = sorted({0, 1, 2, lens[b] // 2, max(0, lens[b] - T), max(0, lens[b] - T - 10),
                             lens[b] - T // 2 - 1, lens[b] - 1})
            for i, j in enumerate(p for p in places if p < lens[b]):
                s["v"][s["table"][b, j // ps].long(), i % nkv, j % ps, 7 * i + 1] = value
        same(attend(rb, s, window, sinks), expected(s, clean, window, sinks))
        s["v"].copy_(v0)


@pytest.mark.parametrize("T", [1, 4, 80, 300])
def test_both_signs(rb, T):
    """+inf and -inf in one column, at keys that rows see alone and together."""
    s = make(1, T, 8, 2, 128, 16, [200 + T])
    clean = attend(rb, s)
    for j, value in ((100, INF), (201, -INF)):
        s["v"][s["table"][0, j // 16].long(), :, j % 16, 5] = value
    for j in (3, 150):
        s["v"][s["table"][0, j // 16].long(), :, j % 16, 9] = -INF
    same(attend(rb, s), expected(s, clean, 0, 0))
