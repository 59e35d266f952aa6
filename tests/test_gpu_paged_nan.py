"""Paged attention of rows whose scores are NaN: the row shows it, however
many rows the call has, and the others do not."""
import pytest
import torch

from test_gpu_paged import attend, make

pytestmark = pytest.mark.gpu

NAN = float("nan")

# (B, T, nh, nkv, d, page_size, lengths): single tokens and drafted ones up to
# a tile's 16 rows, up to 128, prompts; groups whole and cut over shares.
SHAPES = [(2, 1, 8, 2, 128, 16, [40, 1]), (2, 1, 8, 2, 64, 32, [130, 6000]), (1, 1, 8, 2, 128, 16, [20000]),
          (2, 4, 8, 2, 128, 16, [4, 90]), (1, 4, 16, 4, 64, 64, [7000]), (2, 5, 8, 2, 128, 32, [5, 300]),
          (1, 5, 8, 2, 64, 16, [9000]), (2, 80, 8, 2, 128, 16, [80, 500]), (1, 80, 8, 2, 64, 16, [4000]),
          (1, 300, 8, 1, 128, 64, [700])]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_nan_query(rb, shape):
    """NaN in one head of one row's query: that head's row alone is NaN."""
    s = make(*shape)
    clean = attend(rb, s)
    B, T, nh, _, d = shape[:5]
    for b, t, h in ((0, 0, 0), (B - 1, T - 1, nh - 1), (0, T // 2, nh // 2)):
        q0 = s["q"].clone()
        s["q"].view(B, T, nh, d)[b, t, h, 3] = NAN
        out, want = attend(rb, s).view(B, T, nh, d), clean.clone().view(B, T, nh, d)
        s["q"].copy_(q0)
        assert torch.isnan(out[b, t, h]).all()
        out[b, t, h] = want[b, t, h]
        assert torch.equal(out, want)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_nan_keys(rb, shape):
    """Every key NaN, of one kv head: its heads' rows are NaN. And the keys of
    positions 64 to 191 alone: the same for rows that see any of them."""
    B, T, nh, nkv, d, ps, lens = shape
    s = make(*shape)
    clean, rep = attend(rb, s).view(B, T, nkv, nh // nkv, d), nh // nkv
    k0 = s["k"].clone()
    s["k"][:, nkv - 1] = NAN
    out = attend(rb, s).view(B, T, nkv, rep, d)
    assert torch.isnan(out[:, :, nkv - 1]).all() and torch.equal(out[:, :, :nkv - 1], clean[:, :, :nkv - 1])
    s["k"].copy_(k0)
    j = torch.arange(64, 192, device="cuda")
    for b in range(B):
        at = j[j < lens[b]]
        s["k"][s["table"][b, at // ps].long(), 0, at % ps] = NAN
    out = attend(rb, s).view(B, T, nkv, rep, d)
    p = s["pos"].long()[:, None] + torch.arange(T, device="cuda")
    hit = p >= 64
    assert torch.isnan(out[:, :, 0][hit]).all() and torch.isfinite(out[:, :, 0][~hit]).all()
    assert torch.equal(out[:, :, 1:], clean[:, :, 1:])


@pytest.mark.parametrize("T", [1, 4, 5, 80, 300])
def test_only_key_is_nan(rb, T):
    """One key in the whole cache, and it is NaN: rows that see it are NaN,
    the others see nothing and are zero."""
    s = make(1, T, 8, 2, 128, 16, [T])
    s["pos"].fill_(-(T // 2))
    s["table"][:, 1:] = -1
    s["k"][s["table"][0, 0].long(), :, 0] = NAN
    out = attend(rb, s, 1).view(T, -1)
    t = torch.arange(T, device="cuda") - T // 2
    assert torch.isnan(out[t == 0]).all() and (out[t < 0] == 0).all()
    assert torch.isfinite(out[t > 0]).all()
