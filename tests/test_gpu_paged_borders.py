"""Paged attention's borders, key by key, and the few-row kernel's weights.

With q = 0 every weight is exactly 1 and a row's result is the mean of the
values it sees: a value at one key alone, 0 elsewhere, comes out as itself
over the number of keys, or as 0 where the row does not see it. A key lost or
seen twice is thereby off by all of it, however long the cache. Tolerance: the
sums and the number of keys are exact, their quotient is rounded in float32
(three times at most, 2^-22) and once to bf16 (2^-8).
"""
import math

import pytest
import torch

from test_gpu_paged import attend, make, visible

pytestmark = pytest.mark.gpu

# (B, T, nh, nkv, d, page_size, lengths, window, sinks)
LONG = [(1, 1, 32, 8, 128, 16, [30001], 0, 0), (1, 1, 16, 8, 64, 64, [16385], 0, 0),
        (2, 1, 32, 8, 128, 32, [9000, 20011], 4096, 4), (1, 4, 32, 8, 128, 16, [12003], 0, 0),
        (3, 2, 32, 8, 64, 128, [5000, 2, 7001], 1000, 70), (2, 6, 48, 8, 128, 32, [6, 4001], 0, 0),
        (1, 32, 32, 8, 128, 16, [8005], 0, 0), (1, 20, 32, 8, 64, 64, [9001], 2048, 4),
        (1, 300, 8, 8, 128, 64, [5000], 0, 0), (1, 300, 16, 8, 64, 16, [5000], 1000, 4),
        (1, 130, 32, 8, 128, 128, [2311], 0, 0), (70, 1, 32, 8, 128, 16, [1 + 61 * i for i in range(70)], 0, 0)]


@pytest.mark.parametrize("case", LONG, ids=str)
def test_every_border(rb, case):
    B, T, nh, nkv, d, ps, lens, window, sinks = case
    s = make(*case[:7])
    s["q"].zero_()
    s["v"].zero_()
    rep, slots = nh // nkv, nkv * d
    want = torch.zeros(B, T, nkv, rep, d, dtype=torch.float64, device="cuda")
    for b in range(B):
        n = lens[b]
        ends = [0, 1, n - 1, n - T, n - T - 1, sinks - 1, sinks]
        if window:
            ends += [p - window + e for p in (n - T, n - 1) for e in (-1, 0, 1, 2)]
        ends += [j for i in range(0, n, 64) for j in (i, i + 63)]
        ends += [j for i in range(0, n, 16) for j in (i, i + 15)]
        keys = list(dict.fromkeys(j for j in ends if 0 <= j < n))[:slots]
        j = torch.tensor(keys, device="cuda")
        i = torch.arange(len(keys), device="cuda")
        value = torch.exp2((i % 5 + 8).float())
        s["v"][s["table"][b, j // ps].long(), i // d, j % ps, i % d] = value.to(torch.bfloat16)
        for t in range(T):
            seen = visible(s, b, t, window, sinks)
            if seen.numel():
                want[b, t, i // d, :, i % d] = (torch.isin(j, seen) * value.double() / seen.numel())[:, None]
    out = attend(rb, s, window, sinks).double().view(B, T, nkv, rep, d)
    assert torch.equal(out == 0, want == 0)
    assert ((out - want).abs() <= want * (2.0 ** -8 + 2.0 ** -22)).all()


@pytest.mark.parametrize("T,nh,d", [(1, 8, 128), (1, 32, 64), (4, 8, 64), (2, 16, 128)])
def test_few_rows_keep_15_bits_of_a_weight(rb, T, nh, d):
    """Three values that almost cancel, so that the output's rounding does not
    hide the weights' errors. A weight is held as two bf16 numbers, the first
    above 1 - 2^-7 of it, so the second's rounding is 2^-8 of 2^-7 of it.
    Scores come from one product, exact in float32, and lie within 8 octaves:
    their rounding, the exponential and the sums are below 2^-18 of A. A
    weight rounded once to bf16 is off by up to 2^-8: that alone, put into the
    64-bit form, is far outside."""
    nkv, L, g = 2, T + 2, torch.Generator().manual_seed(T * 100 + d)
    B, rep = 16, nh // nkv
    s = make(B, T, nh, nkv, d, 16, [L] * B)
    s["pos"].fill_(L - 1)   # every row sees all L keys ...
    s["table"][:, 1:] = -1
    page = s["table"][:, 0].long().cpu()
    q, k, v = (torch.zeros_like(s[x], device="cpu", dtype=torch.float64) for x in ("q", "k", "v"))
    q.view(B, T, nh, d)[..., 0] = (torch.rand(B, T, nh, generator=g).double() + 0.5).bfloat16().double()
    k[page, :, :3, 0] = (torch.rand(B, nkv, 3, generator=g).double() * 3.0 * math.sqrt(d / 64)).bfloat16().double()
    k[page, :, 3:, 0] = -2.0 ** 14  # ... but all except three have no weight
    score = torch.einsum("btgr,bgj->bgtrj", q.view(B, T, nkv, rep, d)[..., 0], k[page, :, :, 0]) / math.sqrt(d)
    score[..., L:] = -math.inf
    p = torch.softmax(score, -1)[..., :3].reshape(B, nkv, T * rep, 3)
    row = torch.arange(d) % (T * rep)                     # the row whose result dimension i is to be nearly 0
    v[page, :, 0] = (torch.rand(B, nkv, d, generator=g).double() + 0.5).bfloat16().double()
    v[page, :, 1] = (torch.rand(B, nkv, d, generator=g).double() - 0.5).bfloat16().double()
    at = p[:, :, row]                                     # [B, nkv, d, 3]
    v[page, :, 2] = (-(at[..., 0] * v[page, :, 0] + at[..., 1] * v[page, :, 1]) / at[..., 2]).bfloat16().double()
    for name, x in (("q", q), ("k", k), ("v", v)):
        s[name].copy_(x)
        assert torch.equal(s[name].double().cpu(), x)
    vv = v[page, :, :3]                                   # [B, nkv, 3, d]
    want, A = p @ vv, p @ vv.abs()
    tol = want.abs() * 2.0 ** -8 + A * (2.0 ** -15 + 2.0 ** -18)
    out = attend(rb, s).double().cpu().view(B, T, nkv, rep, d).permute(0, 2, 1, 3, 4).reshape(B, nkv, T * rep, d)
    assert ((out - want).abs() <= tol).all()
    top = p.amax(-1, keepdim=True)
    once = ((p / top).bfloat16().double() * top) @ vv
    assert ((once - want).abs() > 8 * tol).any()


@pytest.mark.parametrize("shape", [(2, 6, 48, 8, 128, 32, [4001, 77]), (1, 700, 32, 8, 128, 64, [900]),
                                   (3, 1, 32, 8, 128, 16, [9000, 3, 500]), (2, 300, 16, 2, 64, 16, [2000, 300])], ids=str)
def test_same_bits_every_time(rb, shape):
    s = make(*shape)
    first = attend(rb, s)
    for _ in range(10):
        assert torch.equal(attend(rb, s), first)
