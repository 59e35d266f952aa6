"""The rotary append into pages and the attention over them against plain
64-bit implementations.

Tolerances. A stored bf16 value is off by at most half a step, 2^-8 of it.
Attention: a row's result is sum_j p_j v_j with sum p_j = 1. Rounding each
weight to bf16 moves it by at most 2^-8 A, A = sum_j p_j |v_j|. A float32
score is off by at most d 2^-24 sum_i |q_i k_i| / sqrt(d), under 2^-12 for
the inputs here (sum |q k| < 250, d = 128), which moves the weights by the
same share, numerator and denominator: 2^-11 A. In all
2^-8 |out| + (2^-8 + 2^-11) A. Rotation: two float32 products and a sum,
3 2^-24 (|x1| + |x2|), and an angle good to 2^-22: within 2^-20 (|x1| + |x2|).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

NAN = float("nan")


def _bf(*shape, gen, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(torch.bfloat16)


def make(B, T, nh, nkv, d, ps, lens, seed=0, extra=3, holes=(), fill=None, width=None):
    """A cache whose sequences hold lens[b] positions (this call's T last
    ones among them), pages in random order, table entries past them -1."""
    g = torch.Generator(device="cuda").manual_seed(seed * 1009 + B * 31 + T)
    per = [-(-max(0, n) // ps) for n in lens]
    width = max(1, max(per)) if width is None else width
    num = sum(per) + extra
    order = torch.randperm(num, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table, at = torch.full((B, width), -1, dtype=torch.int32), 0
    for b in range(B):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
    for b, i, value in holes:
        table[b, i] = value
    s = dict(B=B, T=T, nh=nh, nkv=nkv, d=d, ps=ps, table=table.cuda(),
             pos=torch.tensor([n - T for n in lens], dtype=torch.int32, device="cuda"),
             q=_bf(B * T, nh * d, gen=g, scale=1.5), k=_bf(num, nkv, ps, d, gen=g), v=_bf(num, nkv, ps, d, gen=g))
    return s


def visible(s, b, t, window, sinks):
    """Positions that row (b, t) sees, ascending."""
    p = int(s["pos"][b]) + t
    j = torch.arange(s["table"].shape[1] * s["ps"], device="cuda")
    ok = (j <= p) & ((s["table"][b] >= 0) & (s["table"][b] < s["k"].shape[0])).repeat_interleave(s["ps"])
    if window:
        ok &= (j > p - window) | (j < sinks)
    return j[ok]


def reference(s, window=0, sinks=0):
    """(out, A) in 64 bits, a row and a head at a time over the keys seen."""
    B, T, nh, nkv, d, ps = (s[x] for x in ("B", "T", "nh", "nkv", "d", "ps"))
    rep = nh // nkv
    out = torch.zeros(B * T, nh, d, dtype=torch.float64, device="cuda")
    A = torch.zeros_like(out)
    q = s["q"].view(B * T, nh, d).double()
    for b in range(B):
        for t in range(T):
            j = visible(s, b, t, window, sinks)
            if j.numel() == 0:
                continue
            page = s["table"][b, j // ps].long()
            for kh in range(nkv):
                k, v = s["k"][page, kh, j % ps].double(), s["v"][page, kh, j % ps].double()
                h = slice(kh * rep, (kh + 1) * rep)
                p = torch.softmax(q[b * T + t, h] @ k.t() / math.sqrt(d), -1)
                out[b * T + t, h], A[b * T + t, h] = p @ v, p @ v.abs()
    return out.view(B * T, nh * d), A.view(B * T, nh * d)


def attend(rb, s, window=0, sinks=0, **kw):
    return rb.paged_attention(s["q"], s["pos"], s["table"], s["k"], s["v"], window=window, sinks=sinks, **kw)


def check(out, ref):
    want, A = ref
    err = (out.double() - want).abs()
    tol = want.abs() * 2.0 ** -8 + A * (2.0 ** -8 + 2.0 ** -11) + 1e-30
    assert torch.isfinite(out.float()).all()
    worst = (err / tol).max().item()
    assert worst <= 1.0, f"error {worst:.2f} times the tolerance"


def poison(s, window=0, sinks=0):
    """NaN and infinities wherever no row of the call sees the position."""
    seen = torch.zeros(s["k"].shape[0], s["ps"], dtype=torch.bool, device="cuda")
    for b in range(s["B"]):
        for t in range(s["T"]):
            j = visible(s, b, t, window, sinks)
            seen[s["table"][b, j // s["ps"]].long(), j % s["ps"]] = True
    bad = (~seen)[:, None, :, None].expand_as(s["k"])
    for x, value in ((s["k"], NAN), (s["v"], float("inf"))):
        x[bad] = value
    s["v"][..., ::2][bad[..., ::2]] = NAN
    return s


# (B, T, nh, nkv, d, page_size, lengths): single tokens; one key; empty
# sequences (length 0 gives p = -1); ragged; page ends inside tiles; drafted
# tokens; more heads per kv head; T * rep beyond one tile.
SHAPES = [
    (1, 1, 32, 8, 128, 16, [57]),
    (1, 1, 8, 2, 128, 16, [1]),
    (3, 1, 8, 2, 128, 32, [0, 65, 2]),
    (4, 1, 32, 4, 64, 64, [700, 64, 65, 1]),
    (2, 1, 48, 8, 128, 128, [129, 1000]),
    (2, 1, 4, 4, 64, 16, [333, 15]),
    (1, 1, 16, 1, 64, 16, [200]),
    (2, 1, 15, 5, 128, 16, [77, 130]),
    (2, 3, 8, 2, 128, 16, [3, 100]),
    (3, 6, 48, 8, 128, 32, [6, 301, 4]),
    (2, 8, 16, 2, 64, 16, [8, 523]),
    (1, 17, 8, 2, 128, 64, [17]),
    (2, 33, 32, 8, 128, 32, [40, 161]),
    (1, 130, 8, 2, 128, 16, [130]),
    (2, 65, 16, 2, 64, 64, [65, 300]),
    (1, 257, 8, 1, 128, 128, [400]),
    (1, 40, 48, 8, 128, 16, [555]),
    (2, 1, 32, 1, 128, 16, [90, 300]),
    (1, 1, 128, 1, 64, 32, [700]),
    (2, 3, 64, 1, 64, 16, [40, 130]),
    (1, 5, 33, 1, 128, 64, [200]),
]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 4), (100, 70)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(rb, shape, window, sinks):
    s = poison(make(*shape), window, sinks)
    check(attend(rb, s, window, sinks), reference(s, window, sinks))


# 17 to 64 rows per kv head: each number of row tiles, whole and not, many
# sequences, few long ones.
SOME_ROWS = [
    (2, 17, 4, 4, 128, 16, [17, 130]),
    (3, 5, 32, 8, 128, 64, [700, 5, 64]),
    (2, 8, 8, 2, 64, 16, [8, 1000]),
    (2, 11, 6, 2, 128, 32, [11, 333]),
    (40, 6, 12, 2, 128, 32, [6 + (i * 53) % 300 for i in range(40)]),
    (2, 4, 24, 2, 64, 128, [260, 7]),
    (1, 7, 14, 2, 128, 16, [4001]),
    (2, 9, 14, 2, 64, 64, [1500, 77]),
    (3, 16, 8, 2, 128, 16, [16, 81, 500]),
    (1, 1, 64, 1, 128, 16, [900]),
    (2, 1, 39, 1, 64, 32, [33, 1200]),
]


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (20, 4), (100, 70)])
@pytest.mark.parametrize("shape", SOME_ROWS, ids=str)
def test_attention_some_rows(rb, shape, window, sinks):
    s = poison(make(*shape), window, sinks)
    check(attend(rb, s, window, sinks), reference(s, window, sinks))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T", [5, 9, 13, 16])
def test_some_rows_later_token(rb, T, d):
    """A token that is not finite does not reach the rows before it, in
    whichever row tile they lie; the pool itself is not changed."""
    s = make(2, T, 8, 2, d, 32, [150 + T, 40 + T])
    clean, k0, v0 = attend(rb, s), s["k"].clone(), s["v"].clone()
    for b, start in ((0, 150), (1, 40)):
        for off in (0, T // 2, T - 1):
            at = start + off
            page, slot = int(s["table"][b, at // 32]), at % 32
            for name, value in (("v", NAN), ("v", float("inf")), ("k", NAN)):
                s[name][page, :, slot] = value
                held = s[name].clone()
                out = attend(rb, s).float().view(2, T, -1)
                assert torch.equal(torch.nan_to_num(s[name].float(), 7.0), torch.nan_to_num(held.float(), 7.0))
                s["k"].copy_(k0), s["v"].copy_(v0)
                want = clean.float().view(2, T, -1)
                assert torch.equal(out[1 - b], want[1 - b]) and torch.equal(out[b, :off], want[b, :off])
                assert not torch.isfinite(out[b, off:]).any()


@pytest.mark.parametrize("B,T,lens,window", [(1, 1, [30001], 0), (2, 1, [9000, 20011], 4096), (1, 4, [12003], 0),
                                             (300, 1, [1 + (i * 37) % 400 for i in range(300)], 0),
                                             (1, 300, [5000], 1000)])
def test_attention_long(rb, B, T, lens, window):
    """Long caches (split over the keys) and many short sequences."""
    s = make(B, T, 8, 2, 128, 16, lens)
    check(attend(rb, s, window, 4), reference(s, window, 4))


@pytest.mark.parametrize("T", [1, 5, 80])
def test_pages_not_held(rb, T):
    """Entries outside the pool inside a sequence, and a sequence with none."""
    lens = [100, 90, 128]
    s = make(3, T, 8, 2, 128, 16, lens, holes=[(0, 0, -1), (0, 2, 10**6), (0, 3, -2**31), (1, 5, 2**31 - 1)]
             + [(2, i, -1) for i in range(8)])
    poison(s)
    out = attend(rb, s)
    check(out, reference(s))
    assert (out.view(3, T, -1)[2] == 0).all()


@pytest.mark.parametrize("T", [1, 4, 70])
def test_rows_outside_the_cache(rb, T):
    """Positions before 0 (a padded batch) give zeros; positions past the
    table see what the table holds."""
    s = make(3, T, 8, 2, 64, 16, [100, 100, 100])
    s["pos"] = torch.tensor([-T - 5, -(T // 2), 95], dtype=torch.int32, device="cuda")
    out = attend(rb, s)
    check(out, reference(s))
    assert (out.view(3, T, -1)[0] == 0).all()
    s["pos"] = torch.tensor([2**31 - 1, -2**31, 111], dtype=torch.int32, device="cuda")
    check(attend(rb, s), reference(s))
    check(attend(rb, s, 64, 3), reference(s, 64, 3))


@pytest.mark.parametrize("T", [2, 6, 100])
@pytest.mark.parametrize("window", [0, 40])
def test_later_token_does_not_reach_earlier_rows(rb, T, window):
    """NaN, +inf and -inf in the keys and values of a token of the call: the
    rows before it (and those whose window is past it) are as without it."""
    s = make(1, T, 8, 2, 128, 16, [150 + T])
    clean = attend(rb, s, window)
    at = 150 + T // 2
    page, slot = int(s["table"][0, at // 16]), at % 16
    for name, value in (("v", NAN), ("v", float("inf")), ("v", -float("inf")), ("k", NAN), ("k", float("inf"))):
        x = s[name].clone()
        s[name][page, :, slot] = value
        out = attend(rb, s, window).float()
        s[name].copy_(x)
        p = 150 + torch.arange(T, device="cuda")
        sees = (p >= at) & ((p - at < window) if window else True)
        assert torch.equal(out[~sees], clean[~sees].float())
        assert not torch.isfinite(out[sees]).any()


def test_shared_pages_and_strided_table(rb):
    """Two sequences over one prefix, and a table that is a slice of a wider
    one."""
    s = make(2, 1, 8, 2, 128, 16, [64, 70])
    wide = torch.full((2, 40), 7, dtype=torch.int32, device="cuda")
    wide[:, :5] = s["table"]
    wide[1, :4] = wide[0, :4]
    s["table"] = wide[:, :5]
    check(attend(rb, s), reference(s))
    s["table"] = wide[:, :3]  # fewer positions than pos says
    check(attend(rb, s), reference(s))


@pytest.mark.parametrize("T", [1, 130])
def test_pool_beyond_32_bit_offsets(rb, T):
    """Pages whose first element lies past 2^31, and past 2^32 bytes."""
    num, nkv, ps, d = 20000, 8, 128, 128  # 2.6e9 elements
    k = torch.empty(num, nkv, ps, d, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    small = make(1, T, 32, nkv, d, ps, [300])
    pages = torch.tensor([num - 1, 16500, 3], device="cuda")
    k[pages], v[pages] = small["k"][:3], small["v"][:3]
    s = dict(small, k=k, v=v, table=pages.to(torch.int32)[None])
    ref = dict(small, k=small["k"][:3], v=small["v"][:3], table=torch.tensor([[0, 1, 2]], device="cuda"))
    check(attend(rb, s), reference(ref))


def test_streams_graphs_and_repeats(rb):
    """Two calls at once on two streams, a captured and replayed call whose
    lengths change, and the same bits every time."""
    a, b = make(1, 1, 32, 8, 128, 16, [6000]), make(2, 1, 32, 8, 128, 64, [5000, 1], seed=5)
    ra, rb_ = attend(rb, a), attend(rb, b)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            x = [attend(rb, a) for _ in range(4)]
        with torch.cuda.stream(s2):
            y = [attend(rb, b) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, ra) for o in x) and all(torch.equal(o, rb_) for o in y)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = attend(rb, a)
    with torch.cuda.graph(g2):
        o2 = attend(rb, b)
    for n in (6000, 17, 1, 3001):
        a["pos"].fill_(n - 1)
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            g1.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        torch.cuda.synchronize()
        check(o1, reference(a))
        assert torch.equal(o2, rb_)


def test_attention_out_and_refusals(rb):
    s = make(1, 1, 8, 2, 128, 16, [40])
    out = torch.empty_like(s["q"])
    assert attend(rb, s, out=out) is out
    check(out, reference(s))
    for bad in (dict(q=s["q"].float()), dict(k=s["k"].transpose(1, 2)), dict(v=s["v"][:2]),
                dict(pos=s["pos"].long()), dict(table=s["table"].long()), dict(table=s["table"].cpu()),
                dict(q=s["q"][:, :100]), dict(q=s["q"][:, ::2]), dict(q=torch.cat([s["q"]] * 65, 1)),
                dict(table=torch.cat([s["table"]] * 2))):
        with pytest.raises(rb.ConfigError):
            attend(rb, dict(s, **bad))
    with pytest.raises(rb.ConfigError, match="negative"):
        attend(rb, s, window=-1)
    for bad in (2**31, 1.5, None):
        with pytest.raises(rb.ConfigError, match="32-bit"):
            attend(rb, s, window=bad)
    with pytest.raises(rb.ConfigError, match="out must"):
        attend(rb, s, out=out.float())
    shifted = torch.empty(8 * 128 + 8, dtype=torch.bfloat16, device="cuda")[1:8 * 128 + 1].view(1, -1)
    with pytest.raises(rb.RiallmError, match="aligned"):
        attend(rb, dict(s, q=shifted))
    empty = dict(s, q=s["q"][:0])
    assert attend(rb, empty).shape == (0, 8 * 128)


# ----------------------------------------------------------------- append

def _rotated(x, p, inv_freq):
    """x [rows, heads, d] at positions p [rows], in 64 bits."""
    h = x.shape[-1] // 2
    a, b = x.double()[..., :h], x.double()[..., h:]
    ang = p.double()[:, None, None] * inv_freq.double()
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


@pytest.mark.parametrize("B,T,nh,nkv,d,ps,pos", [
    (1, 1, 32, 8, 128, 16, [0]), (3, 1, 8, 2, 128, 32, [31, 32, 95]), (2, 5, 48, 8, 128, 16, [13, 90]),
    (2, 70, 32, 4, 64, 64, [0, 25]), (4, 3, 4, 4, 64, 128, [-2, -3, 254, 300]), (1, 1, 16, 1, 64, 16, [7]),
    (3, 2, 15, 5, 64, 16, [2**31 - 2, -2**31, 5]), (1, 513, 8, 2, 128, 16, [0])])
def test_append(rb, B, T, nh, nkv, d, ps, pos):
    width = 2 if ps == 128 else (600 if T > 100 else 110) // ps
    s = make(B, T, nh, nkv, d, ps, [width * ps] * B, holes=[(B - 1, width // 2, -1)] if B > 1 else ())
    g = torch.Generator(device="cuda").manual_seed(T)
    qkv = _bf(B * T, (nh + 2 * nkv) * d, gen=g, scale=2.0)
    qkv.view(-1)[5] = float("inf")       # a q element; its pair is not finite either
    qkv[-1, (nh + nkv) * d + 3] = NAN    # v is copied as it is
    inv = torch.tensor([1e6 ** (-i / d) for i in range(0, d, 2)], dtype=torch.float32, device="cuda")
    s["pos"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
    k0, v0 = s["k"].clone(), s["v"].clone()
    q = rb.rope_paged_append(qkv, s["pos"], s["table"], s["k"], s["v"], inv)
    p = (s["pos"].long()[:, None] + torch.arange(T, device="cuda")).reshape(-1)
    x = qkv.view(B * T, nh + 2 * nkv, d)
    want = _rotated(x[:, :nh + nkv], p, inv)
    h = d // 2
    mag = x[:, :nh + nkv].double().abs()
    tol = want.abs() * 2.0 ** -8 + 2.0 ** -20 * (mag[..., :h] + mag[..., h:]).repeat(1, 1, 2) + 1e-30

    def close(got, want, tol):
        fine = torch.isfinite(want)
        assert torch.equal(fine, torch.isfinite(got.float()))
        assert ((got.double() - want).abs()[fine] <= tol[fine]).all()
    close(q.view(B * T, nh, d), want[:, :nh], tol[:, :nh])
    for i in range(B * T):
        b, j = i // T, int(p[i])
        if not 0 <= j < width * ps or int(s["table"][b, j // ps]) < 0:
            continue
        page, slot = int(s["table"][b, j // ps]), j % ps
        close(s["k"][page, :, slot], want[i, nh:], tol[i, nh:])
        assert torch.equal(s["v"][page, :, slot].view(torch.int16), x[i, nh + nkv:].view(torch.int16))
        k0[page, :, slot], v0[page, :, slot] = s["k"][page, :, slot], s["v"][page, :, slot]
    assert torch.equal(s["k"].view(torch.int16), k0.view(torch.int16))  # nothing else was written
    assert torch.equal(s["v"].view(torch.int16), v0.view(torch.int16))


def test_append_far_positions(rb):
    """Angles of positions up to 2^31: as exact as near ones."""
    p = torch.tensor([100003, 2**24 + 1, 2**30 + 12345, 2**31 - 1], dtype=torch.int32, device="cuda")
    s = make(4, 1, 8, 2, 128, 16, [16] * 4)
    inv = torch.tensor([1e6 ** (-i / 128) for i in range(0, 128, 2)], dtype=torch.float32, device="cuda")
    qkv = _bf(4, 12 * 128, gen=torch.Generator(device="cuda").manual_seed(3))
    q = rb.rope_paged_append(qkv, p, s["table"], s["k"], s["v"], inv)
    want = _rotated(qkv.view(4, 12, 128)[:, :8], p.long(), inv)
    mag = qkv.view(4, 12, 128)[:, :8].double().abs()
    tol = want.abs() * 2.0 ** -8 + 2.0 ** -20 * (mag[..., :64] + mag[..., 64:]).repeat(1, 1, 2)
    assert ((q.view(4, 8, 128).double() - want).abs() <= tol).all()


def test_append_refusals_and_out(rb):
    s = make(1, 1, 8, 2, 128, 16, [40])
    inv = torch.ones(64, device="cuda")
    qkv = torch.zeros(1, 12 * 128, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(1, 1024, dtype=torch.bfloat16, device="cuda")
    ok = dict(qkv=qkv, pos=s["pos"], page_table=s["table"], k_pages=s["k"], v_pages=s["v"], inv_freq=inv)
    assert rb.rope_paged_append(**ok, q_out=out) is out
    for bad in (dict(qkv=qkv[:, :4 * 128]), dict(qkv=qkv.half()), dict(inv_freq=inv[:63]), dict(inv_freq=inv.double()),
                dict(k_pages=s["k"][:, :1]), dict(pos=s["pos"].cpu())):
        with pytest.raises(rb.ConfigError):
            rb.rope_paged_append(**dict(ok, **bad))
    with pytest.raises(rb.ConfigError, match="q_out"):
        rb.rope_paged_append(**ok, q_out=out.view(-1))


def test_current_device_and_launch_count(rb):
    s = make(1, 1, 8, 2, 128, 16, [40])
    ctx = rb.Context.get(0)
    n = ctx.launch_count()
    attend(rb, s, ctx=ctx)
    assert ctx.launch_count() > n and torch.cuda.current_device() == 0
