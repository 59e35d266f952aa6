"""verify_draft against a plain 64-bit implementation on the CPU. Results are
whole numbers and have to be equal: p, its sums and the comparisons are
64-bit on both sides, so they could differ only where a border lies within
about 1e-14 of the number compared with it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def distribution(row, temp):
    """p of one row of logits (float64)."""
    clean = torch.where(torch.isnan(row), torch.tensor(-INF, dtype=torch.float64), row)
    top = int((clean == clean.max()).nonzero()[0])
    if not temp > 0 or torch.isnan(row).any() or not math.isfinite(float(clean.max())):
        p = torch.zeros_like(row)
        p[top] = 1.0
        return p
    e = torch.exp((row - row.max()) / temp)
    return e / e.sum()


def reference(logits, drafts, accept_u, sample_u, temps, probs):
    B, n1, V = logits.shape
    n = n1 - 1
    tokens, accepted = torch.full((B, n1), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        a = 0
        while True:
            p = distribution(logits[b, a].double(), float(temps[b]))
            x = int(drafts[b, a]) if a < n else -1
            if not 0 <= x < V:
                rest = p
                break
            q = probs[b, a].double() if probs is not None else torch.nn.functional.one_hot(
                torch.tensor(x), V).double()
            if not float(accept_u[b, a].double() * q[x]) < float(p[x]):
                rest = (p - q).clamp(min=0)
                if not float(rest.sum()) > 0:
                    rest = p
                break
            tokens[b, a] = x
            a += 1
        c = rest.cumsum(0)
        hit = ((c > sample_u[b].double() * c[-1]) & (rest > 0)).nonzero()
        tokens[b, a] = int(hit[0]) if len(hit) else int(rest.nonzero()[-1])
        accepted[b] = a
    return tokens, accepted


def inputs(B, n, V, seed=0, dtype=torch.float32, one_hot=False, scale=2.5, noise=0.7):
    g = torch.Generator().manual_seed(seed * 7919 + B * 131 + n * 17 + V)
    logits = (torch.randn(B, n + 1, V, generator=g) * scale).to(dtype)
    probs = torch.softmax(logits[:, :n].float() + torch.randn(B, n, V, generator=g) * noise, -1)
    drafts = (torch.multinomial(probs.reshape(-1, V), 1, generator=g).view(B, n).to(torch.int32) if n and B
              else torch.zeros(B, n, dtype=torch.int32))
    return [logits, drafts, torch.rand(B, n, generator=g), torch.rand(B, generator=g),
            torch.full((B,), 0.9), None if one_hot else probs]


def run(rb, a):
    d = [x.cuda() if x is not None else None for x in a]
    t, c = rb.verify_draft(d[0], d[1], d[2], d[3], temperature=d[4], draft_probs=d[5])
    return t.cpu(), c.cpu()


def check(rb, a):
    got, want = run(rb, a), reference(*a)
    assert torch.equal(got[1], want[1]), (got[1], want[1])
    assert torch.equal(got[0], want[0])
    return want


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("one_hot", [False, True])
@pytest.mark.parametrize("B,n,V", [(1, 4, 32000), (5, 3, 1001), (33, 8, 257), (2, 1, 1), (3, 2, 2), (1, 0, 5000),
                                   (4, 0, 33), (2, 255, 40), (2, 3, 150001), (200, 2, 130)])
def test_against_64_bits(rb, B, n, V, dtype, one_hot):
    for seed in range(4):
        a = inputs(B, n, V, seed, dtype, one_hot, noise=0.05 if seed == 3 else 0.7)
        if seed == 1:
            a[4] = torch.tensor([0.0, 0.3, 1.0, 2.0, -1.0])[torch.arange(B) % 5]
        check(rb, a)


def test_all_accepted_and_all_rejected(rb):
    a = inputs(6, 5, 3001, noise=0.0)
    a[2].zero_()
    assert (check(rb, a)[1] == 5).all()      # u = 0
    a[5] = torch.softmax(a[0][:, :5].float() / 0.9, -1)
    a[2] = torch.full_like(a[2], 1.0 - 2.0 ** -24)
    a[5][..., :] *= 2.0                       # u q > p everywhere
    assert (check(rb, a)[1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_any_place_and_extreme_temperatures(rb, dtype):
    """Logits that begin at any element, and temperatures from the smallest
    number to infinity (all weights alike) and NaN (greedy)."""
    B, n, V = 7, 2, 1003
    for shift in range(4):
        a = inputs(B, n, V, seed=shift, dtype=dtype)
        a[4] = torch.tensor([1e-45, 1e-10, 1e-2, 1e6, 3e38, INF, NAN])
        a[0][:, :, 5] = -INF
        # An infinite temperature as the number it tends to: finite logits alike.
        flat = [x.clone() for x in a]
        flat[0][5][torch.isfinite(flat[0][5])] = 0.0
        flat[4][5] = 1.0
        want = reference(*flat)
        d = [x.cuda() for x in a]
        room = torch.empty(d[0].numel() + 8, dtype=dtype, device="cuda")
        place = room[shift:shift + d[0].numel()].view(B, n + 1, V).copy_(d[0])
        got = rb.verify_draft(place, d[1], d[2], d[3], temperature=d[4], draft_probs=d[5])
        assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_draft_ends_early(rb):
    a = inputs(6, 4, 500)
    a[2].zero_()
    for b, (at, bad) in enumerate([(0, -1), (1, 500), (2, 2**31 - 1), (3, -2**31)]):
        a[1][b, at] = bad
    assert check(rb, a)[1].tolist() == [0, 1, 2, 3, 4, 4]


def test_accept_borders(rb):
    """Numbers one float32 step to either side of p / q."""
    B, n, V = 64, 1, 4001
    a = inputs(B, n, V, noise=1.0)
    p = torch.stack([distribution(a[0][b, 0].double(), float(a[4][b])) for b in range(B)])
    x = a[1].long()
    # Drafts with p < q, so that the border lies below 1.
    for b in range(B):
        ok = (p[b] < 0.98 * a[5][b, 0].double()) & (p[b] > 0)
        x[b, 0] = int(torch.where(ok, a[5][b, 0], torch.tensor(0.0)).argmax())
    a[1] = x.to(torch.int32)
    ratio = p.gather(1, x) / a[5][:, 0].double().gather(1, x)
    near = ratio.float()
    for step in (torch.zeros_like(near), torch.ones_like(near)):
        a[2] = torch.nextafter(near, step)
        want = check(rb, a)[1]
    assert (want == 0).all()


def test_sample_borders_and_ends(rb):
    """sample_u of 0 and of the largest float32 below 1, weights of zero at
    both ends, and borders exactly hit."""
    V = 1000
    a = inputs(4, 0, V)
    a[0][:, :, :7] = -INF
    a[0][:, :, -9:] = -INF
    a[3] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 0.5, 0.25])
    got = check(rb, a)[0][:, 0]
    assert got[0] == 7 and got[1] <= V - 10
    # Four equal weights: 0.25 and 0.5 lie on borders and go to the token above.
    b = inputs(5, 0, V)
    b[0].fill_(-INF)
    b[0][:, :, 100:104] = 3.0
    b[3] = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.2499])
    assert check(rb, b)[0][:, 0].tolist() == [100, 101, 102, 103, 100]
    # Numbers outside [0, 1) still give a token with weight.
    for u, want in ((2.0, 103), (-1.0, 100), (NAN, 103)):
        b[3].fill_(u)
        assert run(rb, b)[0][:, 0].tolist() == [want] * 5


def test_undefined_rows_are_greedy(rb):
    V = 300
    a = inputs(6, 1, V, one_hot=True)
    a[0][0, 0, 17] = NAN
    a[0][1, 0, 250] = INF
    a[0][2, 0] = -INF
    a[0][3, 0] = NAN
    a[0][4, 0, 5] = INF
    a[0][4, 0, 3] = INF
    a[0][5, 0, 40:] = -INF
    a[2].fill_(0.5)
    check(rb, a)
    a[1][:, 0] = torch.tensor([0, 250, 0, 0, 3, 1], dtype=torch.int32)
    want = check(rb, a)
    assert want[1][1:5].tolist() == [1, 1, 1, 1]


def test_greedy_ties_and_residual(rb):
    """Temperature 0: the lowest index of the maximum; a rejected draft is
    replaced by it; where q covers p entirely, p itself is sampled."""
    a = inputs(3, 2, 64)
    a[0].clamp_(max=1.0)
    a[4].zero_()
    check(rb, a)
    V = 8
    one = torch.zeros(1, 2, V)
    one[0, 0, 3] = 50.0
    b = [one, torch.tensor([[5]], dtype=torch.int32), torch.tensor([[0.5]]), torch.tensor([0.3]), torch.zeros(1),
         torch.ones(1, 1, V)]
    t, c = check(rb, b)
    assert c.tolist() == [0] and t.tolist() == [[3, -1]]


def test_distribution_of_the_result(rb):
    """Over many numbers, the first token is distributed as p whatever q the
    draft came from: chi-square over 6 tokens, 40000 sequences. The statistic
    has 5 degrees of freedom and exceeds 40 with probability 1.5e-7."""
    B, V = 40000, 6
    g = torch.Generator().manual_seed(11)
    logits, other = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p, q = torch.softmax(logits, 0), torch.softmax(other, 0)
    drafts = torch.multinomial(q.expand(B, V), 1, generator=g).to(torch.int32)
    a = [logits.expand(B, 2, V).contiguous(), drafts, torch.rand(B, 1, generator=g), torch.rand(B, generator=g),
         torch.ones(B), q.expand(B, 1, V).contiguous()]
    first = run(rb, a)[0][:, 0]
    count = torch.bincount(first.long(), minlength=V).double()
    chi = ((count - B * p.double()) ** 2 / (B * p.double())).sum()
    assert chi < 40, chi


def test_streams_and_graph(rb):
    a, b = inputs(3, 4, 32000), inputs(40, 2, 5000, seed=2)
    wa, wb = reference(*a), reference(*b)
    da, db = ([x.cuda() for x in y] for y in (a, b))
    call = lambda d: rb.verify_draft(d[0], d[1], d[2], d[3], temperature=d[4], draft_probs=d[5])
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        x = [call(da) for _ in range(5)]
    with torch.cuda.stream(s2):
        y = [call(db) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(o[0].cpu(), wa[0]) for o in x) and all(torch.equal(o[0].cpu(), wb[0]) for o in y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call(da)
    da[3].fill_(0.1)
    a[3].fill_(0.1)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out[0].cpu(), reference(*a)[0])


@pytest.mark.parametrize("B,V", [(1, 200003), (1, 70000), (2, 1023), (7, 128001), (64, 32768), (70, 128001)])
def test_every_border_is_found(rb, B, V):
    """Uniform logits: every weight is exactly 1, so that sample_u = (k + 1/2)
    / V takes token k; its rounding moves the target by at most V * 2^-25 <
    0.01. Numbers of 1 and more, or none, take the last token. The same for
    what a rejected draft leaves: the second half of the vocabulary."""
    g = torch.Generator().manual_seed(V)
    k = torch.randint(0, V, (B,), generator=g)
    k[0] = V - 1
    u = ((k.double() + 0.5) / V).float()
    if B > 4:
        u[1], u[2], u[3], k[1:4] = 1.0, NAN, INF, V - 1
    logits = torch.zeros(B, 1, V, device="cuda", dtype=torch.bfloat16)
    t, _ = rb.verify_draft(logits, None, None, u.cuda(), 0.9)
    assert t[:, 0].tolist() == k.tolist()

    h = V // 2
    q = torch.zeros(B, 1, V, device="cuda")
    q[:, :, :h] = 1.0 / h  # above 1 / V: rejected with accept_u of 0.9, and nothing of it is left
    k = h + torch.randint(0, V - h, (B,), generator=g)
    k[0] = h
    u = ((k.double() - h + 0.5) / (V - h)).float()
    d = torch.randint(0, h, (B, 1), generator=g, dtype=torch.int32)
    t, c = rb.verify_draft(torch.zeros(B, 2, V, device="cuda"), d.cuda(), torch.full((B, 1), 0.9, device="cuda"), u.cuda(),
                           0.9, draft_probs=q)
    assert t[:, 0].tolist() == k.tolist() and c.tolist() == [0] * B and t[:, 1].tolist() == [-1] * B


def test_batch_as_its_sequences(rb):
    """A batch whose verdicts are found in a launch of their own gives what
    each sequence gives alone."""
    B, n, V = 60, 2, 128001
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn(B, n + 1, V, device="cuda", generator=g) * 3
    q = torch.softmax(logits[:, :n] + 0.7 * torch.randn(B, n, V, device="cuda", generator=g), -1)
    d = torch.multinomial(q.view(B * n, V), 1, generator=g).view(B, n).int()
    d[5, 1], d[6, 0] = -1, V
    au, su = (torch.rand(*x, device="cuda", generator=g) for x in ((B, n), (B,)))
    temp = torch.full((B,), 1.0, device="cuda")
    temp[7] = 0.0
    logits[8, 0, 77], logits[9, 1, 5] = NAN, INF
    t, c = rb.verify_draft(logits, d, au, su, temp, q)
    assert len(set(c.tolist())) == n + 1
    for b in range(B):
        s = slice(b, b + 1)
        tb, cb = rb.verify_draft(logits[s], d[s], au[s], su[s], temp[s], q[s])
        assert torch.equal(tb, t[s]) and torch.equal(cb, c[s]), b


def test_refusals(rb):
    d = [x.cuda() if x is not None else None for x in inputs(2, 3, 50)]
    ok = dict(logits=d[0], draft_tokens=d[1], accept_u=d[2], sample_u=d[3], temperature=d[4], draft_probs=d[5])
    rb.verify_draft(**ok)
    rb.verify_draft(**dict(ok, temperature=0.7))
    for bad in (dict(logits=d[0].half()), dict(logits=d[0][:, :, ::2]), dict(logits=d[0][0]),
                dict(draft_tokens=d[1].long()), dict(draft_tokens=d[1][:, :2]), dict(draft_tokens=None),
                dict(accept_u=None), dict(accept_u=d[2].double()), dict(sample_u=d[3][:1]),
                dict(temperature=d[4].double()), dict(draft_probs=d[5][:, :2]), dict(draft_probs=d[5].cpu())):
        with pytest.raises(rb.ConfigError):
            rb.verify_draft(**dict(ok, **bad))
    t, c = rb.verify_draft(d[0][:0], d[1][:0], d[2][:0], d[3][:0], temperature=d[4][:0], draft_probs=d[5][:0])
    assert t.shape == (0, 4) and c.shape == (0,)
