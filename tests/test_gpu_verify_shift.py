"""verify_draft where only differences of logits count: rows far below zero,
runs masked with a finite number, low temperatures. Compared with the plain
64-bit implementation, and a shifted row with the row itself; the tokens have
to be equal. Every input is built from exact values, so that a shift is exact
in the logits' type."""
import pytest
import torch

from test_gpu_verify import check, inputs, run

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


def on_grid(a, step, dtype, to=0.0):
    """The inputs `a` with their logits rounded to multiples of `step`, shifted
    by `to`; the rounding of dtype changes nothing."""
    grid = torch.round(a[0].double() / step) * step + to
    logits = grid.to(dtype)
    assert torch.equal(logits.double(), grid)
    return [logits] + list(a[1:])


def not_greedy(a, want):
    """Some sequence's sampled token is not the most likely one of its row, so
    that an answer of the maximum alone would be seen."""
    b = torch.arange(a[0].shape[0])
    row, at = a[0][b, want[1].long()].float(), want[1].long()
    assert (want[0][b, at].long() != row.argmax(-1)).any()


# (shift, step of the logits, temperature): -128 and -9984 with steps that
# bf16 holds there too.
SHIFTS = [(torch.float32, -100.0, 2.0 ** -6, 0.9), (torch.float32, -10000.0, 2.0 ** -6, 1.0),
          (torch.float32, -40.0, 2.0 ** -6, 0.3), (torch.float32, -1e6, 0.25, 1.0),
          (torch.bfloat16, -128.0, 1.0, 0.9), (torch.bfloat16, -32.0, 0.25, 0.25),
          (torch.bfloat16, -9984.0, 64.0, 60.0), (torch.float32, 10000.0, 2.0 ** -6, 1.0)]


@pytest.mark.parametrize("dtype,shift,step,temp", SHIFTS)
@pytest.mark.parametrize("B,n,V", [(6, 3, 1001), (3, 2, 40003), (8, 0, 257), (2, 1, 150001)])
@pytest.mark.parametrize("one_hot", [False, True])
def test_shift(rb, B, n, V, dtype, shift, step, temp, one_hot):
    a = inputs(B, n, V, seed=3, one_hot=one_hot, scale=2.5 if step < 1 else 2.5 * step)
    a[0].clamp_(-11 * max(step, 1.0), 11 * max(step, 1.0))
    a[4].fill_(temp)
    plain, moved = on_grid(a, step, dtype), on_grid(a, step, dtype, shift)
    want = check(rb, plain)
    not_greedy(plain, want)
    got = run(rb, moved)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check(rb, moved)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", [-1e4, -1e9, None])
@pytest.mark.parametrize("where", ["start", "middle", "end", "all but one", "all but some"])
def test_masked_by_a_number(rb, dtype, low, where):
    """Runs of the vocabulary masked by a finite number: they have no weight,
    and the others keep theirs."""
    low = torch.finfo(dtype).min if low is None else low
    for V in (1003, 33001):
        B, n = 6, 2
        a = inputs(B, n, V, seed=1, dtype=dtype)
        a[4] = torch.tensor([0.2, 0.9, 1.0, 1.3, 0.05, 0.9])
        some = torch.tensor([3, 64, V // 3, V // 2 + 1, V - 2])
        if where == "start":
            a[0][..., :512] = low
        elif where == "middle":
            a[0][..., V // 3:V // 3 + 400] = low
        elif where == "end":
            a[0][..., -600:] = low
        elif where == "all but one":
            one = a[0][..., V // 2].clone()
            a[0].fill_(low)
            a[0][..., V // 2] = one
        else:
            live = (torch.arange(5) % 3 * 0.0625 - 20.0).to(dtype)  # as likely as one another, below zero
            a[0].fill_(low)
            a[0][..., some] = live
        want = check(rb, a)
        if where == "all but one":
            assert (want[0][torch.arange(B), want[1].long()] == V // 2).all()
        else:
            not_greedy(a, want)
        # The same with infinities in the place of the number.
        hard = [torch.where(a[0] == low, torch.tensor(-float("inf"), dtype=dtype), a[0])] + a[1:]
        got = run(rb, hard)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temp", [0.05, 0.1, 0.3])
def test_cold_rows_keep_their_spread(rb, dtype, temp):
    """Low temperatures over logits that lie close together: several tokens
    have weight wherever the logits lie."""
    for V in (700, 32000):
        for to in (-16.0, -60.0, 8.0):
            a = inputs(8, 2, V, seed=5, scale=2.0 * temp)
            a[0].clamp_(-1.9, 1.9)
            a[4].fill_(temp)
            a = on_grid(a, 2.0 ** -8 if dtype is torch.float32 else 0.25, dtype, to)
            not_greedy(a, check(rb, a))


@pytest.mark.parametrize("temp", [0.2, 0.9, 1.0])
def test_log_probabilities(rb, temp):
    """log_softmax of the logits in their place: its maximum is below zero
    throughout."""
    for V in (513, 32001):
        a = inputs(6, 3, V, seed=9)
        a[0] = torch.log_softmax(a[0] * 0.3, -1) - 10.0
        a[4].fill_(temp)
        not_greedy(a, check(rb, a))
