"""verify_draft at the corners of its definition: rows of NaN and -inf alone,
temperatures and logits at the ends of float32's range."""
import math

import pytest
import torch

from test_gpu_verify import check, inputs, run

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temp", [0.0, 0.7])
@pytest.mark.parametrize("V", [9, 1000, 70001])
def test_rows_of_nan_and_minus_infinity(rb, dtype, temp, V):
    """All of p lies on the lowest token of the maximum, NaN left out; on
    token 0 where nothing else is there. The same with and without a
    temperature."""
    a = inputs(6, 1, V, dtype=dtype, one_hot=True)
    a[4].fill_(temp)
    low = a[0][:, 0]
    low.fill_(-INF)
    low[0, 0] = NAN                     # token 1
    low[1, :7] = NAN                    # token 7
    low[2, :V - 1] = NAN                # the last
    low[3].fill_(NAN)                   # token 0
    low[4, 5] = NAN                     # token 0
    low[5, 0], low[5, 3] = NAN, INF     # token 3
    a[1][:, 0] = torch.tensor([1, 7, V - 1, 0, 0, 3], dtype=torch.int32)
    a[2].fill_(0.5)
    got = run(rb, a)
    assert got[1].tolist() == [1] * 6   # each draft is that token
    a[1][:, 0] = torch.tensor([0, 0, 0, 1, 1, 0], dtype=torch.int32)
    got = run(rb, a)
    assert got[1].tolist() == [0] * 6 and got[0][:, 0].tolist() == [1, 7, V - 1, 0, 0, 3]


# (temperature, scale of the logits): ends of the range, with logits of the
# temperature's size, so that several tokens are likely.
ENDS = [(1e31, 1e31), (3e38, 1e38), (1e-31, 1e-31), (1e-36, 3e-36), (2.0 ** -126, 2.0 ** -124), (1e30, 1e30),
        (2.0 ** -140, 2.0 ** -138), (2.0 ** -149, 2.0 ** -143)]


@pytest.mark.parametrize("temp,scale", ENDS)
def test_ends_of_the_range(rb, temp, scale):
    for V in (500, 20001):
        a = inputs(12, 3, V, seed=2)
        grid = torch.round(a[0].clamp_(-3, 3) * 64) / 64  # as exact after scaling by a number near a power of two
        power = 2.0 ** round(math.log2(scale))
        a[0] = grid * power
        assert torch.isfinite(a[0]).all()
        a[4].fill_(temp)
        want = check(rb, a)
        b = torch.arange(12)
        assert (want[0][b, want[1].long()].long() != a[0][b, want[1].long()].argmax(-1)).any()
