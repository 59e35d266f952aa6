"""verify_draft at the corners of its definition: rows of NaN and -inf alone."""
import pytest
import torch

from test_gpu_verify import inputs, run

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
