"""Draws at the ends of what counts, against the definition in 64 bits as in test_gpu_sampling.py."""

import pytest
import torch

from tests.test_gpu_sampling import DEV, _check

pytestmark = pytest.mark.gpu

GAPS = [30.0, 31.0, 33.0, 35.0, 37.0, 39.0, 39.5, 40.0]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [1, 60, 100, 200, 1500, 6000])
def test_the_first_number_takes_the_first_kept_token(dtype, n):
    """With u = 0 the first token, by index, that is kept at all, however little of the mass it has: 30 to 40 temperatures below the
    largest, beside n tokens near it, which the slices' lists hold (ranked at once, or drawn by runs of indexes) or do not."""
    print(f"sample: u = 0, {n} near the largest, {dtype}", flush=True)
    vocab, b = 100000, len(GAPS)
    x = torch.full((b, vocab), float("-inf"), device=DEV)
    x[:, 5 + torch.arange(n, device=DEV) * ((vocab - 6) // n)] = -0.25
    x[:, 5] = 0.0
    x[:, 0] = -torch.tensor(GAPS, device=DEV)
    for t in (1.0, 0.5, 2.0):
        rows = (x * t).to(dtype)
        for filters in (dict(), dict(m=1e-18), dict(k=n + 1), dict(k=n + 1, m=1e-18)):
            assert _check(rows, 0.0, t, **filters).tolist() == [0] * b
        assert _check(rows, 2.0 ** -24, t).tolist() == [5] * b             # (which is past the masses of all of these)
    assert _check(x.to(dtype), 0.0, k=n).tolist() == [5] * b               # and without it
