"""Draws at the ends of what counts: tokens far below the largest that are still kept, infinity beside the largest finite logit of a
type, logits far from zero. Against the definition in 64 bits, as in test_gpu_sampling.py."""

import math

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import ops
from tests.test_gpu_sampling import DEV, MOST, _check, _want

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


def _most(dtype):
    return torch.finfo(dtype).max


def _check_by_logit(x, u, t, k=None, p=None, m=None):
    """The definition with the tokens ordered by logit, which orders them by probability: below a logit of 3.4e38 the differences of
    all others are lost in 64 bits (whose step there is 2^75), and with them the order of what _want subtracts."""
    per = lambda v, d=torch.float32: None if v is None else torch.full((x.shape[0],), v, device=DEV, dtype=d)  # noqa: E731
    heat, share, least = per(t), per(p), per(m)
    tokens, logprobs = ops.sample_tokens(x, u, heat, per(k, torch.int32), share, least, return_logprobs=True)
    for r, row in enumerate(x.float().cpu().numpy().astype(np.float64)):
        row = np.where(np.isnan(row), -np.inf, np.minimum(row, MOST))
        if t == 0.0:
            assert tokens[r] == int(np.argmax(row)) and logprobs[r] == 0.0
            continue
        below, heat64 = row - row.max(), heat[r].item()
        mass = np.where(below >= -40.0 * heat64, np.exp(np.maximum(below, -1e300) / heat64), 0.0)
        order = np.argsort(-row, kind="stable")
        order = order[mass[order] > 0][:k]
        if p is not None:
            w = mass[order]
            order = order[: max(1, int(np.sum(np.cumsum(w) - w < share[r].item() * w.sum() * (1 - 1e-12))))]
        if m is not None:
            order = order[below[order] >= heat64 * math.log(least[r].item())]
        kept = np.zeros_like(mass)
        kept[order] = mass[order]
        upto = np.cumsum(kept)
        want = int(np.argmax(upto > u[r].item() * upto[-1] * (1 + 1e-12)))
        lp = math.log(mass[want] / upto[-1])
        assert tokens[r] == want, (r, t, k, p, m)
        # one rounding to fp32, masses good to 2^-40 (|x| / T of all that can be drawn beside each other are below 12 here)
        assert abs(logprobs[r].item() - lp) <= abs(lp) * 2.0 ** -24 + 2.0 ** -39
    return tokens


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [50, 30000])
def test_infinity_is_above_every_finite_logit(dtype, vocab):
    """+inf counts as the largest finite number of float32, which of 16-bit logits none else is."""
    print(f"sample: infinity beside the largest finite logit, {dtype} {vocab}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn(6, vocab, generator=g, device=DEV).to(dtype)
    x[:, 3] = _most(dtype)
    x[:, 7] = float("inf")
    x[1, 9] = x[1, vocab - 1] = float("inf")
    x[2, 11:40] = _most(dtype)
    x[3] = float("-inf")
    x[3, 5] = x[3, 7] = float("inf")
    x[4, 20] = float("nan")
    u = torch.rand(6, generator=g, device=DEV)
    assert ops.sample_tokens(x, u, torch.zeros(6, device=DEV)).tolist() == [7, 7, 7, 5, 7, 7]
    assert x[:4].float().argmax(-1).tolist() == [7, 7, 7, 5]
    # (at these the largest finite logit of bf16, and then all others, are near enough to be drawn)
    for t in (0.0, 1.0, 1e-3, 3e37, 3e38):
        for k, p, m in ((None, None, None), (1, None, None), (2, None, None), (3, 0.9, None), (None, 0.5, None), (None, None, 0.5),
                        (40, 0.95, 0.01)):
            _check_by_logit(x, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("many", [100, 3000, 9000])
def test_many_infinities(dtype, many):
    """More of them than a slice lists, and than a row's list takes, the largest finite logit between them."""
    print(f"sample: {many} infinities, {dtype}", flush=True)
    x = torch.zeros(5, 40000, device=DEV, dtype=dtype)
    x[:, 2:4 * many:2] = _most(dtype)
    x[:, 1:4 * many:4] = float("inf")
    u = torch.tensor([0.0, 0.25, 0.5, 0.999, 1 - 2.0 ** -24], device=DEV)
    for k, p, m in ((None, None, None), (many // 2, None, None), (many + 50, None, None), (None, 0.3, None), (many, 0.6, 0.5)):
        got = _check_by_logit(x, u, 1.0, k, p, m)
        if k is None or k <= many:
            assert (got % 4 == 1).all()
    _check_by_logit(x, u, 3e37, 2 * many)


@pytest.mark.parametrize("offset", [-3e7, 1e6, 2e5])
def test_logits_far_from_zero(offset):
    """x / T is rounded to 64 bits before the row's largest is subtracted: 2^-53 |x| / T of it for each, twice where a token is set
    against the rest, beside what draws near zero are good to."""
    print(f"sample: offset {offset}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(17)
    x = 4 * torch.randn(40, 30000, generator=g, device=DEV) + offset
    u = torch.rand(40, generator=g, device=DEV)
    for k, p, m in ((None, None, None), (50, 0.9, None), (None, 0.95, None), (None, None, 0.05)):
        per = lambda v, d=torch.float32: None if v is None else torch.full((40,), v, device=DEV, dtype=d)  # noqa: E731
        tokens, logprobs = ops.sample_tokens(x, u, None, per(k, torch.int32), per(p), per(m), return_logprobs=True)
        for r in range(40):
            p32 = 1.0 if p is None else per(p)[r].item()
            m32 = 0.0 if m is None else per(m)[r].item()
            want, lp = _want(x[r].cpu().numpy(), u[r].item(), 1.0, k or 0, p32, m32)
            assert tokens[r].item() == want
            assert abs(logprobs[r].item() - lp) <= abs(lp) * 2.0 ** -24 + 2.0 ** -39 + abs(offset) * 1.01 * 2.0 ** -51
