"""Drawn tokens against the definition, evaluated per row in 64 bits on the CPU: the tokens are equal."""

import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import continuous_batching, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
MOST = float(np.finfo(np.float32).max)


def _want(x, u, t, k, p, m):
    """One row: (token, logprob)."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, MOST))
    if x.max() == -np.inf:
        return -1, -np.inf
    if not t > 0:
        return int(np.argmax(x)), 0.0
    below = x - x.max()
    mass = np.where(below >= -40.0 * t, np.exp(np.maximum(below, -1e300) / t), 0.0)
    order = np.argsort(-below, kind="stable")
    order = order[mass[order] > 0]
    if k > 0:
        order = order[:k]
    if p < 1:
        w = mass[order]
        # a run that reaches its share exactly has reached it, whatever its sum's last bits are
        order = order[: max(1, int(np.sum(np.cumsum(w) - w < p * w.sum() * (1 - 1e-12))))]
    if m > 0:
        order = order[below[order] >= min(0.0, t * math.log(m))]
    kept = np.zeros_like(mass)
    kept[order] = mass[order]
    upto = np.cumsum(kept)
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    token = int(np.argmax(upto > u * upto[-1] * (1 + 1e-12)))
    return token, math.log(mass[token] / upto[-1])


def _check(logits, u, t=None, k=None, p=None, m=None):
    b = logits.shape[0]
    per = lambda x, dtype: None if x is None else torch.as_tensor(x, dtype=dtype, device=DEV).expand(b).contiguous()  # noqa: E731
    u = per(u, torch.float32)
    t, k, p, m = per(t, torch.float32), per(k, torch.int32), per(p, torch.float32), per(m, torch.float32)
    tokens, logprobs = ops.sample_tokens(logits, u, t, k, p, m, return_logprobs=True)
    assert tokens.dtype is torch.int64
    rows, got, got_lp = logits.float().cpu().numpy(), tokens.cpu().tolist(), logprobs.cpu().tolist()
    at = lambda x, r, d: d if x is None else x[r].item()  # noqa: E731
    for r in range(b):
        want, lp = _want(rows[r], u[r].item(), at(t, r, 1.0), at(k, r, 0), at(p, r, 1.0), at(m, r, 0.0))
        assert got[r] == want, (r, got[r], want, got_lp[r], lp)
        # one rounding to fp32 behind masses good to 2^-41
        assert got_lp[r] == lp or abs(got_lp[r] - lp) <= abs(lp) * 2.0 ** -24 + 2e-11, (r, got_lp[r], lp)
    return tokens


def _logits(seed, b, v, dtype=torch.float32, spread=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = spread * torch.randn(b, v, generator=g, device=DEV)
    x.scatter_add_(1, torch.randint(0, v, (b, 5), generator=g, device=DEV), 8 + torch.randn(b, 5, generator=g, device=DEV))
    return x.to(dtype), torch.rand(b, generator=g, device=DEV)


FILTERS = [(None, None, None), (50, None, None), (None, 0.9, None), (None, None, 0.05), (40, 0.95, None), (40, 0.8, 0.02),
           (None, 0.97, 0.001), (20000, 0.99, None), (3, None, 0.3)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [1, 2, 7, 1000, 8191, 8193, 40001, 151936])
def test_against_the_definition(dtype, v):
    print(f"sample {dtype} vocab={v}", flush=True)
    for i, (k, p, m) in enumerate(FILTERS):
        logits, u = _logits(v + i, 5, v, dtype)
        _check(logits, u, [0.7, 1.0, 1.6, 0.3, 0.0], k, p, m)


@pytest.mark.parametrize("spread,t", [(0.0, 1.0), (0.02, 1.0), (0.5, 3.0), (20.0, 1.0), (2.0, 0.01), (2.0, 100.0)])
def test_flat_and_steep_rows(spread, t):
    """All tokens in one bin (more than a workgroup lists), in a few, in many, and a single one."""
    print(f"sample spread={spread} T={t}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = (spread * torch.randn(4, 60000, generator=g, device=DEV) + 3.0)
    for dtype in (torch.float32, torch.bfloat16):
        for k, p, m in FILTERS + [(30000, 0.5, None), (59999, None, 1e-4), (None, 0.5, 0.5)]:
            _check(logits.to(dtype), torch.rand(4, generator=g, device=DEV), t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("first", [3, 100, 7000])
def test_top_k_that_ends_between_two_distant_logits(dtype, first):
    """The first top_k are apart from all others: what lies below them is not drawn, whether a slice's list holds them or not."""
    print(f"sample: top_k ends with a bin, {dtype} {first}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(90)
    x = 3 + 3 * torch.rand(64, 9001, generator=g, device=DEV)
    x[:, torch.randperm(9001, generator=g, device=DEV)[:first]] = 7.0
    u = (torch.arange(64, device=DEV) + 0.5) / 64
    for k in (first, first - 1, first + 1):
        _check(x.to(dtype), u, k=k)
        _check(x.to(dtype), u, k=k, p=0.99, m=0.2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spread", [0.01, 2.0])
def test_one_kept_token_has_probability_1(dtype, spread):
    """Its logarithm is 0 and nothing beside it, by each filter, from the lists and from the row."""
    print(f"sample: one kept {dtype} {spread}", flush=True)
    x, u = _logits(80, 40, 50000, dtype, spread)
    x[:, 77] = x.max(1).values + x.abs().max() * 2.0 ** -6
    t, full = torch.linspace(0.3, 2.0, 40, device=DEV), lambda v, d=torch.float32: torch.full((40,), v, device=DEV, dtype=d)  # noqa: E731
    for filters in (dict(top_k=full(1, torch.int32)), dict(top_p=full(1e-6)), dict(min_p=full(1.0))):
        tokens, logprobs = ops.sample_tokens(x, u, t, **filters, return_logprobs=True)
        assert (tokens == 77).all() and (logprobs == 0).all(), (filters, logprobs)


def test_ties_go_to_the_lowest_index():
    print("sample: ties", flush=True)
    for v in (1000, 20000):
        flat = torch.full((6, v), -2.5, device=DEV, dtype=torch.float16)
        u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 1 - 2.0 ** -24], device=DEV)
        assert _check(flat, u).tolist() == [0, v // 4, v // 2, 3 * v // 4, 999 * v // 1000 - (0 if u[4] >= 0.999 else 1), v - 1]
        assert max(_check(flat, u, k=10).tolist()) == 9
        assert max(_check(flat, u, p=0.5).tolist()) == v // 2 - 1           # half of them is half of the mass
        assert _check(flat, u, m=1.0).tolist()[-1] == v - 1
        assert _check(flat, u, 0.0).tolist() == [0] * 6
        two = flat.clone()
        two[:, [7, v - 3]] = 4.0
        assert set(_check(two, u, k=1).tolist()) == {7}
        assert set(_check(two, u, k=2).tolist()) == {7, v - 3}
        assert set(_check(two, u, 0.0).tolist()) == {7}
        assert set(_check(two, u, p=1e-30).tolist()) == {7}
        _check(two, u, k=v // 2)


def test_masked_rows():
    """-inf, the type's lowest value, NaN and +inf; rows with one token left, and with none."""
    print("sample: masks", flush=True)
    for dtype in (torch.float16, torch.bfloat16, torch.float32):
        for v in (500, 30000):
            x, u = _logits(9, 8, v, dtype)
            x[0] = float("-inf")
            x[1] = float("-inf")
            x[1, v - 2] = -60000.0
            x[2, ::2] = float("nan")
            x[3, 1::3] = torch.finfo(dtype).min
            x[4] = torch.finfo(dtype).min
            x[5, 11] = float("inf")
            x[5, 13] = float("inf")
            x[6] = float("nan")
            x[7, : v - 1] = float("-inf")
            for k, p, m in FILTERS:
                got = _check(x, u, 0.8, k, p, m).tolist()
                assert got[0] == got[6] == -1 and got[1] == v - 2 and got[2] % 2 == 1 and got[5] in (11, 13) and got[7] == v - 1
            assert _check(x, u, 0.0).tolist()[0] == -1


def test_the_two_zeros_are_one():
    x = torch.zeros(2, 100, device=DEV)
    x[:, :50] = -0.0
    assert _check(x, 0.0, k=1).tolist() == [0, 0] and _check(x, 0.99, k=60).tolist() == [59, 59]


def test_parameters_out_of_their_range():
    """Off, or the nearest that says something."""
    print("sample: parameters", flush=True)
    x, u = _logits(12, 4, 3000)
    plain = _check(x, u).tolist()
    nan = float("nan")
    assert _check(x, u, k=0).tolist() == plain and _check(x, u, k=-3).tolist() == plain and _check(x, u, k=2 ** 31 - 1).tolist() == plain
    for p in (1.0, 2.0):
        assert _check(x, u, p=p).tolist() == plain
    for m in (0.0, -1.0):
        assert _check(x, u, m=m).tolist() == plain
    greedy = x.argmax(-1).tolist()
    on = lambda y: torch.full((4,), y, device=DEV)  # noqa: E731
    assert ops.sample_tokens(x, u, None, None, on(nan), on(nan)).tolist() == plain
    assert ops.sample_tokens(x, u, on(nan)).tolist() == greedy and ops.sample_tokens(x, u, on(-1.0)).tolist() == greedy
    assert _check(x, u, p=0.0).tolist() == greedy and _check(x, u, p=-1.0).tolist() == greedy
    assert _check(x, u, m=1.0).tolist() == greedy and _check(x, u, m=7.0).tolist() == greedy
    assert ops.sample_tokens(x, on(nan)).tolist() == ops.sample_tokens(x, on(0.0)).tolist() == ops.sample_tokens(x, on(-3.0)).tolist()
    assert ops.sample_tokens(x, on(1.0)).tolist() == ops.sample_tokens(x, on(9.0)).tolist() == _check(x, 1 - 2.0 ** -24).tolist()
    for t in (1e-30, 1e-6, 1e30, 3e38, float("inf")):
        got = ops.sample_tokens(x, u, on(t)).tolist()
        if t < 1:
            assert got == greedy
        else:                                                   # all tokens alike
            assert got == [int(y * 3000) for y in u.tolist()]


def test_strides_and_alignment():
    """Rows of something wider, at any element's alignment."""
    print("sample: strides", flush=True)
    for dtype in (torch.float16, torch.float32):
        for lead in range(0, 9):
            wide, u = _logits(20 + lead, 5, 9100, dtype)
            wide[:, :lead] = wide[:, lead + 9001:] = 50.0               # what is not the row's does not count
            _check(wide[:, lead:lead + 9001], u, 1.1, 300, 0.9)
            _check(wide[:, lead:lead + 9001], u)


def test_a_large_batch():
    print("sample: large batch", flush=True)
    x, u = _logits(30, 700, 1500, torch.float16)
    _check(x, u, torch.linspace(0, 2, 700), torch.arange(700) % 90, torch.linspace(0.2, 1.1, 700), torch.linspace(-0.1, 0.3, 700))


def test_drawn_as_often_as_probable():
    """40 000 draws from one row: each token's count within 5.5 standard deviations (one failure in some 10^7 seeds over 100 tokens)."""
    print("sample: frequencies", flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    row = torch.randn(1, 100, generator=g, device=DEV)
    n = 40000
    got = ops.sample_tokens(row.expand(n, 100), torch.rand(n, generator=g, device=DEV))
    p = torch.softmax(row.double()[0], 0)
    count = torch.bincount(got, minlength=100).double()
    assert ((count - n * p).abs() <= 5.5 * (n * p * (1 - p)).sqrt() + 1).all()


def test_refusals():
    x, u = _logits(40, 3, 50)
    for call in (lambda: ops.sample_tokens(x.double(), u), lambda: ops.sample_tokens(x[0], u), lambda: ops.sample_tokens(x.t(), u[:1]),
                 lambda: ops.sample_tokens(x, u[:2]), lambda: ops.sample_tokens(x, u.double()), lambda: ops.sample_tokens(x, u.cpu()),
                 lambda: ops.sample_tokens(x, u, top_k=u), lambda: ops.sample_tokens(x, u, top_p=u[:1]),
                 lambda: ops.sample_tokens(x, None)):
        with pytest.raises((ValueError, AttributeError)):
            call()
    assert ops.sample_tokens(x[:0], u[:0]).shape == (0,)


def test_replayed_from_a_graph_and_on_two_streams():
    """Each call has a workspace of its own; three replays with new inputs, another stream's draws between them."""
    print("sample: graph, streams", flush=True)
    x, u = _logits(50, 9, 20000, torch.float16)
    y, w = _logits(51, 4, 30000)
    p = torch.full((9,), 0.9, device=DEV)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.sample_tokens(x, u, top_p=p)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            got = ops.sample_tokens(x, u, top_p=p)
    other = ops.sample_tokens(y, w)
    torch.cuda.synchronize()
    for i in range(3):
        a, b = _logits(60 + i, 9, 20000, torch.float16)
        x.copy_(a)
        u.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(ops.sample_tokens(y, w), other)
        torch.cuda.synchronize()
        assert torch.equal(got, _check(a, b, p=0.9)), i


def test_the_backend_draws_with_it():
    """Requests with filters or a seed: the kernel's tokens, the same for a seeded request whatever batch it is in."""
    print("sample: backend", flush=True)
    backend = object.__new__(continuous_batching.ContinuousBatchModelBackend)
    backend.executor, backend._sampler = SimpleNamespace(), continuous_batching.sample_next_token
    logits, _ = _logits(70, 3, 5000, torch.float16)
    make = lambda n, t, **kw: continuous_batching.BatchRequest(n, [1], 4, t, 0.9, **kw)  # noqa: E731
    seeded, greedy, other = make("a", 0.9, seed=5, top_k=30), make("b", 0.0), make("c", 1.2, min_p=0.2)
    got = backend._sample(logits[:, None], [seeded, greedy, other])
    again = backend._sample(logits[[1, 0]], [other, seeded])
    assert got.dtype is torch.int64 and got[0] == again[1] and got[1] == logits[1].argmax()
    assert logits[0, got[0]] >= logits[0].float().topk(30).values[-1]
