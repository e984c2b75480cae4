"""Where the uniform numbers of a batch that the kernel samples come from."""

import random

import torch

from llama_lite_npu_amd import continuous_batching
from llama_lite_npu_amd.continuous_batching import BatchRequest, draw_tokens


def _numbers(monkeypatch, requests):
    seen = []
    monkeypatch.setattr(continuous_batching.ops, "sample_tokens", lambda rows, u, *a: seen.append(u) or rows[:, 0])
    draw_tokens(torch.zeros(len(requests), 8), requests)
    return seen[0]


def test_numbers_of_requests_without_a_seed_come_from_torch(monkeypatch):
    """As those of a batch without filters do: torch.manual_seed fixes them, and Python's generator is not touched."""
    make = lambda n, **kw: BatchRequest(n, [1], 4, 0.7, 0.9, **kw)  # noqa: E731
    for requests in ([make("a"), make("b", top_k=4)], [make("a"), make("s", seed=3), make("b", min_p=0.1)], [make("s", seed=3)]):
        torch.manual_seed(11)
        random.seed(1)
        state = random.getstate()
        first = _numbers(monkeypatch, requests)
        assert random.getstate() == state
        random.seed(2)
        torch.manual_seed(11)
        assert torch.equal(_numbers(monkeypatch, requests), first)
        torch.manual_seed(12)
        other = _numbers(monkeypatch, requests)
        for r, x, y in zip(requests, first.tolist(), other.tolist()):
            assert 0 <= x < 1 and (x == y) == (r.seed is not None)
    assert first.dtype is torch.float32 and first.is_contiguous()
