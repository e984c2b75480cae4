"""Logits of which nothing can be drawn, in a batch that the kernel samples: the request ends, its batch goes on, and no number out of
the vocabulary reaches the model."""

import pytest
import torch

from llama_lite_npu_amd import continuous_batching
from llama_lite_npu_amd.continuous_batching import BatchRequest
from tests.test_continuous_batching_backend import ChunkingExecutor, RecordingExecutor, _backend

EOS = 99


class Failing(ChunkingExecutor):
    """As RecordingExecutor, but a request's rows can be set to something else."""

    def __init__(self, device="cpu"):
        super().__init__()
        self.device, self.bad = device, {}

    def forward(self, input_ids, position_ids):
        rows = self.rows
        logits = super().forward(input_ids, position_ids).to(self.device)
        for i, req in enumerate(self.active):
            if req in self.bad:
                logits[(0, rows[i]) if rows is not None else (i, -1)] = self.bad[req]
        return logits

    def activate_paged_packed_prefill_batch(self, *a):
        return tuple(x.to(self.device) for x in super().activate_paged_packed_prefill_batch(*a))


def _plain_draw(logits, uniforms, temperature, top_k, top_p, min_p):
    clean = torch.where(logits.isnan(), float("-inf"), logits.float())
    return torch.where(clean.amax(-1) > float("-inf"), clean.argmax(-1), -1)


def _requests():
    return [BatchRequest("a", [1, 2], 4, 0.5, 1.0, top_k=3), BatchRequest("b", [3], 4, 0.0, 1.0), BatchRequest("c", [4, 5], 4, 0.0, 1.0)]


def _through(ex):
    """Prefill and three steps; request b has no token at the first of them or at the second step."""
    nothing = torch.full((128,), float("nan"))
    for when in ("prefill", "decode"):
        ex.__init__(ex.device)
        be, reqs = _backend(ex), _requests()
        if when == "prefill":
            ex.bad = {1: nothing}
        first = be.prefill(reqs)
        assert first == ([40, EOS, 42] if when == "prefill" else [40, 41, 42])
        assert [r.failed for r in reqs] == [False, when == "prefill", False]
        stored = [args[1] for args in ex.named("store")]
        assert stored == ([2] if when == "prefill" else [1, 2])               # greedy requests' first tokens, if there are any
        ex.bad = {1: torch.full((128,), float("-inf"))}
        assert be.decode(reqs) == [40, EOS, 42] and [r.failed for r in reqs] == [False, True, False]
        ex.bad = {}
        assert be.decode(reqs) == [40, 41, 42]                                # (a scheduler that does not end it may go on)
        assert be.decode([reqs[2], reqs[0]]) == [42, 40]
        for ids, _ in ex.forwards:
            assert ids.min() >= 0 and ids.max() < 128
        assert ex.forwards[2][0].flatten().tolist() == [40, EOS, 42]


def test_a_row_without_a_token_ends_its_request(monkeypatch, caplog):
    monkeypatch.setattr(continuous_batching.ops, "sample_tokens", _plain_draw)
    _through(Failing())
    assert "'b'" in caplog.text and "'a'" not in caplog.text


@pytest.mark.gpu
def test_a_row_without_a_token_ends_its_request_on_the_gpu():
    print("backend: rows without a token", flush=True)
    _through(Failing("cuda:0"))


def test_tokens_that_stay_on_the_device_are_in_range(monkeypatch):
    """Where nothing is read back nothing can be reported, but the next forward gets a token all the same."""
    monkeypatch.setattr(continuous_batching.ops, "sample_tokens", _plain_draw)
    ex = Failing()
    be, reqs = _backend(ex, return_host_tokens=False), _requests()
    ex.bad = {1: torch.full((128,), float("nan"))}
    assert be.prefill(reqs) == [] and be.decode(reqs) == [] and be.decode(reqs) == []
    assert [f[0].flatten().tolist() for f in ex.forwards[1:]] == [[40, EOS, 42], [40, EOS, 42]]


def test_chunked_prefill_and_replay(monkeypatch):
    monkeypatch.setattr(continuous_batching.ops, "sample_tokens", _plain_draw)
    for cls in (ChunkingExecutor, RecordingExecutor):
        made = type("Made", (Failing, cls), {})()
        if cls is RecordingExecutor:
            made.max_prefill_tokens = 1                                       # too long for one forward: token by token
        be, reqs = _backend(made), _requests()
        made.bad = {0: torch.full((128,), float("nan"))}
        if cls is ChunkingExecutor:
            got = [None] * 3
            while None in got:
                left = [i for i, t in enumerate(got) if t is None]
                for i, t in zip(left, be.prefill_chunk([reqs[i] for i in left], 1)):
                    got[i] = t
        else:
            got = be.prefill(reqs)
        assert got[0] == EOS and reqs[0].failed and not reqs[1].failed and not reqs[2].failed


def test_a_batch_without_filters_is_read_as_before(monkeypatch):
    """No launch and no look at the tokens beside what was there."""
    ex = RecordingExecutor()
    be, reqs = _backend(ex), [BatchRequest(n, [1], 4, 0.0, 1.0) for n in "ab"]
    given = torch.tensor([5, 6])
    be._sampler = lambda logits, **kw: given
    be.prefill(reqs)
    be.decode(reqs)
    assert be._step_tokens is given
