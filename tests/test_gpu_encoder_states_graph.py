"""Steps over an encoder's states captured into graphs: one plan a graph, whatever its layers, and none shared by two."""

import pytest
import torch

from llama_lite_npu_amd import ops
from llama_lite_npu_amd.attention import Attention
from llama_lite_npu_amd.executor import encoder_states
from llama_lite_npu_amd.executor.encoder_states import EncoderStates

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LAYERS, HQ, HKV, D, PAGE = 4, 32, 4, 128, 16


def _capture(run, stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        held = run()
    return graph, held


@pytest.mark.parametrize("eager_first", [False, True])
def test_a_graph_has_one_plan_for_its_layers(eager_first, monkeypatch):
    print(f"encoder states: a captured step of {LAYERS} layers, eager step first: {eager_first}", flush=True)
    made = []
    plan_of = ops.DecodePlan
    monkeypatch.setattr(encoder_states.ops, "DecodePlan", lambda *a, **k: made.append(plan_of(*a, **k)) or made[-1])
    g = torch.Generator(device=DEV).manual_seed(2)
    lengths = [(37 * i) % 1300 for i in range(300)]
    states, layer = EncoderStates(lengths, LAYERS, HKV, D, PAGE, device=DEV), Attention(HQ, HKV, D)
    total = sum(lengths)
    for index in range(LAYERS):
        states.store(index, *(torch.randn(total, HKV, D, generator=g, device=DEV).half() for _ in range(2)))
    q = torch.randn(300, HQ, D, generator=g, device=DEV).half()
    run = lambda: [layer.cross_forward(q, states, index) for index in range(LAYERS)]  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    if eager_first:
        with torch.cuda.stream(stream):
            run()
        torch.cuda.synchronize()
        assert len(made) == 1
    before = len(made)
    graphs = [_capture(run, stream) for _ in range(2)]
    assert len(made) - before == 2                                       # a graph's own
    assert all(plan.schedule == 0 for plan in made)                      # (the schedule that has a plan to make)
    rooms = [{x.data_ptr() for x in (plan.buffer, plan.workspace)} for plan in made[before:]]
    if not eager_first:
        assert not states._plans                                         # nothing that only a replay would fill is kept
    others = [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed in range(3):
        q.copy_(torch.randn(300, HQ, D, generator=g, device=DEV))
        torch.cuda.synchronize()
        for (graph, _), on in zip(graphs, others):                       # at once
            with torch.cuda.stream(on):
                graph.replay()
        torch.cuda.synchronize()
        got = [[x.clone() for x in held] for _, held in graphs]
        want = run()                                                     # (an eager plan, not a graph's)
        torch.cuda.synchronize()
        for kept in got:
            assert all(torch.equal(a, b) for a, b in zip(kept, want)), seed
    assert len(made) == 3 and not rooms[0] & rooms[1]
    # head counts have plans of their own, in a graph too
    few = Attention(HKV, HKV, D)
    two = _capture(lambda: (layer.cross_forward(q, states, 0), few.cross_forward(q[:, :HKV].contiguous(), states, 1),
                            layer.cross_forward(q, states, 2), few.cross_forward(q[:, :HKV].contiguous(), states, 3)), stream)
    assert len(made) == 5
    two[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(two[1][0], want[0]) and torch.equal(two[1][2], want[2])
    assert torch.equal(two[1][3], few.cross_forward(q[:, :HKV].contiguous(), states, 3))


def test_a_stream_that_captures_nothing_has_no_capture():
    stream = torch.cuda.Stream()
    assert ops.capture_id() is None
    seen = []
    x = torch.zeros(4, device=DEV)
    for _ in range(2):
        graph, _ = _capture(lambda: (x.add_(1), seen.append(ops.capture_id()), seen.append(ops.capture_id())), stream)
        graph.replay()
    torch.cuda.synchronize()
    assert None not in seen and seen[0] == seen[1] != seen[2] == seen[3] and ops.capture_id() is None
