"""What the operators for requests with images check on the host: the pairs' axes, the arguments of the C ABI, the tensors of the
wrappers. No GPU."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from llama_lite_npu_amd import _lib, continuous_batching, ops

FAKE = 1 << 20          # an aligned address that is never read: every call here is refused, or has nothing to do


def test_pairs_of_runs_and_interleaved():
    assert ops.axis_of_pair((2, 1, 1), 8) == bytes([0, 0, 1, 2])
    assert ops.axis_of_pair((64,), 128) == bytes(64)
    got = ops.axis_of_pair((24, 20, 20), 128, True)
    assert [got.count(a) for a in range(3)] == [24, 20, 20]
    assert list(got[:7]) == [0, 1, 2, 0, 1, 2, 0] and list(got[57:]) == [0, 1, 2, 0, 0, 0, 0]
    assert ops.axis_of_pair((16, 24, 24), 128, True).count(1) == 21      # pairs end before the axis' last place


@pytest.mark.parametrize("sections", [(), (8, 8, 8), (63,), (16, 16, 16, 8, 8), (-1, 65), (32.0, 32.0)])
def test_sections_that_do_not_fit(sections):
    with pytest.raises(ValueError, match="sections"):
        ops.axis_of_pair(sections, 128)


def _mrope(**change):
    a = dict(q=FAKE, qs=2048, k=FAKE, ks=1024, v=FAKE, vs=1024, qw=None, kw=None, cos=FAKE, sin=FAKE, stride=64, rows=100,
             positions=FAKE, wide=1, axis=4, token=1, axes=3, pairs=bytes(64), slots=FAKE, pool=FAKE, scales=None, format=0, t=4,
             hq=16, hkv=8, d=128, slots_n=64, eps=1e-6, stream=None)
    a.update(change)
    return _lib.load().litekv_qk_norm_mrope_append(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(format=4), b"pool_format"), (dict(t=-1), b"num_tokens"), (dict(d=96, pairs=bytes(48)), b"head_dim"),
    (dict(d=32, pairs=bytes(16), format=3), b"head_dim"), (dict(axes=0), b"num_axes"), (dict(axes=5), b"num_axes"),
    (dict(pairs=None), b"axis_of_pair"), (dict(pairs=bytes(63) + b"\x03"), b"pair 63 has axis 3"), (dict(q=None), b"null"),
    (dict(sin=None), b"null"), (dict(positions=None), b"null"), (dict(format=1), b"scales"), (dict(scales=FAKE), b"scales"),
    (dict(qw=FAKE), b"go together"), (dict(k=FAKE + 8), b"aligned"), (dict(qs=2040), b"strides"), (dict(vs=1028), b"strides"),
    (dict(rows=0), b"tables"), (dict(stride=56), b"tables"), (dict(stride=68), b"tables"), (dict(slots_n=0), b"num_slots"),
    (dict(slots_n=24, format=3), b"num_slots"), (dict(eps=-1.0), b"rms_eps"), (dict(hq=0), b"num_q_heads")])
def test_mrope_refusals(change, message):
    assert _mrope(**change) == 1 and message in _lib.load().litekv_last_error()


def test_mrope_without_tokens():
    assert _mrope(t=0, q=None, k=None, v=None) == 0


def _cross(**change):
    a = dict(q=FAKE, qs=2048, pool=FAKE, scales=None, format=0, table=FAKE, width=4, cu=FAKE, lens=FAKE, out=FAKE, os=2048, b=2,
             hq=16, hkv=8, d=128, page=16, pages=100, most_rows=4, most_keys=64, t=8, slices=1, ws=None, ws_bytes=0, scale=0.1,
             stream=None)
    a.update(change)
    return _lib.load().litekv_paged_cross_attention(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(format=-1), b"pool_format"), (dict(d=256), b"head_dim"), (dict(d=32), b"head_dim"), (dict(lens=None), b"kv_lens"),
    (dict(cu=None), b"null"), (dict(table=None), b"null"), (dict(format=2), b"scales"), (dict(scales=FAKE), b"scales"),
    (dict(page=48), b"page_size"), (dict(width=0), b"block_table_stride"), (dict(hq=12), b"num_q_heads"),
    (dict(hq=8 * 65, qs=8 * 65 * 128, os=8 * 65 * 128), b"query heads"), (dict(os=2044), b"strides"),
    (dict(q=FAKE + 2), b"aligned"), (dict(slices=9), b"key_slices"), (dict(slices=2), b"workspace"),
    (dict(slices=2, ws=FAKE, ws_bytes=8 * 16 * 2 * 129 * 4 - 1), b"workspace"), (dict(b=70000), b"batch"),
    (dict(pages=0), b"num_pages"), (dict(d=64, lens=None, qs=1024, os=1024), b"kv_lens")])
def test_cross_refusals(change, message):
    assert _cross(**change) == 1 and message in _lib.load().litekv_last_error()


def test_cross_without_rows():
    assert _cross(b=0) == 0 and _cross(most_rows=0) == 0 and _cross(d=64, b=0, qs=1024, os=1024) == 0


def _sample(**change):
    a = dict(logits=FAKE, kind=0, stride=1000, u=FAKE, t=None, k=None, p=None, m=None, tokens=FAKE, logprobs=None, b=2, vocab=1000,
             ws=FAKE, ws_bytes=1 << 20, stream=None)
    a.update(change)
    return _lib.load().litekv_sample_tokens(*a.values())


@pytest.mark.parametrize("change,message", [
    (dict(kind=3), b"logits_type"), (dict(b=-1), b"batch"), (dict(vocab=0), b"vocab"), (dict(vocab=(1 << 20) + 1), b"vocab"),
    (dict(logits=None), b"null"), (dict(u=None), b"null"), (dict(tokens=None), b"null"), (dict(logits=FAKE + 1), b"aligned"),
    (dict(logits=FAKE + 2, kind=2), b"aligned"), (dict(stride=-1), b"row stride"), (dict(ws=None), b"workspace"),
    (dict(ws=FAKE + 4), b"workspace"), (dict(ws_bytes=100), b"workspace")])
def test_sample_refusals(change, message):
    assert _sample(**change) == 1 and message in _lib.load().litekv_last_error()


def test_sample_workspace_and_empty_batch():
    lib = _lib.load()
    assert _sample(b=0, logits=None) == 0
    assert lib.litekv_sample_tokens_workspace_bytes(0, 0, 10) == lib.litekv_sample_tokens_workspace_bytes(5, 1, 10) == 0
    small, large = (lib.litekv_sample_tokens_workspace_bytes(1, b, 152000) for b in (1, 300))
    assert 0 < small < large < 300 * 152000 * 2


@pytest.mark.parametrize("call", [
    lambda x: ops.sample_tokens(x, x[:, 0]), lambda x: ops.sample_tokens(x.double(), x[:, 0]),
    lambda x: ops.qk_norm_mrope_append(x, x, x, x, x, x, (1,), x, x),
    lambda x: ops.paged_cross_attention(x, x, x, x)])
def test_tensors_on_the_cpu_are_refused(call):
    with pytest.raises(ValueError, match="GPU"):
        call(torch.zeros(2, 8))


def test_requests_carry_their_filters_and_plain_ones_go_the_old_way(monkeypatch):
    """A batch without top_k, min_p or a seed is sampled as before; one request with any of them sends it to the kernel."""
    seen = []
    monkeypatch.setattr(continuous_batching, "draw_tokens", lambda logits, requests, generated: seen.append(len(requests)) or "drawn")
    backend = object.__new__(continuous_batching.ContinuousBatchModelBackend)
    backend.executor, backend._sampler = SimpleNamespace(), continuous_batching.sample_next_token
    plain = [continuous_batching.BatchRequest("a", [1], 4, 0.0, 1.0), SimpleNamespace(temperature=0.0, top_p=1.0)]
    logits = torch.tensor([[0.0, 2.0], [3.0, 1.0]])
    assert backend._sample(logits, plain).tolist() == [1, 0] and not seen
    for more in (dict(top_k=3), dict(min_p=0.1), dict(seed=0)):
        request = continuous_batching.BatchRequest("b", [1], 4, 0.7, 1.0, **more)
        assert backend._sample(logits, [plain[0], request]) == "drawn"
    backend._sampler = lambda logits, **kw: "given"
    assert backend._sample(logits, [request]) == "given" and seen == [2, 2, 2]


def test_a_seeded_request_draws_the_same_numbers_in_any_batch(monkeypatch):
    calls = []
    monkeypatch.setattr(continuous_batching.ops, "sample_tokens", lambda rows, *a: calls.append([x.tolist() for x in a]) or rows[:, 0])
    make = lambda name, **kw: continuous_batching.BatchRequest(name, [1], 4, 0.5, 0.75, **kw)  # noqa: E731
    one, two = make("a", seed=7, top_k=5), make("b", seed=8, min_p=0.25)
    other = SimpleNamespace(temperature=1.0, top_p=1.0, generated_token_ids=[])
    logits = torch.zeros(2, 3, 4)
    continuous_batching.draw_tokens(logits, [one, two])
    continuous_batching.draw_tokens(logits, [other, one])
    one.generated_token_ids.append(3)
    continuous_batching.draw_tokens(logits[:1], [one])
    (u, t, k, p, m), second, third = calls
    assert u[0] == second[0][1] != third[0][0] and u[0] != u[1] and all(0 <= x < 1 for x in u)
    assert t == [0.5, 0.5] and k == [5, 0] and p == [0.75, 0.75] and m == [0.0, 0.25]


def test_sharded_logits_refuse_filters_and_a_decode_step_counts_by_positions(monkeypatch):
    seen = []
    monkeypatch.setattr(continuous_batching, "draw_tokens", lambda logits, requests, generated: seen.append(generated) or "drawn")
    backend = object.__new__(continuous_batching.ContinuousBatchModelBackend)
    backend.executor, backend._sampler = SimpleNamespace(logits_are_sharded=False), continuous_batching.sample_next_token
    backend._positions = {9: 6}
    request = continuous_batching.BatchRequest("a", [1, 2, 3], 8, 0.7, 1.0, seed=1)
    request.model_request_id = 9                     # its list is empty, its last token's position 6: 4 have been drawn
    assert backend._sample(None, [request], decoding=True) == "drawn" and backend._sample(None, [request]) == "drawn"
    assert seen == [[4], None]
    backend.executor.logits_are_sharded = True
    with pytest.raises(ValueError, match="shards"):
        backend._sample(None, [request])
