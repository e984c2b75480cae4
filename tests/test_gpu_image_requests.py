"""What a step of requests with images runs together, as it would be used: the epilogue with positions of several axes, the attention
over the cache, the attention over an encoder's states, the draw. And what the three share: calls in native code and from Python,
pools past 32-bit offsets, captured steps."""

import math
from types import SimpleNamespace

import pytest
import torch

from llama_lite_npu_amd import _lib, ops
from llama_lite_npu_amd.attention import Attention
from llama_lite_npu_amd.executor.encoder_states import EncoderStates

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HQ, HKV, D, VOCAB, PAGE = 16, 4, 128, 5000, 16


def _tables(rows, d=D):
    angle = torch.arange(rows, device=DEV).double()[:, None] * 1e4 ** (-torch.arange(0, d, 2, device=DEV).double() / d)
    return angle.cos().half(), angle.sin().half()


def _without_native_calls(monkeypatch):
    none = lambda *a: None  # noqa: E731
    monkeypatch.setattr(_lib, "calls", lambda: SimpleNamespace(qk_norm_mrope_append=none, paged_cross_attention=none,
                                                               sample_tokens=none))


def _both(monkeypatch, call):
    """The same call in native code and from Python."""
    asked = _lib.calls()
    native = call()
    with monkeypatch.context() as m:
        _without_native_calls(m)
        plain = call()
    assert _lib.calls() is asked
    return native, plain


@pytest.mark.parametrize("fmt", ["fp16", "fp8", "int8", "int4"])
def test_native_calls_and_those_from_python_are_the_same(fmt, monkeypatch):
    print(f"image requests: native calls {fmt}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(2)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV).half()  # noqa: E731
    t, slots = 40, 256
    row = D // 2 + 2 if fmt == "int4" else D
    dtype = {"fp16": torch.float16, "fp8": torch.float8_e4m3fn, "int8": torch.int8, "int4": torch.uint8}[fmt]
    scales = torch.rand(2 * HKV, generator=g, device=DEV) * 0.02 + 0.02 if fmt in ("fp8", "int8") else None
    given, k, v, wq, wk = randn(t, HQ, D), randn(t, HKV, D), randn(t, HKV, D), randn(D), randn(D)
    at = torch.randperm(slots, generator=g, device=DEV)[:t].to(torch.int32)
    positions = torch.randint(0, 500, (3, t), generator=g, device=DEV)
    cos, sin = _tables(500)

    def epilogue():
        pool = torch.zeros(slots, 2 * HKV, row, device=DEV, dtype=dtype)
        q = ops.qk_norm_mrope_append(given.clone(), k, v, at, pool, positions, (24, 20, 20), cos, sin, wq, wk, 1e-6, scales, True)
        return q, pool

    (q1, pool), (q2, other) = _both(monkeypatch, epilogue)
    assert torch.equal(q1, q2) and torch.equal(pool.view(torch.uint8), other.view(torch.uint8))

    table = torch.arange(slots // PAGE, device=DEV, dtype=torch.int32).view(2, -1).contiguous()
    lens, cu = torch.tensor([128, 33], device=DEV, dtype=torch.int32), torch.tensor([0, 30, 38], device=DEV, dtype=torch.int32)
    for most in (None, 128):
        one, two = _both(monkeypatch, lambda: ops.paged_cross_attention(q1, pool, table, lens, cu, 30, page_size=PAGE,
                                                                        kv_scales=scales, max_kv_len=most)[:38])
        assert torch.equal(one, two)
        one, two = _both(monkeypatch, lambda: ops.paged_cross_attention(q1[:2], pool, table, lens, page_size=PAGE, kv_scales=scales,
                                                                        max_kv_len=most))
        assert torch.equal(one, two)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_native_draws_and_those_from_python_are_the_same(dtype, monkeypatch):
    print(f"image requests: native draws {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(5, VOCAB, generator=g, device=DEV).to(dtype)
    u, t = torch.rand(5, generator=g, device=DEV), torch.linspace(0, 2, 5, device=DEV)
    k, p = torch.tensor([0, 5, 50, 0, 9], device=DEV, dtype=torch.int32), torch.full((5,), 0.9, device=DEV)
    for filters in (dict(), dict(temperature=t, top_k=k, top_p=p), dict(min_p=p - 0.8)):
        one, two = _both(monkeypatch, lambda: ops.sample_tokens(x, u, **filters, return_logprobs=True))
        assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
        assert torch.equal(ops.sample_tokens(x, u, **filters), one[0])


@pytest.mark.parametrize("fmt", ["fp16", "int8", "int4"])
def test_pools_past_32_bit_offsets(fmt):
    """The last pages of a pool of more than 2^32 bytes (and, in fp16, more than 2^31 elements)."""
    print(f"image requests: a large pool {fmt}", flush=True)
    hkv, tokens = 8, 50
    row = D // 2 + 2 if fmt == "int4" else D
    dtype = {"fp16": torch.float16, "int8": torch.int8, "int4": torch.uint8}[fmt]
    slots = (2 ** 32 // (2 * hkv * row) // 16 + 300) * 16 if fmt != "fp16" else (2 ** 31 // (2 * hkv * row) // 16 + 300) * 16
    pool = torch.empty(slots, 2 * hkv, row, device=DEV, dtype=dtype)
    pages = torch.tensor([[slots // 16 - 1, 3, slots // 16 - 200, 0]], device=DEV, dtype=torch.int32)
    at = (pages[0].long()[:, None] * 16 + torch.arange(16, device=DEV)).reshape(-1)[:tokens].to(torch.int32)
    g = torch.Generator(device=DEV).manual_seed(4)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV).half()  # noqa: E731
    q, k, v = randn(tokens, 16, D), randn(tokens, hkv, D), randn(tokens, hkv, D)
    cos, sin = _tables(4)
    scales = torch.full((2 * hkv,), 5.0 / 127, device=DEV) if fmt == "int8" else None
    zero = torch.zeros(3, tokens, device=DEV, dtype=torch.int32)                 # (position 0: rows as they are)
    ops.qk_norm_mrope_append(q, k, v, at, pool, zero, (24, 20, 20), cos, sin, kv_scales=scales)
    lens, cu = torch.tensor([tokens], device=DEV, dtype=torch.int32), torch.tensor([0, tokens], device=DEV, dtype=torch.int32)
    got = ops.paged_cross_attention(q, pool, pages, lens, cu, tokens, page_size=16, kv_scales=scales)
    small = torch.zeros(64, 2 * hkv, row, device=DEV, dtype=dtype)
    ops.qk_norm_mrope_append(q.clone(), k, v, torch.arange(tokens, device=DEV, dtype=torch.int32), small, zero, (24, 20, 20), cos,
                             sin, kv_scales=scales)
    near = torch.arange(4, device=DEV, dtype=torch.int32)[None]
    assert torch.equal(got, ops.paged_cross_attention(q, small, near, lens, cu, tokens, page_size=16, kv_scales=scales))
    one = ops.paged_cross_attention(q[:1], pool, pages, lens, page_size=16, kv_scales=scales)
    assert torch.equal(one, ops.paged_cross_attention(q[:1], small, near, lens, page_size=16, kv_scales=scales))


def test_the_largest_vocabulary():
    print("image requests: 2^20 tokens", flush=True)
    x = torch.zeros(2, (1 << 20) + 1, device=DEV, dtype=torch.float16)
    u = torch.tensor([0.0, 0.75], device=DEV)
    # all alike: the token is the first at which (i + 1) / n exceeds u, in the kept run the lowest indexes
    assert ops.sample_tokens(x[:, :-1], u).tolist() == [0, 3 << 18]
    half = torch.full((2,), 0.5, device=DEV)
    assert ops.sample_tokens(x[:, :-1], u, top_p=half).tolist() == [0, 3 << 17]
    assert ops.sample_tokens(x[:, :-1], u, top_k=torch.full((2,), 1 << 16, device=DEV, dtype=torch.int32)).tolist() == [0, 3 << 14]
    x[:, (1 << 20) - 1] = 30
    assert ops.sample_tokens(x[:, :-1], u + 0.2).tolist() == [(1 << 20) - 1] * 2
    with pytest.raises(_lib.LiteKVError, match="vocab"):
        ops.sample_tokens(x, u)


class _Step:
    """One layer of a decoder over an encoder's states, and its logits."""

    def __init__(self, g, lengths, batch_pages):
        randn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
        self.width = 256
        self.wqkv = (randn(self.width, (HQ + 2 * HKV) * D) / 16).half()
        self.wcross, self.whead = (randn(HQ * D, HQ * D) / 45).half(), (randn(HQ * D, VOCAB) / 8).half()
        self.wq, self.wk = (1 + 0.1 * randn(D)).half(), (1 + 0.1 * randn(D)).half()
        self.cos, self.sin = _tables(400)
        self.layer = Attention(HQ, HKV, D)
        self.states = EncoderStates(lengths, 1, HKV, D, PAGE, device=DEV)
        self.states.store(0, randn(sum(lengths), HKV, D).half(), randn(sum(lengths), HKV, D).half())
        b = len(lengths)
        self.pool = torch.zeros(b * batch_pages * PAGE, 2 * HKV, D, device=DEV, dtype=torch.float16)
        self.table = torch.arange(b * batch_pages, device=DEV, dtype=torch.int32).view(b, -1).contiguous()

    def info(self, slots):
        return SimpleNamespace(kv_buffer=[self.pool], kv_scales=[None], cur_select_index=slots)

    def qkv(self, x, slots, positions):
        rows = (x @ self.wqkv).view(-1, HQ + 2 * HKV, D)
        return self.layer.qkv_epilogue_axes(rows[:, :HQ], rows[:, HQ:HQ + HKV], rows[:, HQ + HKV:], self.info(slots), 0, positions,
                                            (24, 20, 20), self.cos, self.sin, self.wq, self.wk, interleaved=True)

    def draw(self, mixed, u):
        logits = mixed.reshape(-1, HQ * D) @ self.whead
        return logits, ops.sample_tokens(logits, u, top_p=torch.full_like(u, 0.9))

    def cross(self, mixed, *rows):
        return self.layer.cross_forward((mixed.reshape(-1, HQ * D) @ self.wcross).view(-1, HQ, D), self.states, 0, *rows)


def _attended(q, pool, slots, last):
    """Row i of q over the slots [0, last[i]] in 64 bits."""
    k, v = pool[slots.long()].double().split([HKV, HKV], 1)
    out = torch.empty(q.shape, device=DEV, dtype=torch.double)
    for h in range(HQ):
        scores = q[:, h].double() @ k[:, h // (HQ // HKV)].t().contiguous() / math.sqrt(D)
        scores.masked_fill_(torch.arange(k.shape[0], device=DEV) > last[:, None], float("-inf"))
        out[:, h] = scores.softmax(-1) @ v[:, h // (HQ // HKV)].contiguous()
    return out


def test_prompts_then_captured_steps():
    """Prompts with images, then steps captured into a graph: each part against 64 bits from the inputs that it was given, and every
    replay against the same step run eagerly."""
    print("image requests: prompts", flush=True)
    g = torch.Generator(device=DEV).manual_seed(6)
    prompts, lengths = [37, 5, 18], [140, 0, 33]
    step, b = _Step(g, lengths, 8), 3
    cu = torch.tensor([0, 37, 42, 60], device=DEV, dtype=torch.int32)
    slots = torch.cat([torch.arange(n, device=DEV, dtype=torch.int32) + i * 8 * PAGE for i, n in enumerate(prompts)])
    # an image of 4 rows of 5 behind two tokens of text, say: time stands still, height and width go on
    grid = torch.arange(60, device=DEV)
    positions = torch.stack((grid // 20, grid // 5 % 4 + grid // 20, grid % 5 + grid // 20)) + 2
    x = torch.randn(60, step.width, generator=g, device=DEV).half()
    q = step.qkv(x, slots, positions)
    mixed = ops.paged_prefill(q, step.pool, step.table, cu, torch.zeros(b, device=DEV, dtype=torch.int32), 37, page_size=PAGE)
    for i, n in enumerate(prompts):
        rows = slice(int(cu[i]), int(cu[i + 1]))
        want = _attended(q[rows], step.pool, slots[rows], torch.arange(n, device=DEV))
        assert ((mixed[rows].double() - want).abs() <= 2e-3 + 1e-2 * want.abs()).all()
    crossed = step.cross(mixed, cu, 37)
    q_cross = (mixed.reshape(-1, HQ * D) @ step.wcross).view(-1, HQ, D)
    for i, n in enumerate(lengths):
        rows = slice(int(cu[i]), int(cu[i + 1]))
        own = (step.states.block_table[i].long()[:, None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(-1)[:n]
        want = _attended(q_cross[rows], step.states.kv_buffer[0], own, torch.full((prompts[i],), n, device=DEV)) if n else 0 * q_cross[rows].double()
        assert ((crossed[rows].double() - want).abs() <= 2e-3 + 1e-2 * want.abs()).all()

    print("image requests: captured steps", flush=True)
    x, u = torch.zeros(b, step.width, device=DEV, dtype=torch.float16), torch.zeros(b, device=DEV)
    at, lens = torch.zeros(b, device=DEV, dtype=torch.int32), torch.zeros(b, device=DEV, dtype=torch.int32)
    axes = torch.zeros(3, b, device=DEV, dtype=torch.int64)

    def run():
        q = step.qkv(x, at, axes)
        mixed = ops.paged_decode(q, step.pool, step.table, lens, page_size=PAGE)
        crossed = step.cross(mixed)                                     # (its plan first made while the graph is captured)
        return (mixed, crossed) + step.draw(mixed + crossed, u)

    def set_step(n):
        h = torch.Generator(device=DEV).manual_seed(100 + n)
        x.copy_(torch.randn(b, step.width, generator=h, device=DEV))
        u.copy_(torch.rand(b, generator=h, device=DEV))
        upto = torch.tensor([p + n for p in prompts], device=DEV, dtype=torch.int32)
        at.copy_(upto + torch.arange(b, device=DEV, dtype=torch.int32) * 8 * PAGE)
        lens.copy_(upto + 1)
        axes.copy_(upto[None].expand(3, b))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        set_step(0)
        step.draw(step.qkv(x, at, axes), u)                             # (libraries of the products start up outside the graph)
        mixed = ops.paged_decode(q[:b], step.pool, step.table, lens, page_size=PAGE)
        mixed.reshape(-1, HQ * D) @ step.wcross
        torch.cuda.synchronize()
        assert not step.states._plans
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            held = run()
    assert not step.states._plans                                        # nothing that only a replay would fill is kept
    for n in range(4):
        set_step(n)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in held]
        eager = run()
        torch.cuda.synchronize()
        for a, e in zip(got, eager):
            assert torch.equal(a, e), n
        mixed, crossed, logits, tokens = got
        assert (crossed[1] == 0).all() and ((tokens >= 0) & (tokens < VOCAB)).all()
        p = logits.double().softmax(-1)
        order = p.sort(descending=True, stable=True)
        kept = torch.zeros_like(p).scatter_(1, order.indices, ((order.values.cumsum(-1) - order.values) < 0.9).double())
        assert (kept.gather(1, tokens[:, None]) == 1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.uint4])
def test_a_batch_without_states(dtype):
    """No sequence has any: nothing to store, rows of zeros in both forms."""
    print(f"image requests: no states {dtype}", flush=True)
    states, layer = EncoderStates([0, 0], 1, HKV, D, PAGE, dtype, DEV), Attention(HQ, HKV, D)
    none = torch.empty(0, HKV, D, device=DEV, dtype=torch.float16)
    states.store(0, none, none)
    q = torch.randn(5, HQ, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)).half()
    cu = torch.tensor([0, 2, 5], device=DEV, dtype=torch.int32)
    assert (layer.cross_forward(q, states, 0, cu, 3) == 0).all() and (layer.cross_forward(q[:2], states, 0) == 0).all()


def test_two_streams_at_once():
    """Calls that overlap on two streams have workspaces of their own: each is what it is alone."""
    print("image requests: two streams", flush=True)
    g = torch.Generator(device=DEV).manual_seed(8)
    sides = []
    for n in (2000, 900):
        pool = torch.randn(2048 + 16 * n % 512, 2 * HKV, D, generator=g, device=DEV).half()
        table = torch.randperm(pool.shape[0] // PAGE, generator=g, device=DEV).to(torch.int32)[None, :128].contiguous()
        q, x = torch.randn(4, HQ, D, generator=g, device=DEV).half(), torch.randn(7, 30000, generator=g, device=DEV)
        lens, cu = torch.tensor([n], device=DEV, dtype=torch.int32), torch.tensor([0, 4], device=DEV, dtype=torch.int32)
        u, p = torch.rand(7, generator=g, device=DEV), torch.full((7,), 0.9, device=DEV)

        def call(q=q, pool=pool, table=table, lens=lens, cu=cu, x=x, u=u, p=p, n=n):
            return (ops.paged_cross_attention(q, pool, table, lens, cu, 4, page_size=PAGE, max_kv_len=n),
                    ops.paged_cross_attention(q[:1], pool, table, lens, page_size=PAGE, max_kv_len=n), ops.sample_tokens(x, u, top_p=p))

        sides.append((call, call(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for (call, _, stream), kept in zip(sides, got):
            with torch.cuda.stream(stream):
                kept.append(call())
    torch.cuda.synchronize()
    for (_, want, _), kept in zip(sides, got):
        for one in kept:
            assert all(torch.equal(a, b) for a, b in zip(one, want))
