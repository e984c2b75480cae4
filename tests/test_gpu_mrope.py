"""The QKV epilogue with positions of several axes against its definition in 64 bits, over every pool format."""

import pytest
import torch

from llama_lite_npu_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TABLE = 3000


def _inputs(seed, t, hq, hkv, d, fmt, norm=True, axes=3, wide=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    qkv = (randn(t, hq + 2 * hkv, d) * 1.7).half()                         # strided views, as after a fused projection
    s = dict(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
    s["wq"], s["wk"] = ((1 + 0.2 * randn(d)).half(), (1 + 0.2 * randn(d)).half()) if norm else (None, None)
    angle = torch.arange(TABLE, device=DEV).double()[:, None] * 1e4 ** (-torch.arange(0, d, 2, device=DEV).double() / d)
    s["cos"], s["sin"] = angle.cos().half(), angle.sin().half()
    s["positions"] = torch.randint(0, TABLE, (axes, t), generator=g, device=DEV, dtype=torch.int64 if wide else torch.int32)
    slots = max(64, 2 * t) // 16 * 16 + 16
    s["slots"] = torch.randperm(slots, generator=g, device=DEV)[:t].to(torch.int32)
    row = d // 2 + 2 if fmt == "int4" else d
    s["pool"] = torch.zeros(slots, 2 * hkv, row, device=DEV, dtype={"fp16": torch.float16, "fp8": torch.float8_e4m3fn,
                                                                    "int8": torch.int8, "int4": torch.uint8}[fmt])
    s["scales"] = None
    if fmt in ("fp8", "int8"):
        s["scales"] = (0.7 + 0.6 * torch.rand(2 * hkv, generator=g, device=DEV)) * (9.0 / (448 if fmt == "fp8" else 127))
    return s


def _run(s, sections, interleaved=False, **change):
    a = {**s, **change}
    return ops.qk_norm_mrope_append(a["q"], a["k"], a["v"], a["slots"], a["pool"], a["positions"], sections, a["cos"], a["sin"],
                                    a["wq"], a["wk"], 1e-6, kv_scales=a["scales"], interleaved=interleaved)


def _want(s, sections, interleaved):
    """q, K and V rows in 64 bits, and the largest parts that the rotation adds up."""
    d = s["q"].shape[2]
    axis = torch.tensor(list(ops.axis_of_pair(tuple(sections), d, interleaved)), device=DEV)
    at = s["positions"].long().clamp(0, TABLE - 1)[axis].t()                   # [T, D / 2]
    pair = torch.arange(d // 2, device=DEV)
    cos, sin = s["cos"].double()[at, pair][:, None], s["sin"].double()[at, pair][:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1), torch.cat((a.abs() + b.abs(),) * 2, -1)

    q, q_parts = turned(s["q"], s["wq"])
    k, k_parts = turned(s["k"], s["wk"])
    v = s["v"].double()
    return q, q_parts, torch.cat((k, v), 1), torch.cat((k_parts, v.abs()), 1)


def _values(s):
    """What the pool holds, in 64 bits."""
    pool, hkv = s["pool"], s["k"].shape[1]
    if pool.dtype is torch.float16:
        return pool.double()
    if pool.dtype is not torch.uint8:
        return pool.float().double() * s["scales"].double()[:, None]
    out = torch.zeros(pool.shape[0], 2 * hkv, s["q"].shape[2], device=DEV, dtype=torch.float16)
    ops.page_dequant(pool, out, torch.arange(pool.shape[0] // 16, device=DEV, dtype=torch.int32), None, None, 16)
    return out.double()


def _check(s, sections, interleaved, live):
    """fp32 arithmetic: about eight roundings of 2^-24 of the parts; then one rounding, of half a step."""
    want_q, q_parts, rows, parts = _want(s, sections, interleaved)
    before = _values(s)
    out = _run(s, sections, interleaved)
    assert out is s["q"]
    torch.cuda.synchronize()
    err = (s["q"].double() - want_q).abs()
    assert (err <= want_q.abs() * 2.0 ** -11 + q_parts * 2.0 ** -21 + 2.0 ** -25).all(), err.max()
    slots = s["slots"].long()[live]
    got, rows, parts = _values(s), rows[live], parts[live]
    held = got[slots]
    noise = parts * 2.0 ** -21
    if s["pool"].dtype is torch.float16:
        half = rows.abs() * 2.0 ** -11 + 2.0 ** -25
    elif s["pool"].dtype is torch.uint8:      # half of a step of (range / 15), the step rounded up by at most 2^-6
        span = rows.amax(-1, keepdim=True).clamp(min=0) - rows.amin(-1, keepdim=True).clamp(max=0)
        half = span * (0.5 / 15 * (1 + 2.0 ** -6)) + 2.0 ** -19
    else:
        scale = s["scales"].double()[:, None]
        most = (448 if s["pool"].dtype is torch.float8_e4m3fn else 127) * scale
        rows = rows.clamp(-most, most)
        half = 0.5 * scale.expand_as(rows)
        if s["pool"].dtype is torch.float8_e4m3fn:
            half = torch.maximum(rows.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    err = (held - rows).abs()
    assert (err <= half * (1 + 2.0 ** -12) + noise).all(), (err - half).max()
    rest = torch.ones(got.shape[0], dtype=torch.bool, device=DEV)
    rest[slots] = False
    assert torch.equal(got[rest], before[rest])                                # other slots are left alone


CASES = [
    # tokens, heads, head dim, format, sections, interleaved, norm, int64 positions
    (1, 16, 8, 128, "fp16", (16, 24, 24), False, True, True),
    (33, 64, 8, 128, "fp16", (24, 20, 20), True, True, False),
    (7, 28, 4, 128, "fp8", (16, 24, 24), False, False, True),
    (36, 64, 8, 128, "int8", (24, 20, 20), True, True, True),
    (19, 32, 4, 128, "int4", (24, 20, 20), True, True, False),
    (130, 32, 8, 64, "fp16", (11, 13, 8), False, True, True),         # runs that end inside a lane's eight pairs
    (65, 14, 2, 64, "fp8", (8, 12, 12), True, True, True),
    (17, 32, 8, 64, "int4", (8, 12, 12), False, False, True),
    (5, 9, 3, 32, "fp16", (4, 6, 6), True, True, True),
    (40, 5, 1, 32, "int8", (6, 5, 5), False, False, False),
    (12, 16, 4, 256, "fp16", (44, 42, 42), True, True, True),
    (21, 3, 1, 256, "fp8", (32, 48, 48), False, True, False),
    (9, 8, 8, 128, "fp16", (64,), False, True, True),                  # one axis
    (10, 16, 8, 128, "fp16", (20, 20, 12, 12), True, True, True),      # four
    (11, 16, 8, 128, "int8", (0, 64), False, True, True),
    (3000, 16, 8, 128, "fp16", (24, 20, 20), True, True, True),
    (2500, 64, 8, 64, "int8", (8, 12, 12), False, True, True),
]


@pytest.mark.parametrize("t,hq,hkv,d,fmt,sections,interleaved,norm,wide", CASES)
def test_against_the_definition(t, hq, hkv, d, fmt, sections, interleaved, norm, wide):
    print(f"mrope T={t} {hq}/{hkv} D={d} {fmt} {sections} interleaved={interleaved} norm={norm}", flush=True)
    s = _inputs(t + d, t, hq, hkv, d, fmt, norm, len(sections), wide)
    live = torch.ones(t, dtype=torch.bool, device=DEV)
    if t > 3:                                          # padding rows: q is processed, nothing is stored
        s["slots"][t // 2], s["slots"][3] = -1, s["pool"].shape[0] + 5
        live[t // 2] = live[3] = False
    _check(s, sections, interleaved, live)


@pytest.mark.parametrize("fmt", ["fp16", "int8", "int4"])
def test_equal_axes_are_one_axis(fmt):
    """A text token's axes are one number: an expanded row of positions gives what one axis does, to the bit, wherever the
    pairs' axes lie."""
    print(f"mrope: expanded positions, {fmt}", flush=True)
    outs = []
    for sections, interleaved in (((64,), False), ((16, 24, 24), False), ((24, 20, 20), True)):
        s = _inputs(5, 29, 16, 8, 128, fmt)
        s["positions"] = s["positions"][:1].expand(len(sections), -1)
        _run(s, sections, interleaved)
        outs.append((s["q"].clone(), s["pool"].clone()))
    for q, pool in outs[1:]:
        assert torch.equal(q, outs[0][0]) and torch.equal(pool, outs[0][1])


@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_plain_rope_with_rows_of_the_table(d):
    """One axis without norm is the rotation that the epilogue of one-axis positions makes, which for such rows is the same
    arithmetic."""
    print(f"mrope: one axis, D={d}", flush=True)
    s = _inputs(6, 23, 8, 2, d, "fp16", norm=False, axes=1)
    q, pool, at = s["q"].clone(), s["pool"].clone(), s["positions"][0]
    ops.qk_norm_rope_append(q, s["k"], s["v"], s["slots"], pool, None, None, s["cos"][at], s["sin"][at])
    _run(s, (d // 2,))
    # (fused there: each product and sum rounded by itself here; one fp16 step of the larger at most)
    assert ((q.float() - s["q"].float()).abs() <= q.float().abs().clamp(min=2.0 ** -14) * 2.0 ** -10).all()
    assert torch.equal(pool[:, 2:], s["pool"][:, 2:])


def test_positions_outside_the_tables_and_other_strides():
    print("mrope: positions outside, strides", flush=True)
    s = _inputs(7, 31, 16, 8, 128, "fp16")
    s["positions"][0, :3] = torch.tensor([-1, TABLE, 1 << 40], device=DEV)
    twin = {n: x.clone() if n in ("q", "pool") else x for n, x in s.items()}
    twin["positions"] = s["positions"].clamp(0, TABLE - 1).t().contiguous().t()          # axis by axis inside a token
    wide = torch.zeros(TABLE, 96, device=DEV, dtype=torch.float16)
    wide[:, :64] = s["cos"]
    sine = torch.zeros_like(wide)
    sine[:, :64] = s["sin"]
    _run(s, (16, 24, 24))
    _run(twin, (16, 24, 24), cos=wide, sin=sine)
    assert torch.equal(s["q"], twin["q"]) and torch.equal(s["pool"], twin["pool"])


def test_values_that_are_not_finite():
    """8-bit codes: NaN becomes the most negative code and infinities the outermost; in q they stay what they are. Other rows are
    not touched."""
    print("mrope: not finite", flush=True)
    for fmt, most in (("fp8", 448.0), ("int8", 127.0)):
        s = _inputs(8, 6, 4, 2, 128, fmt, norm=False)
        s["v"][1, 0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")], device=DEV).half()
        s["q"][2, 0, 5] = float("nan")
        _run(s, (16, 24, 24))
        row = s["pool"][s["slots"][1].long(), 2].float()
        assert row[:3].tolist() == [most, -most, -most]
        assert s["q"][2, 0].isnan().sum() == 2 and s["q"].isnan().sum() == 2


def test_no_tokens():
    s = _inputs(9, 4, 4, 2, 128, "fp16")
    pool = s["pool"].clone()
    _run(s, (16, 24, 24), q=s["q"][:0], k=s["k"][:0], v=s["v"][:0], slots=s["slots"][:0], positions=s["positions"][:, :0])
    assert torch.equal(pool, s["pool"])


def test_refusals():
    s = _inputs(10, 4, 4, 2, 128, "fp16")
    for change in (dict(positions=s["positions"].float()), dict(positions=s["positions"][:2]), dict(cos=s["cos"].float()),
                   dict(cos=s["cos"][:, :32], sin=s["sin"][:, :32]), dict(sin=s["sin"][:5]), dict(slots=s["slots"][:2]),
                   dict(wk=None), dict(scales=torch.ones(4, device=DEV)), dict(k=s["k"][:, :1]), dict(cos=s["cos"].cpu()),
                   dict(positions=s["positions"].cpu()), dict(q=s["q"].float())):
        with pytest.raises(ValueError):
            _run(s, (16, 24, 24), **change)
    with pytest.raises(ValueError, match="sections"):
        _run(s, (16, 24, 23))


def test_replayed_from_a_graph_on_another_stream():
    """Positions and slots are read at each replay; three replays beside eager work, each checked."""
    print("mrope: graph", flush=True)
    s = _inputs(11, 12, 16, 8, 128, "int8")
    given, stream = s["q"].clone(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _run(s, (24, 20, 20), True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            _run(s, (24, 20, 20), True)
    for i in range(3):
        s["positions"].copy_(torch.randint(0, TABLE, s["positions"].shape, device=DEV))
        s["slots"].copy_(torch.randperm(s["pool"].shape[0], device=DEV)[:12].to(torch.int32))
        s["q"].copy_(given)
        s["pool"].zero_()
        twin = {**s, "q": given.clone(), "pool": s["pool"].clone()}
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _run(twin, (24, 20, 20), True)
        torch.cuda.synchronize()
        assert torch.equal(s["q"], twin["q"]) and torch.equal(s["pool"], twin["pool"]), i
