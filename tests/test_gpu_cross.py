"""Attention over an encoder's states in pages against the formula in 64 bits: rows of several a sequence and one a sequence, every
pool format, lengths from none to many."""

import math

import pytest
import torch

from llama_lite_npu_amd import ops
from llama_lite_npu_amd.attention import Attention
from llama_lite_npu_amd.executor.encoder_states import EncoderStates

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _pool(g, slots, hkv, d, fmt):
    """(pool, scales, the values it stands for in 64 bits [slots, 2 * Hkv, D])"""
    x = torch.randn(slots, 2 * hkv, d, generator=g, device=DEV).half()
    if fmt == "fp16":
        return x, None, x.double()
    if fmt == "int4":
        pool = torch.zeros(slots, 2 * hkv, d // 2 + 2, device=DEV, dtype=torch.uint8)
        at = torch.arange(slots, device=DEV, dtype=torch.int32)
        ops.kv_append_quantised(x[:, :hkv], x[:, hkv:], at, pool)
        out = torch.empty_like(x)
        ops.page_dequant(pool, out, at[:slots // 16], None, None, 16)
        return pool, None, out.double()
    scales = (0.8 + 0.4 * torch.rand(2 * hkv, generator=g, device=DEV)) * (5.0 / (448 if fmt == "fp8" else 127))
    codes = x.float() / scales[:, None]
    codes = codes.clamp(-448, 448).to(torch.float8_e4m3fn) if fmt == "fp8" else codes.round().clamp(-127, 127).to(torch.int8)
    return codes, scales, codes.float().double() * scales.double()[:, None]


def _case(rows, keys, hq, hkv, d, fmt="fp16", page=16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    each = [-(-n // page) for n in keys]
    pages = sum(each) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(keys), max(1, max(each))), -7, device=DEV, dtype=torch.int32)     # entries that nobody may use
    first = 0
    for b, n in enumerate(each):
        table[b, :n] = order[first:first + n]
        first += n
    pool, scales, values = _pool(g, pages * page, hkv, d, fmt)
    cu = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], device=DEV, dtype=torch.int32)
    q = torch.randn(sum(rows), hq, d, generator=g, device=DEV).half()
    return dict(q=q, pool=pool, scales=scales, values=values, table=table, lens=torch.tensor(keys, device=DEV, dtype=torch.int32),
                cu=cu, rows=rows, keys=keys, page=page, hkv=hkv)


def _want(c, scale=None):
    q, hkv = c["q"].double(), c["hkv"]
    group = q.shape[1] // hkv
    out, first = torch.zeros_like(q), 0
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    for b, (r, n) in enumerate(zip(c["rows"], c["keys"])):
        if n and r:
            at = (c["table"][b].long()[:, None] * c["page"] + torch.arange(c["page"], device=DEV)).reshape(-1)[:n]
            k, v = c["values"][at][:, :hkv], c["values"][at][:, hkv:]
            for h in range(q.shape[1]):
                p = torch.softmax((q[first:first + r, h] @ k[:, h // group].t().contiguous()) * scale, -1)
                out[first:first + r, h] = p @ v[:, h // group]
        first += r
    return out


def _tolerance(c):
    """Probabilities are rounded to fp16 (2^-11 of each, in the sum over keys and in the sum that it is divided by), or to a step
    of 2^-25 of the largest; the output once more. Scores: fp32 sums of up to 128 exact products, and an exponential good to some
    2^-22, for which half a rounding is left."""
    return (3.5 * 2.0 ** -11 + max(c["keys"] + [1]) * 2.0 ** -25) * float(c["values"].abs().max())


def _run(c, **more):
    most = max(c["rows"] + [0])
    return ops.paged_cross_attention(c["q"], c["pool"], c["table"], c["lens"], c["cu"], most, page_size=c["page"],
                                     kv_scales=c["scales"], **more)


def _check(c, got, scale=None):
    assert got.isfinite().all()
    err = (got.double() - _want(c, scale)).abs().max().item()
    assert err <= _tolerance(c), (err, _tolerance(c))


LAYOUTS = [(16, 8, 128), (64, 8, 128), (8, 8, 64), (32, 8, 64), (9, 1, 128), (33, 1, 64)]


@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
@pytest.mark.parametrize("fmt", ["fp16", "fp8", "int8", "int4"])
def test_rows_against_the_formula(hq, hkv, d, fmt):
    """Lengths around the key tile and the page, none among them; more rows than keys and fewer."""
    print(f"cross {hq}/{hkv} D={d} {fmt}", flush=True)
    rows = [1, 3, 17, 70, 5, 130, 2, 0, 40]
    keys = [1, 64, 65, 63, 0, 31, 1000, 77, 128]
    c = _case(rows, keys, hq, hkv, d, fmt, 16, seed=hq)
    _check(c, _run(c))
    _check(c, _run(c, max_kv_len=1000))


@pytest.mark.parametrize("page", [32, 64, 128, 256])
@pytest.mark.parametrize("fmt", ["fp16", "int8", "int4"])
def test_larger_pages(page, fmt):
    print(f"cross page={page} {fmt}", flush=True)
    c = _case([33, 4, 6, 1], [page + 1, page, 3 * page - 5, 2], 16, 4, 128, fmt, page)
    _check(c, _run(c))


@pytest.mark.parametrize("slices", [2, 3, 8])
@pytest.mark.parametrize("fmt", ["fp16", "fp8", "int8", "int4"])
@pytest.mark.parametrize("d", [64, 128])
def test_key_slices(slices, fmt, d):
    """Cut along the keys: short sequences and empty ones have slices without keys."""
    print(f"cross slices={slices} {fmt} D={d}", flush=True)
    c = _case([5, 1, 18, 2, 3], [3000, 0, 64, 129, 1], 16, 4, d, fmt)
    got = _run(c, key_slices=slices)
    _check(c, got)
    assert (got[5] == 0).all()


def test_a_launch_of_many_blocks_and_one_of_one():
    """Each form of the launch: 128 columns a workgroup, 64, and two groups of wavefronts."""
    print("cross: launch forms", flush=True)
    for rows, keys in (([700] * 8, [500, 900, 64, 1, 0, 100, 333, 640]), ([9], [2500]), ([300, 260], [2111, 1500]), ([600], [700])):
        for hq, hkv, d in ((64, 8, 128), (32, 8, 64)):
            c = _case(rows, keys, hq, hkv, d)
            _check(c, _run(c, max_kv_len=max(keys)))


@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
@pytest.mark.parametrize("fmt", ["fp16", "fp8", "int8", "int4"])
def test_one_row_a_sequence(hq, hkv, d, fmt):
    print(f"cross rows {hq}/{hkv} D={d} {fmt}", flush=True)
    keys = [1, 0, 16, 17, 400, 1000, 2500]
    c = _case([1] * len(keys), keys, hq, hkv, d, fmt, seed=3)
    for most in (None, 2500):
        got = ops.paged_cross_attention(c["q"], c["pool"], c["table"], c["lens"], kv_scales=c["scales"], max_kv_len=most)
        err = (got.double() - _want(c)).abs()
        assert (err <= 2e-3 + 1e-2 * _want(c).abs()).all(), err.max()          # the decode kernels' bound
        assert (got[1] == 0).all()
    rows = _run(c, max_kv_len=2500)                                             # the form for several rows says the same
    _check(c, rows)


def test_many_sequences_of_one_row():
    print("cross rows: a large batch", flush=True)
    keys = [(37 * i) % 1300 for i in range(300)]
    c = _case([1] * 300, keys, 32, 4, 128, seed=4)
    got = ops.paged_cross_attention(c["q"], c["pool"], c["table"], c["lens"], max_kv_len=1299)
    assert ((got.double() - _want(c)).abs() <= 2e-3 + 1e-2 * _want(c).abs()).all()


def test_rows_behind_the_last_sequence_and_strides():
    """Rows of padding are left as they are, in every form; q and out may be rows of something wider."""
    print("cross: padding rows, strides", flush=True)
    c = _case([4, 0, 9], [100, 50, 700], 16, 8, 128)
    for slices in (1, 4):
        wide = torch.zeros(20, 16 + 5, 128, device=DEV, dtype=torch.float16)
        q, into = wide[:, :16], torch.full((20, 32, 128), 3.0, device=DEV, dtype=torch.float16)
        q[:13] = c["q"]
        out = into[:, :16]
        got = ops.paged_cross_attention(q, c["pool"], c["table"], c["lens"], c["cu"], 9, out=out, key_slices=slices)
        assert got is out
        _check(c, got[:13].contiguous())
        assert (into[13:] == 3.0).all() and (into[:, 16:] == 3.0).all()


def test_values_in_masked_places_do_not_matter():
    """What lies behind a sequence's last key (in its last page, in pages of others) may be anything."""
    print("cross: NaN behind the last key", flush=True)
    for fmt in ("fp16", "fp8"):
        c = _case([3, 20], [70, 1], 16, 8, 128, fmt)
        want = _run(c).clone()
        used = torch.zeros(c["pool"].shape[0], dtype=torch.bool, device=DEV)
        for b, n in enumerate(c["keys"]):
            at = (c["table"][b].long()[:, None] * 16 + torch.arange(16, device=DEV)).reshape(-1)[:n]
            used[at] = True
        raw = c["pool"].view(torch.uint8)
        raw[~used] = 0x7f if fmt == "fp8" else 0x7e
        for slices in (1, 2):
            got = _run(c, key_slices=slices)
            assert ((got.float() - want.float()).abs() <= _tolerance(c)).all()


def test_lengths_beyond_the_table():
    """More keys than a row of the block table can name: those that it can."""
    print("cross: lengths beyond the table", flush=True)
    c = _case([5, 3], [64, 40], 16, 8, 128)
    c["lens"] = torch.tensor([2 ** 31 - 1, 40], device=DEV, dtype=torch.int32)
    _check(c, _run(c))
    c["lens"] = torch.tensor([-5, 40], device=DEV, dtype=torch.int32)
    c["keys"] = [0, 40]
    _check(c, _run(c))


@pytest.mark.parametrize("scale", [0.01, 0.5])
def test_other_scales(scale):
    c = _case([20, 3], [90, 333], 16, 4, 64, seed=6)
    c["q"] *= 3
    _check(c, _run(c, softmax_scale=scale), scale)


def test_refusals():
    c = _case([2, 3], [10, 20], 16, 8, 128)
    good = dict(q=c["q"], kv_pool=c["pool"], block_table=c["table"], kv_lens=c["lens"], cu_q_lens=c["cu"], max_q_len=3)
    ops.paged_cross_attention(**good)
    for change in (dict(q=c["q"].float()), dict(q=c["q"][:, :, :64]), dict(kv_lens=c["lens"][:1]), dict(block_table=c["table"][:1]),
                   dict(kv_lens=c["lens"].cpu()), dict(kv_scales=torch.ones(16, device=DEV)), dict(softmax_scale=0.0),
                   dict(softmax_scale=-1.0), dict(out=torch.empty(4, 16, 128, device=DEV, dtype=torch.float16)),
                   dict(cu_q_lens=None), dict(block_table=c["table"][:, :0]),
                   dict(key_slices=2, workspace=torch.empty(4, device=DEV))):
        with pytest.raises(ValueError):
            ops.paged_cross_attention(**{**good, **change})
    with pytest.raises(ValueError):
        ops.paged_cross_attention(c["q"][:2], c["pool"], c["table"], c["lens"], key_slices=2)
    pool = torch.zeros(64, 16, 256, device=DEV, dtype=torch.float16)
    with pytest.raises(ValueError, match="head_dim"):
        ops.paged_cross_attention(torch.zeros(5, 16, 256, device=DEV, dtype=torch.float16), pool, c["table"], c["lens"], c["cu"], 3)


def test_replayed_from_a_graph():
    """The lengths are read at each replay."""
    print("cross: graph", flush=True)
    c = _case([6, 3], [700, 300], 16, 8, 128)
    for more in (dict(key_slices=4), dict()):
        out = torch.empty_like(c["q"])
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            _run(c, out=out, **more)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                _run(c, out=out, **more)
        for lens in ([700, 300], [0, 1], [65, 299], [700, 0]):
            c["lens"].copy_(torch.tensor(lens))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c["keys"] = lens
            _check(c, out)
        c["lens"].copy_(torch.tensor([700, 300]))
        c["keys"] = [700, 300]


@pytest.mark.parametrize("dtype", [torch.float16, torch.int8, torch.uint4])
def test_states_stored_once_and_attended_by_a_layer(dtype):
    """EncoderStates through Attention.cross_forward: a prompt's rows, then steps of one row each."""
    print(f"cross: layer over {dtype}", flush=True)
    lengths, hq, hkv, d = [130, 0, 33, 64], 16, 4, 128
    g = torch.Generator(device=DEV).manual_seed(12)
    scales = [torch.full((2 * hkv,), 4.5 / 127, device=DEV)] * 2 if dtype is torch.int8 else None
    states = EncoderStates(lengths, 2, hkv, d, 32, dtype, DEV, scales)
    layer = Attention(hq, hkv, d)
    for index in range(2):
        k, v = (torch.randn(sum(lengths), hkv, d, generator=g, device=DEV).half() for _ in range(2))
        states.store(index, k, v)
        c = dict(rows=[5, 2, 7, 1], keys=lengths, page=32, hkv=hkv, table=states.block_table)
        c["q"] = torch.randn(15, hq, d, generator=g, device=DEV).half()
        held = torch.zeros(states.kv_buffer[0].shape[0], 2 * hkv, d, device=DEV, dtype=torch.float16)
        pages = torch.arange(held.shape[0] // 32, device=DEV, dtype=torch.int32)
        if dtype is torch.float16:
            held = states.kv_buffer[index]
        else:
            ops.page_dequant(states.kv_buffer[index], held, pages, None, states.kv_scales[index], 32)
        c["values"] = held.double()
        # half a code's step: of the scale, beyond whose 127 codes values stay at the last; or of a fifteenth of the row's range, rounded up
        # by 2^-6 at most; and half a rounding to fp16 of what is read back
        given = torch.cat((k, v), 1).double()
        span = given.amax(-1, keepdim=True).clamp(min=0) - given.amin(-1, keepdim=True).clamp(max=0)
        half = {torch.float16: 0.0, torch.int8: 0.5 * 4.5 / 127, torch.uint4: span * (0.5 / 15 * (1 + 2.0 ** -6))}[dtype]
        if dtype is torch.int8:
            given = given.clamp(-4.5, 4.5)
        assert ((held[states.slot_mapping.long()].double() - given).abs() <= half + given.abs() * 2.0 ** -11 * (dtype is not torch.float16)).all()
        cu = torch.tensor([0, 5, 7, 14, 15], device=DEV, dtype=torch.int32)
        _check(c, layer.cross_forward(c["q"], states, index, cu, 7))
        c["q"], c["rows"] = c["q"][:4].contiguous(), [1] * 4
        got = layer.cross_forward(c["q"], states, index)
        assert ((got.double() - _want(c)).abs() <= 2e-3 + 1e-2 * _want(c).abs()).all()
    assert len(states._plans) == 1
