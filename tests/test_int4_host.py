"""4-bit pools without a GPU: what the format promises, and the calls the library refuses before it launches anything."""

import ctypes

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import _lib, ops
from oracle import int4


def rows(seed=0, n=400, d=64):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, d)) * 10.0 ** rng.uniform(-4, 4, (n, 1)) + rng.choice([0.0, 1.0, -30.0], (n, 1))
    x[0], x[1], x[2] = 0.0, 3.0, -3.0
    x[3], x[4, 5] = 65504.0, -65504.0
    x[5] = 6e-8
    return x.astype(np.float16)


def test_every_value_is_an_fp16_number_and_half_a_step_from_its_element():
    x = rows()
    c, s, z = int4.quantise(x)
    values = s[..., None] * (c.astype(np.float64) - z[..., None])
    assert np.array_equal(values.astype(np.float16).astype(np.float64), values)
    assert np.isfinite(values.astype(np.float16)).all()
    clipped = x.astype(np.float64).clip(-int4.MOST, int4.MOST)
    assert (np.abs(values - clipped) <= s[..., None] / 2 * (1 + 1e-12)).all()
    lo, hi = np.minimum(clipped.min(-1), 0), np.maximum(clipped.max(-1), 0)
    assert (s <= np.maximum((hi - lo) / 15 * (1 + 2.0 ** -6), 2.0 ** -20)).all()      # what rounding up may cost
    assert ((s.astype(np.float16).view(np.uint16) & 15) == 0).all()                   # where the zero point goes


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv", [1, 3])
def test_layout_names_every_byte_once(hkv, d):
    at, upper, word = int4.places(hkv, d)
    seen = np.zeros((int4.block_bytes(hkv, d), 2), dtype=int)
    np.add.at(seen, (at, upper.astype(int)), 1)
    np.add.at(seen, (np.stack([word, word + 1]),), 1)
    assert (seen == 1).all()
    for t in range(16):      # no byte belongs to two slots
        mine = set(at[t].ravel()) | set(word[t].ravel()) | set((word[t] + 1).ravel())
        for other in range(t):
            assert not mine & (set(at[other].ravel()) | set(word[other].ravel()) | set((word[other] + 1).ravel()))


def test_store_and_decode_agree():
    rng = np.random.default_rng(3)
    for d in (64, 128):
        pool = rng.integers(0, 256, (64, 4, d // 2 + 2), dtype=np.uint8)
        k, v = rows(1, 40, d).reshape(20, 2, d), rows(2, 40, d).reshape(20, 2, d)
        slots = rng.permutation(64)[:20]
        int4.store(pool, slots, k, v)
        values, _ = int4.decode_pool(pool, 2, d)
        c, s, z = int4.quantise(np.concatenate([k, v], 1))
        assert np.array_equal(values[slots], s[..., None] * (c - z[..., None]))


def test_pools_are_told_apart():
    four = torch.zeros(32, 4, 66, dtype=torch.uint8)
    eight = torch.zeros(32, 4, 128, dtype=torch.uint8)
    assert ops.is_int4_pool(four) and not ops.is_fp8_pool(four) and not ops.is_quantised_pool(four)
    assert not ops.is_int4_pool(eight) and ops.is_fp8_pool(eight) and ops.is_quantised_pool(eight)
    assert not ops.is_int4_pool(torch.zeros(32, 4, 66, dtype=torch.int8))
    assert ops.pool_dtype(four) is torch.uint4 and ops.pool_dtype(eight) is torch.uint8
    assert ops.pool_geometry(four, 16) == (32, 2, 128, 2, 16 * 4 * 66)
    assert ops.int4_row_bytes(64) == 34 and ops.int4_row_bytes(128) == 66
    for d in (32, 96, 256):
        with pytest.raises(ValueError):
            ops.int4_row_bytes(d)


def test_executor_pools_of_four_bits():
    from llama_lite_npu_amd.executor.paged_attention import PagedKVCacheManager

    pages = PagedKVCacheManager(2, 8, 128, 5, 32, torch.uint4, "cpu")
    assert [tuple(p.shape) for p in pages.gpu_kv_buffer] == [(160, 16, 66)] * 2
    assert all(ops.is_int4_pool(p) for p in pages.gpu_kv_buffer) and pages.kv_scales == [None, None]
    with pytest.raises(ValueError):
        pages.set_kv_scales(0, [1.0] * 8, [1.0] * 8)
    with pytest.raises(ValueError):
        PagedKVCacheManager(1, 8, 256, 5, 16, torch.uint4, "cpu")
    with pytest.raises(ValueError):
        PagedKVCacheManager(1, 8, 128, 5, 8, torch.uint4, "cpu")


@pytest.mark.parametrize("args", [(1, 8, 49), (32, 8, 256), (64, 4, 1024), (1, 8, 1), (200, 8, 2), (128, 4, 2048)])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_split_rule_stays_inside_its_bounds(args, page):
    batch, hkv, pages16 = args
    pages = -(-pages16 * 16 // page)
    splits, least = ops.int4_decode_splits(batch, hkv, pages, page_size=page)
    assert 1 <= splits <= 65535 and least >= 1
    assert splits == 1 or (splits - 1) * least < 2 * pages          # not more splits than twice what the pages fill
    assert ops.int4_decode_splits(batch, hkv, pages, batch * pages, page)[0] == splits


def _buffer():
    raw = ctypes.create_string_buffer(4096)
    return raw, (ctypes.addressof(raw) + 63) // 64 * 64


def test_refusals_of_the_library():
    """Host checks: every call below returns before a launch, so the addresses are never read by a GPU."""
    lib = _lib.load()
    raw, p = _buffer()
    good = dict(q=p, q_stride=16 * 128, pool=p, table=p, bt=4, lens=p, k=None, v=None, ks=0, vs=0, out=p, ws=None, wsb=0, b=2,
                hq=16, hkv=8, d=128, page=16, pages=8, splits=1, least=1, scale=0.1)

    def decode(**kw):
        a = {**good, **kw}
        return lib.litekv_paged_decode_int4(a["q"], a["q_stride"], a["pool"], a["table"], a["bt"], a["lens"], a["k"], a["v"],
                                            a["ks"], a["vs"], a["out"], a["ws"], a["wsb"], a["b"], a["hq"], a["hkv"], a["d"],
                                            a["page"], a["pages"], a["splits"], a["least"], a["scale"], None)

    bad = [dict(d=32), dict(d=256), dict(d=96), dict(page=8), dict(page=512), dict(hq=15), dict(hq=0), dict(hkv=0), dict(b=-1),
           dict(b=70000), dict(q=None), dict(pool=None), dict(table=None), dict(lens=None), dict(out=None), dict(q=p + 2),
           dict(pool=p + 8), dict(k=p), dict(k=p, v=p, ks=8, vs=8), dict(k=p, v=p, ks=1028, vs=1024), dict(q_stride=100),
           dict(q_stride=16 * 128 + 4), dict(bt=0), dict(pages=0), dict(pages=1 << 40), dict(splits=0), dict(splits=70000),
           dict(least=0), dict(splits=4), dict(splits=4, ws=p, wsb=16), dict(hq=8 * 65), dict(hkv=2048, hq=2048, q_stride=2048 * 128)]
    for kw in bad:
        assert decode(**kw) == 1, kw
        assert b"paged_decode_int4" in lib.litekv_last_error(), kw
    assert decode(b=0) == 0

    def append(t=4, k=p, v=p, ks=1024, vs=1024, slots=p, pool=p, hkv=8, d=128, n=64):
        return lib.litekv_kv_append_int4(k, v, ks, vs, slots, pool, t, hkv, d, n, None)

    for kw in (dict(t=-1), dict(k=None), dict(slots=None), dict(pool=None), dict(pool=p + 4), dict(ks=1000), dict(vs=1025),
               dict(hkv=0), dict(d=32), dict(d=256), dict(n=0), dict(n=40)):
        assert append(**kw) == 1, kw
    assert append(t=0) == 0

    def epilogue(q=p, qs=2048, qw=None, kw=None, cos=None, sin=None, cs=0, hq=16, d=128, eps=1e-6, n=64):
        return lib.litekv_qk_norm_rope_append_int4(q, qs, p, 1024, p, 1024, qw, kw, cos, sin, cs, p, p, 3, hq, 8, d, n, eps, None)

    for kw in (dict(q=None), dict(hq=0), dict(hq=-2), dict(qs=2000), dict(qw=p), dict(cos=p), dict(cos=p, sin=p, cs=32),
               dict(cos=p, sin=p, cs=65), dict(qw=p + 2, kw=p), dict(d=96), dict(eps=-1.0), dict(n=24)):
        assert epilogue(**kw) == 1, kw

    def dequant(src=p, dst=p, ids=p, out_ids=p, n=2, hkv=8, d=128, page=16, ns=4, nd=4):
        return lib.litekv_page_dequant_int4(src, dst, ids, out_ids, n, hkv, d, page, ns, nd, None)

    for kw in (dict(src=None), dict(dst=None), dict(ids=None), dict(n=-1), dict(hkv=0), dict(d=256), dict(page=24), dict(src=p + 4),
               dict(ns=0), dict(nd=0), dict(out_ids=None, n=5)):
        assert dequant(**kw) == 1, kw
    assert dequant(n=0) == 0

    def prefill(q=p, qs=2048, pool=p, table=p, cu=p, out=p, os=2048, b=1, hq=16, hkv=8, d=128, page=16, pages=8, rows=4, t=4,
                slices=1, ws=None, wsb=0, bt=4):
        return lib.litekv_paged_prefill_int4(q, qs, pool, table, bt, cu, None, out, os, b, hq, hkv, d, page, pages, rows, 64, t,
                                             slices, ws, wsb, 0.1, None)

    for kw in (dict(d=32), dict(d=256), dict(page=8), dict(q=None), dict(pool=None), dict(cu=None), dict(table=None), dict(qs=100),
               dict(os=2052), dict(hq=15), dict(rows=-1), dict(pages=0), dict(bt=0), dict(slices=9), dict(slices=0), dict(slices=2),
               dict(slices=2, ws=p, wsb=8), dict(pool=p + 8), dict(hq=8 * 65, qs=8 * 65 * 128, os=8 * 65 * 128)):
        assert prefill(**kw) == 1, kw
    assert prefill(b=0) == 0


def test_refusals_of_the_wrappers():
    four, q = torch.zeros(32, 4, 66, dtype=torch.uint8), torch.zeros(2, 4, 128, dtype=torch.float16)
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: ops.kv_append_quantised(q[:, :2], q[:, :2], lens, four),
                 lambda: ops.paged_decode(q, four, table, lens),
                 lambda: ops.paged_prefill(q, four, table, torch.tensor([0, 1, 2]), None, 1),
                 lambda: ops.page_dequant(four, q, lens, None, None)):
        with pytest.raises(ValueError, match="must live on the GPU"):
            call()


def test_splits_are_powers_of_two_that_hold_still():
    """Growing sequences ask for a new number of splits (a new captured step) a handful of times, and never back and forth."""
    for batch, hkv, start in ((1, 8, 1), (4, 2, 900), (12, 8, 100), (40, 8, 3000)):
        seen = []
        for tokens in range(start, 140000, 160):
            splits, least = ops.int4_decode_splits(batch, hkv, -(-tokens // 16))
            assert splits & (splits - 1) == 0 and (splits, least) == ops.int4_decode_splits(batch, hkv, -(-tokens // 16), batch * -(-tokens // 16))
            assert splits == 1 or splits // 2 * least * 16 < tokens
            seen.append(splits)
        assert seen == sorted(seen) and seen[0] == 1 and len(set(seen)) <= 7
    assert ops.int4_decode_splits(32, 8, 256)[0] == 1               # 256 pairs fill the device
    # one long sequence among short ones
    assert ops.int4_decode_splits(32, 8, 4096, 4096 + 31)[0] >= 8
    for bad in ((-1, 8, 1, None, 16), (1, 0, 1, None, 16), (1, 8, 4, 5, 16), (1, 8, 1, None, 17), (1, 8, -1, None, 16)):
        with pytest.raises(ValueError):
            ops.int4_decode_splits(*bad)


def test_prefill_workspace_holds_the_keys_where_they_are_decoded_once():
    lib = _lib.load()

    def room(b=1, hq=64, hkv=8, d=128, rows=512, kv=8113, tokens=512, slices=1):
        return lib.litekv_paged_prefill_int4_workspace_bytes(b, hq, hkv, d, rows, kv, tokens, slices)

    pages = -(-8113 // 256)
    assert room() >= pages * 256 * 16 * 128 * 2 + 4 * pages
    assert room(slices=4) >= room() + lib.litekv_paged_prefill_split_workspace_bytes(512, 64, 128, 4)
    assert room(d=64, rows=1024) >= pages * 256 * 16 * 64 * 2 + 4 * pages
    # few blocks of rows a key, lengths not known, more than 1 GiB of keys, heads of another size: the partial rows' alone, or nothing
    assert room(rows=64) == room(kv=0) == room(kv=-1) == room(kv=300000) == room(d=96) == room(b=0) == 0
    assert 0 < room(rows=64, slices=2) < 1 << 26


def test_refusal_of_another_device(monkeypatch):
    """Launches go to the current device: a pool, or a tensor beside it, that lives elsewhere is refused."""
    class Elsewhere:
        is_cuda, shape = True, (32, 4, 66)

        def __init__(self, index):
            self.index, self.device = index, f"cuda:{index}"

        def get_device(self):
            return self.index

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    ops._dev_int4_pool(Elsewhere(0), None, Elsewhere(0), None)
    with pytest.raises(ValueError, match="not the current device"):
        ops._dev_int4_pool(Elsewhere(1), None)
    with pytest.raises(ValueError, match="another device"):
        ops._dev_int4_pool(Elsewhere(0), None, Elsewhere(0), Elsewhere(1))
