"""The 4-bit pool's operators against the format's definition and attention in 64 bits (oracle/int4.py)."""

import math

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import _lib, ops
from oracle import int4

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = 2.0 ** -11        # fp16: half a step, relative


def half(rng, *shape, spread=0.0):
    x = rng.standard_normal(shape)
    if spread:
        x = x * 10.0 ** rng.uniform(-spread, spread, shape[:-1] + (1,))
    return x.astype(np.float16)


def dev(x, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV, dtype) if dtype else torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def odd_rows(rng, n, h, d):
    """Rows of every kind: ordinary, of many sizes, offset, constant, empty, with outliers, saturating, infinite, not numbers, tiny, and
    rows on the borders between codes."""
    x = half(rng, n, h, d, spread=3.0)
    flat = x.reshape(n * h, d)
    kinds = [lambda r: r * 0, lambda r: r * 0 + np.float16(2.5), lambda r: r * 0 - np.float16(0.1), np.abs, lambda r: -np.abs(r),
             lambda r: np.where(np.arange(d) == 7, np.float16(1000.0), r), lambda r: np.where(np.arange(d) == 3, np.float16(65504.0), r),
             lambda r: np.where(np.arange(d) < 2, np.float16(np.inf) * np.array([1, -1] + [1] * (d - 2)), r),
             lambda r: np.where(np.arange(d) == d - 1, np.float16(np.nan), r), lambda r: (rng.integers(0, 40, d) * 6e-8),
             lambda r: rng.integers(-15, 16, d) * 0.25, lambda r: rng.integers(-15, 16, d) * 0.5 * 1.09375,
             lambda r: np.concatenate([[7.5, -7.5], rng.integers(-15, 16, d - 2) * 0.5])]
    with np.errstate(invalid="ignore"):
        for i in range(min(len(flat), 3 * len(kinds))):
            flat[i] = kinds[i % len(kinds)](flat[i]).astype(np.float16)
    return x


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv,tokens", [(1, 1), (2, 5), (8, 33), (3, 70), (8, 300)])
def test_append_stores_the_bytes_of_the_definition(d, hkv, tokens):
    rng = np.random.default_rng(d + tokens)
    slots_all = -(-max(64, 2 * tokens) // 16) * 16
    pool = rng.integers(0, 256, (slots_all, 2 * hkv, d // 2 + 2), dtype=np.uint8)
    k, v = odd_rows(rng, tokens, hkv, d), odd_rows(rng, tokens, hkv, d)[::-1].copy()
    slots = rng.permutation(slots_all)[:tokens].astype(np.int64)
    if tokens > 4:
        slots[1], slots[3], slots[4] = -1, slots_all, 2 ** 31 - 1
    got = dev(pool)
    kv = dev(np.concatenate([k, v], 1))      # the two halves of one tensor: strides of their own
    ops.kv_append_quantised(kv[:, :hkv], kv[:, hkv:], dev(slots, torch.int32), got)
    int4.store(pool, slots, k, v)
    assert np.array_equal(got.cpu().numpy(), pool)


@pytest.mark.parametrize("d,hkv,page", [(64, 1, 16), (64, 8, 64), (128, 1, 32), (128, 8, 16), (128, 3, 256)])
def test_dequant_gives_the_values_and_pages_move_as_bytes(d, hkv, page):
    rng = np.random.default_rng(page)
    pages = 7
    pool = np.zeros((pages * page, 2 * hkv, d // 2 + 2), dtype=np.uint8)
    rows = odd_rows(rng, pages * page, 2 * hkv, d)
    int4.store(pool, np.arange(pages * page), rows[:, :hkv], rows[:, hkv:])
    values, _ = int4.decode_pool(pool, hkv, d)
    src, ids, out_ids = dev(pool), np.array([4, 0, 9, 6, -1, 2]), np.array([1, 3, 0, 5, 2, 7])
    dst = torch.full((6 * page, 2 * hkv, d), 7.0, dtype=torch.float16, device=DEV)
    ops.page_dequant(src, dst, dev(ids, torch.int32), dev(out_ids, torch.int32), None, page)
    want = np.full((6, page, 2 * hkv, d), 7.0)
    for i, o in ((4, 1), (0, 3), (6, 5)):    # pages 9 and -1, and place 7, are outside
        want[o] = values.reshape(pages, page, 2 * hkv, d)[i]
    assert np.array_equal(dst.cpu().numpy().reshape(want.shape).astype(np.float64), want)
    ops.page_dequant(src, dst, dev(np.array([5, 1]), torch.int32), None, None, page)
    want[0], want[1] = values.reshape(want[0:0].shape[:0] + (pages, page, 2 * hkv, d))[[5, 1]]
    assert np.array_equal(dst.cpu().numpy().reshape(want.shape).astype(np.float64), want)

    ops.page_copy(src, dev(np.array([1, 2]), torch.int32), dev(np.array([5, 0]), torch.int32), page)
    pool = pool.reshape(pages, -1)
    pool[[5, 0]] = pool[[1, 2]]
    assert np.array_equal(src.cpu().numpy().reshape(pages, -1), pool)
    other = torch.zeros_like(src)
    ops.page_gather(src, other, dev(np.array([6, 3]), torch.int32), None, page)
    assert np.array_equal(other.cpu().numpy().reshape(pages, -1)[:2], pool[[6, 3]])


def epilogue64(x, weight, cos, sin, eps):
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight.astype(np.float64)
    if cos is not None:
        a, b = np.split(x, 2, -1)
        c, s = cos.astype(np.float64)[:, None], sin.astype(np.float64)[:, None]
        x = np.concatenate([a * c - b * s, b * c + a * s], -1)
    return x


@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("hq,hkv,d,tokens", [(4, 1, 64, 1), (32, 8, 64, 77), (16, 8, 128, 9), (5, 5, 128, 40), (64, 8, 128, 700)])
def test_epilogue_norm_rotation_and_append(hq, hkv, d, tokens, norm, rope):
    rng = np.random.default_rng(tokens + hq)
    slots_all = -(-max(64, tokens + 40) // 16) * 16
    pool = rng.integers(0, 256, (slots_all, 2 * hkv, d // 2 + 2), dtype=np.uint8)
    q, k, v = half(rng, tokens, hq, d, spread=1.0), half(rng, tokens, hkv, d, spread=1.0), odd_rows(rng, tokens, hkv, d)
    qw, kw = (half(rng, d), half(rng, d, spread=0.0) + np.float16(1)) if norm else (None, None)
    cos = sin = None
    if rope:
        angle = rng.uniform(0, 6.3, (tokens, d // 2))
        cos, sin = (np.concatenate([f(angle)] * 2, -1).astype(np.float16) for f in (np.cos, np.sin))
    slots = rng.permutation(slots_all)[:tokens].astype(np.int64)
    if tokens > 5:
        slots[2] = -1
    got_q, got = dev(q), dev(pool)
    args = [dev(x) if x is not None else None for x in (qw, kw, cos, sin)]
    back = ops.qk_norm_rope_append(got_q, dev(k), dev(v), dev(slots, torch.int32), got, *args, 1e-5)
    assert back is got_q
    first = None if cos is None else cos[:, : d // 2]
    second = None if sin is None else sin[:, : d // 2]
    want_q = epilogue64(q, qw, first, second, np.float32(1e-5))
    # one rounding to fp16 (2^-25: half its smallest step); in front of it five fp32 roundings of the two products' sizes
    size = np.abs(epilogue64(np.abs(q), None if qw is None else np.abs(qw), None if first is None else np.abs(first),
                             None if second is None else -np.abs(second), np.float32(1e-5)))
    if rope:
        size = np.maximum(size, np.roll(size, d // 2, -1))
    assert (np.abs(got_q.cpu().numpy().astype(np.float64) - want_q) <= HALF * np.abs(want_q) + 2.0 ** -25 + 2.0 ** -21 * size).all()

    x = epilogue64(k, kw, first, second, np.float32(1e-5))
    kept = (slots >= 0)
    values, scales = int4.decode_pool(got.cpu().numpy(), hkv, d)
    held, s = values[slots[kept], :hkv], scales[slots[kept], :hkv]
    want_s, _ = int4.scale_of(x[kept])
    # fp32 moves an element by at most 2^-21 of its row's largest; a scale by a step of its 7 bits where it lies at the border
    most = np.abs(x[kept]).max(-1)
    assert (np.abs(s - want_s) <= want_s * 2.0 ** -6 * 1.01).all()
    assert ((s == want_s) | (np.abs(int4.scale_of(x[kept] * (1 + 2.0 ** -19))[0] - int4.scale_of(x[kept] * (1 - 2.0 ** -19))[0]) > 0)).all()
    # with s the held values are within half a step; and the zero point's own rounding may cost as much where the range is full
    assert (np.abs(held - x[kept]) <= (0.5 * s + 2.0 ** -20 * most)[..., None]).all()
    # V and everything else byte by byte
    code, vs, vz = int4.quantise(v[kept])
    assert np.array_equal(values[slots[kept], hkv:], vs[..., None] * (code - vz[..., None]))
    untouched = np.setdiff1d(np.arange(slots_all), slots[kept])
    before, _ = int4.decode_pool(pool, hkv, d)
    assert np.array_equal(values[untouched], before[untouched], equal_nan=True)


def test_rows_in_pool_do_not_depend_on_how_they_came():
    """The fused append stores what the append alone stores where there is nothing in between."""
    rng = np.random.default_rng(5)
    k, v, q = dev(odd_rows(rng, 40, 2, 128)), dev(odd_rows(rng, 40, 2, 128)), dev(half(rng, 40, 4, 128))
    slots = dev(rng.permutation(64)[:40], torch.int32)
    a, b = (torch.zeros(64, 4, 66, dtype=torch.uint8, device=DEV) for _ in range(2))
    ops.kv_append_quantised(k, v, slots, a)
    ops.qk_norm_rope_append(q, k, v, slots, b)
    assert torch.equal(a, b)


class Sequences:
    """Sequences of the given lengths in a pool whose unwritten bytes are poison (scales that are not numbers)."""

    def __init__(self, lens, hq, hkv, d, page, seed=0, spread=0.0, rows=None):
        rng = np.random.default_rng(seed)
        each = [-(-n // page) for n in lens]
        self.pages = sum(each) + 3
        order = rng.permutation(self.pages)
        self.table = rng.integers(-5, 2 * self.pages, (len(lens), max(1, max(each)) + 1)).astype(np.int32)
        at = 0
        for b, n in enumerate(each):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.pool = np.full((self.pages * page, 2 * hkv, d // 2 + 2), 255, dtype=np.uint8)
        self.lens, self.hq, self.hkv, self.d, self.page = lens, hq, hkv, d, page
        for b, n in enumerate(lens):
            if n:
                kv = half(rng, n, 2 * hkv, d, spread=spread) if rows is None else rows(rng, n, 2 * hkv, d)
                int4.store(self.pool, int4.tokens_of(self.table[b], n, page), kv[:, :hkv], kv[:, hkv:])
        self.rng = rng

    def values(self, b):
        values, _ = int4.decode_pool(self.pool, self.hkv, self.d)
        mine = values[int4.tokens_of(self.table[b], self.lens[b], self.page)]
        return mine[:, : self.hkv], mine[:, self.hkv:]


def score_error(q, k, scale):
    """What fp32 may move a score by (natural units): sums of d products of codes up to 15 steps and the zero point's share."""
    if k.shape[0] == 0:
        return 0.0
    d = q.shape[-1]
    step = np.abs(k).max(-1).max() / 7.0 + 1e-9        # at least 8 codes of the row lie on its larger side
    return 2.0 ** -24 * 6 * math.sqrt(d) * np.abs(q.astype(np.float64)).sum(-1).max() * 15 * step * scale


def check(got, q, seqs, rows_of, scale, p_error):
    """Every output within fp16's rounding, what fp32 may move the scores by, and `p_error` of the probabilities."""
    for b in range(len(seqs.lens)):
        rows, seen = rows_of(b)
        if len(rows) == 0:
            continue
        k, v = seqs.values(b)
        want, size = int4.attend(q[rows], k, v, scale, seen)
        off = np.abs(got[rows].astype(np.float64) - want)
        rel = 2 * (math.expm1(min(1.0, score_error(q[rows], k, scale))) + p_error) + 2.0 ** -18
        assert np.isfinite(got[rows]).all()
        allowed = HALF * np.abs(want) + 2.0 ** -25 + rel * (size + np.abs(want)) + 2.0 ** -24 * 16 * np.abs(v).max(initial=0.0)
        assert (off <= allowed).all(), (b, seqs.lens[b], float((off / allowed).max()))


LAYOUTS = [(8, 8, 64), (16, 8, 128), (8, 1, 128), (64, 8, 128), (12, 1, 64), (16, 1, 128), (40, 1, 128), (64, 1, 64), (6, 2, 64)]


@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
@pytest.mark.parametrize("page", [16, 64])
def test_decode(hq, hkv, d, page):
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 47, 48, 64, 65, 100, 257, 300, 0, 511]
    s = Sequences(lens, hq, hkv, d, page, seed=hq + d)
    q = half(s.rng, len(lens), hq, d)
    scale = 1.0 / math.sqrt(d)
    one = lambda b: ([b] if lens[b] else [], [lens[b]])  # noqa: E731
    for kw in (dict(), dict(num_splits=1), dict(num_splits=3), dict(num_splits=16), dict(max_splits=5, min_pages_per_split=2)):
        out = ops.paged_decode(dev(q), dev(s.pool), dev(s.table), dev(np.array(lens), torch.int32), scale, page_size=page, **kw)
        got = out.cpu().numpy()
        assert (got[[0, 15]] == 0).all()
        # p s' are kept to 2^-20 (two fp16 parts, each rounded toward zero)
        check(got, q, s, one, scale, 2.0 ** -19)


@pytest.mark.parametrize("page", [32, 128, 256])
def test_decode_page_sizes_and_long_rows(page):
    lens = [3000, 1, 700, 2049]
    s = Sequences(lens, 16, 2, 128, page, seed=page)
    q = half(s.rng, 4, 16, 128)
    out = ops.paged_decode(dev(q), dev(s.pool), dev(s.table), dev(np.array(lens), torch.int32), page_size=page)
    check(out.cpu().numpy(), q, s, lambda b: ([b], [lens[b]]), 1 / math.sqrt(128), 2.0 ** -19)


@pytest.mark.parametrize("kind", ["spread", "spikes", "zero_values", "one_big_value", "large_q", "tiny_q", "negative_scale"])
@pytest.mark.parametrize("d", [64, 128])
def test_decode_ranges(kind, d):
    """Scores and scales that grow, shrink and differ by many powers of two along a sequence."""
    lens = [5, 200, 333]

    def rows(rng, n, h2, d):
        x = half(rng, n, h2, d)
        h = h2 // 2
        if kind == "spread":
            x = half(rng, n, h2, d, spread=3.0)
            x[:, :h] = half(rng, n, h, d, spread=0.5)
        if kind == "spikes":
            for at in range(0, n, 23):
                x[at, :h] *= np.float16(1 + at / 20)
        if kind == "zero_values":
            x[:, h:] = 0
            x[::3, h:] = half(rng, len(x[::3]), h, d)
            x[1::5, :h] *= np.float16(6)
        if kind == "one_big_value":
            x[n // 2, h:] = half(rng, 1, h, d)[0] * np.float16(15000)
            x[n // 2, :h] = 0
        return x

    s = Sequences(lens, 8, 2, d, 16, seed=d, rows=rows)
    q = half(s.rng, 3, 8, d)
    scale = 1.0 / math.sqrt(d)
    if kind == "one_big_value":
        q = np.abs(q) * np.float16(1)
    if kind == "large_q":
        q = q * np.float16(300)
        scale /= 300
    if kind == "tiny_q":
        q = (q * np.float16(1e-4)).astype(np.float16)
        scale *= 1e4
    if kind == "negative_scale":
        scale = -scale
    for n in (1, 4):
        out = ops.paged_decode(dev(q), dev(s.pool), dev(s.table), dev(np.array(lens), torch.int32), scale, num_splits=n)
        check(out.cpu().numpy(), q, s, lambda b: ([b], [lens[b]]), abs(scale) if scale < 0 else scale, 2.0 ** -19) if scale > 0 else \
            check_signed(out.cpu().numpy(), q, s, lens, scale)


def check_signed(got, q, s, lens, scale):
    check(got, -q, s, lambda b: ([b], [lens[b]]), -scale, 2.0 ** -19)      # the same scores


def test_decode_not_a_number_stays_in_its_row():
    s = Sequences([40, 40], 4, 1, 128, 16)
    q = half(s.rng, 2, 4, 128)
    q[0, 1, 5] = np.nan
    q[0, 2, 6] = np.inf
    out = ops.paged_decode(dev(q), dev(s.pool), dev(s.table), dev(np.array([40, 40]), torch.int32)).cpu().numpy()
    assert np.isnan(out[0, 1]).all() and not np.isfinite(out[0, 2]).any()
    q[0, 1, 5] = q[0, 2, 6] = 0
    clean = ops.paged_decode(dev(q), dev(s.pool), dev(s.table), dev(np.array([40, 40]), torch.int32)).cpu().numpy()
    assert np.array_equal(out[0, [0, 3]], clean[0, [0, 3]]) and np.array_equal(out[1], clean[1])


def test_decode_lengths_and_pages_the_table_cannot_name():
    """A length beyond the row re-reads its last entry, page ids outside the pool are clamped, nothing is appended there."""
    s = Sequences([64, 20], 8, 2, 128, 16)
    s.table = np.ascontiguousarray(s.table[:, :4])
    s.table[1, 2:] = [10 ** 6, -7]
    q, k = half(s.rng, 2, 8, 128), half(s.rng, 2, 2, 128)
    pool = dev(s.pool)
    out = ops.paged_decode(dev(q), pool, dev(s.table), dev(np.array([1000, 20]), torch.int32), k_new=dev(k), v_new=dev(k))
    assert torch.isfinite(out[1]).all()
    int4.store(s.pool, int4.tokens_of(s.table[1], 20, 16)[-1:], k[1:], k[1:])
    assert np.array_equal(pool.cpu().numpy(), s.pool)
    s.lens = [64, 20]
    check(out.cpu().numpy(), q, s, lambda b: ([b] if b else [], [20]), 1 / math.sqrt(128), 2.0 ** -19)


@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 64), (20, 1, 128, 32), (4, 4, 64, 16)])
@pytest.mark.parametrize("splits", [None, 1, 8])
def test_decode_appends_on_the_way(hq, hkv, d, page, splits):
    lens = [1, 0, 16, 17, 32, 33, 129, 400]
    s = Sequences(lens, hq, hkv, d, page, seed=d)
    q, kv = half(s.rng, len(lens), hq, d), odd_rows(s.rng, len(lens), 2 * hkv, d)
    pool, both = dev(s.pool), dev(kv)
    kw = {} if splits is None else dict(num_splits=splits)
    out = ops.paged_decode(dev(q), pool, dev(s.table), dev(np.array(lens), torch.int32), page_size=page, k_new=both[:, :hkv],
                           v_new=both[:, hkv:], **kw)
    live = [b for b, n in enumerate(lens) if n]
    slots = [int4.tokens_of(s.table[b], lens[b], page)[-1] for b in live]
    int4.store(s.pool, slots, kv[live, :hkv], kv[live, hkv:])
    assert np.array_equal(pool.cpu().numpy(), s.pool)
    # rows of 10^3 times others' size: scores of thousands, and a bound to match
    check(out.cpu().numpy(), q, s, lambda b: ([b] if lens[b] else [], [lens[b]]), 1 / math.sqrt(d), 2.0 ** -19)


@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (64, 8, 128, 16), (32, 8, 64, 64), (8, 8, 64, 16), (12, 1, 128, 32),
                                           (40, 1, 64, 16)])
@pytest.mark.parametrize("rows,history", [([1], [0]), ([5, 1, 40, 0, 64, 33], [0, 3, 16, 9, 63, 100]), ([200, 130], [0, 0]),
                                          ([17, 300], [700, 5])])
def test_prefill(hq, hkv, d, page, rows, history):
    lens = [r + h if r else 0 for r, h in zip(rows, history)]
    s = Sequences(lens, hq, hkv, d, page, seed=hq + sum(rows))
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = half(s.rng, int(cu[-1]), hq, d)
    of = lambda b: (list(range(cu[b], cu[b + 1])), [history[b] + i + 1 for i in range(rows[b])])  # noqa: E731
    forms = [dict(), dict(max_kv_len=max(lens)), dict(key_slices=1)] + [dict(key_slices=n) for n in (2, 5)]
    for kw in forms:
        out = ops.paged_prefill(dev(q), dev(s.pool), dev(s.table), dev(cu, torch.int32), dev(np.array(history), torch.int32),
                                max(rows), 1 / math.sqrt(d), page_size=page, **kw)
        # probabilities as fp16, a half step each, in numerator and denominator; 2^-25 where they are small
        check(out.cpu().numpy(), q, s, of, 1 / math.sqrt(d), HALF + 2.0 ** -25 * max(lens))


def test_prefill_two_groups_and_wide_launches():
    """Launches of the other forms of the tile loop: two groups of wavefronts, and more workgroups than compute units."""
    for hq, hkv, d, rows, history in ((64, 8, 128, [512], [3000]), (32, 8, 64, [900], [2000]), (64, 8, 128, [300] * 6, [40] * 6)):
        lens = [r + h for r, h in zip(rows, history)]
        s = Sequences(lens, hq, hkv, d, 16, seed=d)
        cu = np.concatenate([[0], np.cumsum(rows)])
        q = half(s.rng, int(cu[-1]), hq, d)
        pick = [0, rows[0] // 2, rows[0] - 1]
        out = ops.paged_prefill(dev(q), dev(s.pool), dev(s.table), dev(cu, torch.int32), dev(np.array(history), torch.int32),
                                max(rows), 1 / math.sqrt(d), key_slices=1, max_kv_len=max(lens)).cpu().numpy()
        check(out, q, s, lambda b: ([cu[b] + i for i in pick], [history[b] + i + 1 for i in pick]), 1 / math.sqrt(d),
              HALF + 2.0 ** -25 * max(lens))


def test_runs_twice_to_the_same_bits():
    s = Sequences([900, 5, 333], 16, 4, 128, 16)
    q, lens = dev(half(s.rng, 3, 16, 128)), dev(np.array([900, 5, 333]), torch.int32)
    pool, table = dev(s.pool), dev(s.table)
    first = ops.paged_decode(q, pool, table, lens)
    for _ in range(3):
        assert torch.equal(first, ops.paged_decode(q, pool, table, lens))


def test_refusals_on_the_gpu():
    pool = torch.zeros(64, 4, 66, dtype=torch.uint8, device=DEV)
    q = torch.zeros(2, 4, 128, dtype=torch.float16, device=DEV)
    kv = torch.zeros(2, 2, 128, dtype=torch.float16, device=DEV)
    table, lens = torch.zeros(2, 4, dtype=torch.int32, device=DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    scales = torch.ones(4, device=DEV)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    bad = [
        lambda: ops.kv_append_quantised(kv, kv, lens, pool, scales),                       # rows carry their own scales
        lambda: ops.kv_append(kv, kv, lens, pool),                                         # an fp16 operator
        lambda: ops.kv_append_quantised(kv[..., :64], kv[..., :64], lens, pool),           # another head dim
        lambda: ops.kv_append_quantised(kv, kv, lens[:1], pool),
        lambda: ops.kv_append_quantised(kv, kv, lens, pool[:40]),                          # not whole blocks
        lambda: ops.qk_norm_rope_append(q, kv, kv, lens, pool, kv_scales=scales),
        lambda: ops.page_dequant(pool, torch.zeros(64, 4, 128, dtype=torch.float16, device=DEV), lens, None, scales),
        lambda: ops.page_copy(pool, lens, lens, page_size=8),
        lambda: ops.paged_decode(q, pool, table, lens, kv_scales=scales),
        lambda: ops.paged_decode(q, pool, table, lens, schedule="balanced"),
        lambda: ops.paged_decode(q, pool, table, lens, shared_pages=1),
        lambda: ops.paged_decode(q, pool, table, lens, num_splits=2, stage="split"),
        lambda: ops.paged_decode(q, pool, table, lens, k_new=kv),
        lambda: ops.paged_decode(q[..., :64].contiguous(), pool, table, lens),
        lambda: ops.paged_decode(q.float(), pool, table, lens),
        lambda: ops.paged_prefill(q, pool, table, cu, None, 1, kv_scales=scales),
        lambda: ops.paged_prefill(q[..., :64].contiguous(), pool, table, cu, None, 1),
        lambda: ops.DecodePlan(table, lens, 4, 2, 4, shared_pages=2, kv_dtype=torch.uint4),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            raise AssertionError(f"call {i} was taken")


@pytest.mark.parametrize("hq,hkv,d,page,rows,history", [
    (64, 8, 128, 16, [300], [2000]), (64, 8, 128, 64, [1, 0, 333, 260], [500, 20, 0, 77]), (32, 8, 64, 64, [513, 400], [1000, 30]),
    (16, 2, 64, 256, [250, 1], [255, 256]), (48, 3, 128, 32, [129] * 5, [3, 700, 250, 251, 511])])
def test_prefill_with_keys_decoded_once(hq, hkv, d, page, rows, history):
    lib = _lib.load()
    lens = [r + h if r else 0 for r, h in zip(rows, history)]
    s = Sequences(lens, hq, hkv, d, page, seed=sum(rows))
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = half(s.rng, int(cu[-1]), hq, d)
    picks = [sorted({0, r // 2, max(0, r - 2), r - 1}) if r else [] for r in rows]
    of = lambda b: ([cu[b] + i for i in picks[b]], [history[b] + i + 1 for i in picks[b]])  # noqa: E731
    args = (dev(q), dev(s.pool), dev(s.table), dev(cu, torch.int32), dev(np.array(history), torch.int32), max(rows), 1 / math.sqrt(d))
    p_error = HALF + 2.0 ** -25 * max(lens)
    for slices in (1, 3):
        need = lib.litekv_paged_prefill_int4_workspace_bytes(len(rows), hq, hkv, d, max(rows), max(lens), len(q), slices) // 4
        least = ops.paged_prefill_workspace_floats(len(q), hq, d, slices) if slices > 1 else 4
        assert need > least + sum(lens) * hkv * d
        outs = []
        for floats in (need, least):           # decoded once; where they are attended
            room = torch.full((floats,), math.nan, device=DEV)
            out = ops.paged_prefill(*args, page_size=page, key_slices=slices, max_kv_len=max(lens), workspace=room)
            check(out.cpu().numpy(), q, s, of, 1 / math.sqrt(d), p_error)
            outs.append(out)
        again = torch.full((need,), math.nan, device=DEV)
        assert torch.equal(outs[0], ops.paged_prefill(*args, page_size=page, key_slices=slices, max_kv_len=max(lens), workspace=again))
    out = ops.paged_prefill(*args, page_size=page, max_kv_len=max(lens) + 300)     # the lengths need only be bounded
    check(out.cpu().numpy(), q, s, of, 1 / math.sqrt(d), p_error)


@pytest.mark.parametrize("d", [64, 128])
def test_native_calls_and_wrappers_agree(d):
    """A plain call goes through native code, one with an argument of its own through the wrapper's."""
    lens = [70, 1, 0, 333]
    s = Sequences(lens, 16, 4, d, 16, seed=d)
    q, kv = dev(half(s.rng, 4, 16, d)), dev(half(s.rng, 4, 8, d))
    table, n = dev(s.table), dev(np.array(lens), torch.int32)
    pools = [dev(s.pool) for _ in range(2)]
    out = ops.paged_decode(q, pools[0], table, n, k_new=kv[:, :4], v_new=kv[:, 4:])
    mine = torch.empty_like(q)
    ops.paged_decode(q, pools[1], table, n, k_new=kv[:, :4], v_new=kv[:, 4:], out=mine)
    assert torch.equal(out, mine) and torch.equal(*pools)
    slots = dev(np.array([3, -1, 40, 17]), torch.int32)
    ops.kv_append_quantised(kv[:, :4], kv[:, 4:], slots, pools[0])
    ops.kv_append_quantised(kv[:, :4], kv[:, 4:], slots.long(), pools[1])       # (int64 slots: the wrapper converts them)
    assert torch.equal(*pools)
    a, b = (torch.full((s.pool.shape[0], 8, d), 3.0, dtype=torch.float16, device=DEV) for _ in range(2))
    ids = torch.arange(s.pages, dtype=torch.int32, device=DEV).flip(0).contiguous()
    ops.page_dequant(pools[0], a, ids, None, None)
    ops.page_dequant(pools[0], b, ids.long(), None, None)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_prefill_that_was_told_of_too_few_keys():
    """Keys decoded once, for the most keys the caller named: a longer sequence's rows are not numbers, the others' are right."""
    hq, hkv, d, rows, history = 64, 8, 128, [300, 280], [900, 100]
    lens = [1200, 380]
    s = Sequences(lens, hq, hkv, d, 16, seed=9)
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = half(s.rng, 580, hq, d)
    out = ops.paged_prefill(dev(q), dev(s.pool), dev(s.table), dev(cu, torch.int32), dev(np.array(history), torch.int32), 300,
                            1 / math.sqrt(d), max_kv_len=1000).cpu().numpy()
    assert np.isnan(out[:300]).all()
    s.lens = [0, 380]
    check(out, q, s, lambda b: ([300, 301, 440, 579], [101, 102, 241, 380]) if b else ([], []), 1 / math.sqrt(d),
          HALF + 2.0 ** -25 * 380)


def test_a_pool_of_more_than_4_gib():
    """The last pages of a large pool give what the first pages of a small one give."""
    hq, hkv, d, rows = 64, 8, 128, 300
    small = torch.zeros(64 * 16, 2 * hkv, 66, dtype=torch.uint8, device=DEV)
    large = torch.zeros((5 << 30) // (2 * hkv * 66) // 16 * 16, 2 * hkv, 66, dtype=torch.uint8, device=DEV)
    shift = large.shape[0] // 16 - 64
    rng = np.random.default_rng(3)
    k, v, q = (dev(half(rng, 900, h, d)) for h in (hkv, hkv, hq))
    table = dev(rng.permutation(64)[:57].reshape(1, -1), torch.int32)
    slots = (table[0].long()[:, None] * 16 + torch.arange(16, device=DEV)).reshape(-1)[:900].to(torch.int32)
    outs = []
    for pool, pages in ((small, 0), (large, shift)):
        at = slots + 16 * pages
        ops.kv_append_quantised(k[:450], v[:450], at[:450].contiguous(), pool)
        q_in = q[450:].clone()
        ops.qk_norm_rope_append(q_in, k[450:], v[450:], at[450:].contiguous(), pool)
        t, n = table + pages, torch.tensor([900], dtype=torch.int32, device=DEV)
        values = torch.empty(57 * 16, 2 * hkv, d, dtype=torch.float16, device=DEV)
        step = ops.paged_decode(q[:1], pool, t, n, k_new=k[7:8], v_new=v[7:8])
        ops.page_dequant(pool, values, t[0].contiguous(), None, None)
        cu = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
        ctx = torch.tensor([600], dtype=torch.int32, device=DEV)
        chunk = ops.paged_prefill(q[:rows], pool, t, cu, ctx, rows, 0.1, max_kv_len=900)
        direct = ops.paged_prefill(q[:rows], pool, t, cu, ctx, rows, 0.1)
        outs.append((step, values[:900], chunk, direct, pool[16 * pages:16 * pages + 1024]))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert large[: 16 * shift].any() == False  # noqa: E712


@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 64), (12, 1, 128, 32), (32, 2, 64, 16)])
def test_a_new_token_in_every_row_of_its_block(hq, hkv, d, page):
    """The wavefront that attends the last block has the new token in registers: every row of a block, blocks of every place."""
    lens = list(range(1, 52)) + [256 + n for n in (1, 2, 7, 10, 16)] + [2048 + n for n in (0, 4, 11)]
    s = Sequences(lens, hq, hkv, d, page, seed=hq)
    q, kv = half(s.rng, len(lens), hq, d), half(s.rng, len(lens), 2 * hkv, d)
    kv[:, :, 5] *= 4.0                     # (so that a row's element somewhere else would show)
    kv[:, hkv:, d - 9] *= -3.0
    both, slots = dev(kv), [int4.tokens_of(s.table[b], n, page)[-1] for b, n in enumerate(lens)]
    pools = [dev(s.pool) for _ in range(2)]
    args = dev(s.table), dev(np.array(lens), torch.int32), 1 / math.sqrt(d)
    for kw in (dict(), dict(num_splits=4)):
        out = ops.paged_decode(dev(q), pools[0], *args, page_size=page, k_new=both[:, :hkv], v_new=both[:, hkv:], **kw)
        ops.kv_append_quantised(both[:, :hkv], both[:, hkv:], dev(np.array(slots), torch.int32), pools[1])
        assert torch.equal(out, ops.paged_decode(dev(q), pools[1], *args, page_size=page, **kw))
        assert torch.equal(*pools)
        pools[0].copy_(dev(s.pool)), pools[1].copy_(dev(s.pool))
    int4.store(s.pool, slots, kv[:, :hkv], kv[:, hkv:])
    check(out.cpu().numpy(), q, s, lambda b: ([b], [lens[b]]), 1 / math.sqrt(d), 2.0 ** -19)


def test_epilogue_of_rows_that_are_not_finite():
    """An infinite element makes its row's norm infinite: it is not a number itself (nor is what the rotation mixes it into), the others
    are 0; a NaN makes the whole row NaN. In the pool NaN counts as 0."""
    rng = np.random.default_rng(4)
    d, hq, hkv, t = 128, 4, 2, 6
    q, k, v = half(rng, t, hq, d), half(rng, t, hkv, d), half(rng, t, hkv, d)
    q[1, 2, 5], q[2, 1, 100], q[3, 0, 9] = np.inf, -np.inf, np.nan
    k[1, 0, 70], k[2, 1, 3], k[4, 0, 0] = np.inf, np.nan, -np.inf
    w = half(rng, 2, d) + np.float16(2)
    angle = rng.uniform(0, 6, (t, d // 2))
    cos, sin = (np.concatenate([f(angle)] * 2, -1).astype(np.float16) for f in (np.cos, np.sin))
    pool, got = torch.full((16, 2 * hkv, 66), 255, dtype=torch.uint8, device=DEV), dev(q)
    ops.qk_norm_rope_append(got, dev(k), dev(v), torch.arange(t, dtype=torch.int32, device=DEV), pool, dev(w[0]), dev(w[1]), dev(cos),
                            dev(sin), 1e-6)

    def epilogue(x, weight):
        with np.errstate(invalid="ignore"):
            x = x.astype(np.float64)
            y = x * (1 / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)) * weight.astype(np.float64)
            turned = np.concatenate([-y[..., d // 2:], y[..., :d // 2]], -1)
            return y * cos[:, None].astype(np.float64) + turned * sin[:, None].astype(np.float64)

    want, got = epilogue(q, w[0]), got.cpu().numpy()
    assert np.array_equal(np.isnan(want), np.isnan(got)) and np.isnan(want).sum() == 4 + d
    ok = ~np.isnan(want)
    # one rounding to fp16 and a few of fp32
    assert (np.abs(got[ok] - want[ok]) <= HALF * np.abs(want[ok]) + 2.0 ** -25 + 2.0 ** -20 * np.abs(want[ok]).max()).all()
    values, _ = int4.decode_pool(pool.cpu().numpy(), hkv, d)
    k_want = np.nan_to_num(epilogue(k, w[1]))
    span = np.maximum(k_want.max(-1), 0) - np.minimum(k_want.min(-1), 0)
    # half a step, the scale's rounding to 7 bits, an element next to a border
    assert (np.abs(values[:t, :hkv] - k_want) <= (span * (0.5 / 15) * (1 + 2.0 ** -6) + 1e-5 * np.abs(k_want).max() + 2.0 ** -20)[..., None]).all()
    assert (values[[1, 2, 4], [0, 1, 0]] == 0).all()


@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (32, 2, 64)])
def test_decode_of_a_query_that_is_not_finite(hq, hkv, d):
    """Its head's outputs are not numbers; every other head's and sequence's are what they are without it."""
    lens = [40, 700, 33]
    s = Sequences(lens, hq, hkv, d, 16, seed=d)
    q = half(s.rng, 3, hq, d)
    args = dev(s.pool), dev(s.table), dev(np.array(lens), torch.int32)
    want = ops.paged_decode(dev(q), *args).cpu().numpy()
    bad = [(0, 3, np.inf), (1, hq - 1, np.nan), (1, 0, -np.inf)]
    for b, h, x in bad:
        q[b, h, 7] = x
    got = ops.paged_decode(dev(q), *args).cpu().numpy()
    for b, h, _ in bad:
        assert np.isnan(got[b, h]).all()
        got[b, h] = want[b, h]
    assert np.array_equal(got, want)


@pytest.mark.parametrize("d", [64, 128])
def test_a_plan_s_steps_native_and_through_the_wrapper(d):
    lens = [1500, 3, 0, 2600]
    s = Sequences(lens, 8, 2, d, 16, seed=d)
    q, kv = dev(half(s.rng, 4, 8, d)), dev(half(s.rng, 4, 4, d))
    table, n = dev(s.table), dev(np.array(lens), torch.int32)
    for splits in (1, 2, 16):
        pools = [dev(s.pool) for _ in range(2)]
        plan = ops.DecodePlan(table, n, 8, 2, s.pages, kv_dtype=torch.uint4)
        plan.set_schedule(splits)
        out = ops.decode_step(q, pools[0], plan, kv[:, :2], kv[:, 2:], 0.1)
        mine = torch.empty_like(q)
        assert ops.decode_step(q, pools[1], plan, kv[:, :2], kv[:, 2:], 0.1, out=mine) is mine
        assert torch.equal(out, mine) and torch.equal(*pools) and torch.isfinite(out).all()
        assert torch.equal(out, ops.decode_step(q, pools[0], plan, None, None, 0.1))
    with pytest.raises(_lib.LiteKVError):
        plan.split_workspace = plan.split_workspace[:64]
        ops.decode_step(q, pools[0], plan, None, None, 0.1)


def test_views_strides_and_alignment():
    """Columns of a wider block table, 64-bit lengths, rows of a fused projection; rows that are not 16-byte aligned are refused."""
    hq, hkv, d = 16, 4, 128
    lens = [300, 17, 0, 64]
    s = Sequences(lens, hq, hkv, d, 16, seed=2)
    wide = np.full((4, s.table.shape[1] + 9), 7, np.int32)
    wide[:, 4:4 + s.table.shape[1]] = s.table
    table = dev(wide)[:, 4:4 + s.table.shape[1]]
    fused = dev(half(s.rng, 4, hq + 2 * hkv + 1, d))
    q, k, v = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:hq + 2 * hkv]
    n32, n64 = dev(np.array(lens), torch.int32), dev(np.array(lens), torch.int64)
    pools = [dev(s.pool) for _ in range(3)]
    want = ops.paged_decode(q.contiguous(), pools[0], dev(s.table), n32, k_new=k.contiguous(), v_new=v.contiguous())
    assert torch.equal(want, ops.paged_decode(q, pools[1], table, n64, k_new=k, v_new=v)) and torch.equal(pools[0], pools[1])
    plan = ops.DecodePlan(table, n64, hq, hkv, s.pages, kv_dtype=torch.uint4)
    assert torch.allclose(want.float(), ops.decode_step(q, pools[2], plan, k, v).float(), atol=2e-3, rtol=1e-2)
    assert torch.equal(pools[0], pools[2])
    cu, ctx = torch.tensor([0, 2, 3, 3, 4], device=DEV), torch.tensor([298, 16, 0, 63], device=DEV)
    chunk = ops.paged_prefill(q, pools[0], table, cu, ctx, 2)
    assert torch.equal(chunk, ops.paged_prefill(q.contiguous(), pools[0], dev(s.table), cu.int(), ctx.int(), 2))
    odd = torch.zeros(4 * hq * d + 4, dtype=torch.float16, device=DEV)[4:].view(4, hq, d)
    with pytest.raises(_lib.LiteKVError, match="aligned"):
        ops.paged_decode(odd, pools[0], table, n32)
    with pytest.raises((_lib.LiteKVError, ValueError)):
        ops.kv_append_quantised(odd[:, :hkv], odd[:, :hkv], n32, pools[0])
