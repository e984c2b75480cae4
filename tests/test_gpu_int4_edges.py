"""4-bit pools where a call can go wrong without showing it: page ids that name no page, queries with a large channel, rows
behind the last sequence."""

import math

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import ops
from oracle import int4
from tests.test_gpu_int4 import DEV, HALF, Sequences, check, dev, half

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 64), (40, 1, 128, 32), (12, 1, 64, 16)])
@pytest.mark.parametrize("splits", [None, 1, 4])
def test_nothing_is_appended_through_an_id_that_names_no_page(hq, hkv, d, page, splits):
    """The entry that holds a sequence's last token names no page of the pool: no row of any page changes for it, and the other
    sequences' rows are stored and attended as ever."""
    lens = [33, 70, 1, 129, 600, 16, 257]
    s = Sequences(lens, hq, hkv, d, page, seed=hq + page)
    for b, entry in ((0, -1), (1, s.pages), (2, -2 ** 31), (3, 2 ** 31 - 1), (4, s.pages + 5)):
        s.table[b, (lens[b] - 1) // page] = entry
    q, kv = half(s.rng, len(lens), hq, d), half(s.rng, len(lens), 2 * hkv, d)
    good = [5, 6]
    slots = [int4.tokens_of(s.table[b], lens[b], page)[-1] for b in good]
    # (the first and the last page are where an id brought into range would lead: they hold rows of other sequences)
    want = s.pool.copy()
    int4.store(want, slots, kv[good, :hkv], kv[good, hkv:])
    both, n = dev(kv), dev(np.array(lens), torch.int32)
    kw = {} if splits is None else dict(num_splits=splits)
    pool = dev(s.pool)
    out = ops.paged_decode(dev(q), pool, dev(s.table), n, page_size=page, k_new=both[:, :hkv], v_new=both[:, hkv:], **kw).cpu().numpy()
    assert np.array_equal(pool.cpu().numpy(), want)
    stepped = dev(s.pool)
    plan = ops.DecodePlan(dev(s.table), n, hq, hkv, s.pages, page_size=page, kv_dtype=torch.uint4)
    plan.set_schedule(splits or 2)
    ops.decode_step(dev(q), stepped, plan, both[:, :hkv], both[:, hkv:])
    assert np.array_equal(stepped.cpu().numpy(), want)
    s.pool = want
    check(out, q, s, lambda b: ([b], [lens[b]]) if b in good else ([], []), 1 / math.sqrt(d), 2.0 ** -19)


@pytest.mark.parametrize("hq,hkv,d", [(16, 4, 128), (16, 4, 64), (12, 1, 128), (12, 1, 64)])
@pytest.mark.parametrize("large", [100.0, 1000.0, 30000.0])
def test_a_large_channel_of_q_leaves_the_others_their_bits(hq, hkv, d, large):
    """One channel of q is hundreds of times the others, as in models without norms of q and k, and K is small there: scores are made by
    the small elements, every one of which is an error of the same sign if it is held relative to the row's largest."""
    lens = [2, 3, 17, 40, 300]
    at = d // 3

    def rows(rng, n, h2, d):
        x = half(rng, n, h2, d)
        x[:, : h2 // 2] = np.float16(0.5) * rng.choice([-1.0, 1.0], (n, h2 // 2, 1))
        x[:, : h2 // 2, at] = 0
        return x

    s = Sequences(lens, hq, hkv, d, 16, seed=d, rows=rows)
    q = (np.ones((len(lens), hq, d)) * s.rng.uniform(0.05, 0.2, (len(lens), hq, 1))).astype(np.float16)
    q[..., at] = large
    scale = 1 / math.sqrt(d)
    for n in (1, 3):
        got = ops.paged_decode(dev(q), dev(s.pool), dev(s.table), dev(np.array(lens), torch.int32), scale, num_splits=n).cpu().numpy()
        for b, length in enumerate(lens):
            k, v = s.values(b)
            want, size = int4.attend(q[[b]], k, v, scale, [length])
            # a score: codes up to 15 steps of 0.5 / 15, whose products with q are summed in fp32. The row's own sum, times the zero
            # point, goes the same way. Three sums of 128 products and the zero point's: 2^-24 of the whole's size each, and 2^-27 of the
            # largest product for each one added to it
            codes = 0.5 * 1.02
            whole = codes * (large + 0.2 * d) * scale
            error = 2 * 2.0 ** -24 * 4 * whole + 2 * d * 2.0 ** -27 * codes * large * scale
            rel = 2 * (math.expm1(error) + 2.0 ** -19) + 2.0 ** -18
            allowed = HALF * np.abs(want) + 2.0 ** -25 + rel * (size + np.abs(want)) + 2.0 ** -20 * np.abs(v).max()
            off = np.abs(got[[b]].astype(np.float64) - want)
            assert (off <= allowed).all(), (b, n, float((off / allowed).max()))


@pytest.mark.parametrize("fmt", ["fp16", "int4"])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_behind_the_last_sequence_are_left_as_they_were(fmt, d):
    """A launch over key slices folds the rows that cu_q_lens names, whatever the tensors have behind them."""
    hq, hkv, rows, history, behind = 16, 4, [40, 25], [300, 700], 9
    lens = [r + h for r, h in zip(rows, history)]
    s = Sequences(lens, hq, hkv, d, 16, seed=d)
    cu = np.concatenate([[0], np.cumsum(rows)])
    q = half(s.rng, int(cu[-1]) + behind, hq, d)
    pool = dev(s.pool)
    if fmt == "fp16":
        values, _ = int4.decode_pool(s.pool, hkv, d)
        pool = dev(np.nan_to_num(values).astype(np.float16))
    args = dev(s.table), dev(cu, torch.int32), dev(np.array(history), torch.int32), max(rows), 1 / math.sqrt(d)
    for slices in (1, 2, 8):
        room = torch.full((ops.paged_prefill_workspace_floats(len(q), hq, d, max(2, slices)),), 77.0, device=DEV)
        out = torch.full((len(q), hq, d), 5.0, dtype=torch.float16, device=DEV)
        assert ops.paged_prefill(dev(q), pool, *args, out=out, key_slices=slices, workspace=room) is out
        assert (out[cu[-1]:] == 5.0).all(), slices
        check(out.cpu().numpy(), q, s, lambda b: (list(range(cu[b], cu[b + 1])), [history[b] + i + 1 for i in range(rows[b])]),
              1 / math.sqrt(d), HALF + 2.0 ** -25 * max(lens))
