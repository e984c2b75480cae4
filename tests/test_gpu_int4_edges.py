"""4-bit pools where a call can go wrong without showing it: page ids that name no page, queries with a large channel, rows
behind the last sequence, rows of every size under a bound for each head and key."""

import math

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import ops
from oracle import int4
from tests.test_gpu_int4 import DEV, HALF, Sequences, check, dev, half, odd_rows

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
            # a score: codes up to 15 steps of 0.5 / 15. Sums of their products with q, and of q's elements, times the zero point, in
            # fp32: four of them 2^-24 of the whole's size off each, and 2^-27 of the largest product for each one added to it
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


def bounded(q, k, v, k_scales, v_scales, scale):
    """One row q [Hq, D] over keys k, v [N, Hkv, D] with scales [N, Hkv]: the exact output, what a step may be off from it, and its size
    (sum p |v|), float64 [Hq, D].

    A key's score is its scale times a sum of codes up to 15 and elements of q, which are held to 2^-30 of their largest: two sums of
    products, made fp32 and added, the row's own sum (eleven additions), the zero point, three factors, the difference from the
    reference and the exponential, 2^-24 of the whole each: twenty at most. Scores off by e_i weigh a key by
    a factor between exp(-e_i) and exp(e_i); what is off alike for the heaviest key and another changes nothing. A weight times V's scale
    is kept to 2^-20; codes up to 15 and zero points are summed in fp32, 32 keys a step."""
    q = q.astype(np.float64)
    n, group = k.shape[0], q.shape[0] // k.shape[1]
    want, allowed, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    for h in range(q.shape[0]):
        kh, vh, ks, vs = k[:, h // group], v[:, h // group], k_scales[:, h // group], v_scales[:, h // group]
        x = kh @ q[h] * scale
        p = np.exp(x - x.max())
        p /= p.sum()
        error = ks * scale * 15 * 20 * 2.0 ** -24 * np.abs(q[h]).sum()
        error = np.minimum(error + error[p.argmax()], 700.0)
        error[p.argmax()] = 0.0
        want[h], size[h] = p @ vh, p @ np.abs(vh)
        moved = (p * np.expm1(error)) @ np.abs(vh - want[h]) / (p @ np.exp(-error))
        summed = 15 * ((n / 32 + 16) * 2.0 ** -24 * (p @ vs) + 2.0 ** -28 * (p * vs).max())
        allowed[h] = HALF * np.abs(want[h]) + 2.0 ** -25 + moved + 2.0 ** -18 * (size[h] + np.abs(want[h])) + summed
    return want, allowed, size


@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 64), (20, 1, 128, 32), (4, 4, 64, 16)])
@pytest.mark.parametrize("large", [None, 300.0])
def test_steps_over_rows_of_every_size(hq, hkv, d, page, large):
    """History and new rows of all kinds (constant, empty, with outliers, saturating, tiny), ordinary queries and ones with a large
    channel; the append on the way."""
    lens = [1, 2, 16, 17, 33, 129, 400]
    s = Sequences(lens, hq, hkv, d, page, seed=d + hq, rows=odd_rows)
    q, kv = half(s.rng, len(lens), hq, d), odd_rows(s.rng, len(lens), 2 * hkv, d)
    if large:
        q[..., 11] = large
    before, both = dev(s.pool), dev(kv)
    int4.store(s.pool, [int4.tokens_of(s.table[b], n, page)[-1] for b, n in enumerate(lens)], kv[:, :hkv], kv[:, hkv:])
    values, scales = int4.decode_pool(s.pool, hkv, d)
    for splits in (None, 1, 5):
        kw = {} if splits is None else dict(num_splits=splits)
        got = ops.paged_decode(dev(q), before, dev(s.table), dev(np.array(lens), torch.int32), page_size=page, k_new=both[:, :hkv],
                               v_new=both[:, hkv:], **kw).cpu().numpy()
        for b, n in enumerate(lens):
            at = int4.tokens_of(s.table[b], n, page)
            want, allowed, size = bounded(q[b], values[at, :hkv], values[at, hkv:], scales[at, :hkv], scales[at, hkv:], 1 / math.sqrt(d))
            off = np.abs(got[b].astype(np.float64) - want)
            assert (off <= allowed).all(), (b, n, splits, float((off / allowed).max()))
            # most outputs are bounded to a part of themselves: no other output would do
            assert (allowed < 0.5 * np.abs(want)).mean() > 0.25, (b, n)


@pytest.mark.parametrize("hq,hkv,d", [(16, 4, 128), (16, 4, 64), (12, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("large", [30.0, 1000.0, 20000.0])
def test_large_and_small_elements_of_q_meet_ordinary_rows(hq, hkv, d, large):
    """Products of a large element stand beside those of its neighbours in one sum, whose bits they must not cost."""
    lens = [2, 7, 40, 200]
    s = Sequences(lens, hq, hkv, d, 16, seed=hq + d)
    q = half(s.rng, len(lens), hq, d)
    for b in range(len(lens)):
        for h in range(hq):
            q[b, h, s.rng.integers(0, d, 1 + h % 3)] = large * s.rng.choice([-1.0, 1.0])
    values, scales = int4.decode_pool(s.pool, hkv, d)
    scale = 1.0 / (math.sqrt(d) * large)          # (so that more than one key counts)
    for n_splits in (1, 3):
        for factor in (1.0, 30.0):
            got = ops.paged_decode(dev(q), dev(s.pool), dev(s.table), dev(np.array(lens), torch.int32), scale * factor, num_splits=n_splits)
            for b, n in enumerate(lens):
                at = int4.tokens_of(s.table[b], n, 16)
                want, allowed, _ = bounded(q[b], values[at, :hkv], values[at, hkv:], scales[at, :hkv], scales[at, hkv:], scale * factor)
                off = np.abs(got[b].cpu().numpy().astype(np.float64) - want)
                assert (off <= allowed).all(), (b, n_splits, factor, float((off / allowed).max()))
