"""4-bit pools where a call can go wrong without showing it: page ids that name no page."""

import math

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import ops
from oracle import int4
from tests.test_gpu_int4 import Sequences, check, dev, half

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
