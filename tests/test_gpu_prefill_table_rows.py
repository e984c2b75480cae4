"""Paged prefill over block tables that are views of wider ones: a length beyond what a row can name re-reads the row's last entry, and
no row reaches past the tensor's storage."""

import pytest
import torch

from llama_lite_npu_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
VIEWS = {"one row": (slice(1, 2), slice(3, 6)), "the last row": (slice(5, 6), slice(17, 20)), "rows to the end": (slice(4, 6), slice(17, 20)),
         "columns": (slice(0, 3), slice(0, 4))}


@pytest.mark.parametrize("fmt", ["fp16", "int8", "int4"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("view", list(VIEWS))
def test_lengths_beyond_the_row(fmt, d, view):
    hq, hkv, page = 32, 2, 16
    g = torch.Generator(device=DEV).manual_seed(d)
    randn = lambda *s: torch.randn(s, generator=g, device=DEV).half()  # noqa: E731
    wide = torch.randperm(120, generator=g, device=DEV).to(torch.int32).view(6, 20)
    table = wide[VIEWS[view]]
    b, width = table.shape
    kv = randn(120 * page, 2 * hkv, d)
    scales = None
    pool = kv
    if fmt != "fp16":
        shape, dtype = ((120 * page, 2 * hkv, d // 2 + 2), torch.uint8) if fmt == "int4" else (kv.shape, torch.int8)
        pool = torch.zeros(shape, dtype=dtype, device=DEV)
        scales = None if fmt == "int4" else torch.full((2 * hkv,), 0.03, device=DEV)
        ops.kv_append_quantised(kv[:, :hkv], kv[:, hkv:], torch.arange(120 * page, dtype=torch.int32, device=DEV), pool, scales)
    rows = 150
    history = [9 * page + 5] * b                     # the pages that the row does not name: its last one again
    cu = torch.arange(b + 1, dtype=torch.int32, device=DEV) * rows
    q, ctx = randn(rows * b, hq, d), torch.tensor(history, dtype=torch.int32, device=DEV)
    pages = -(-(history[0] + rows) // page)
    spelled = torch.cat([table, table[:, -1:].expand(b, pages - width)], 1).contiguous()
    for kw in (dict(), dict(max_kv_len=history[0] + rows), dict(key_slices=2), dict(out=torch.empty_like(q))):
        want = ops.paged_prefill(q, pool, spelled, cu, ctx, rows, 0.1, kv_scales=scales, page_size=page,
                                 **{k: torch.empty_like(q) if k == "out" else x for k, x in kw.items()})
        got = ops.paged_prefill(q, pool, table, cu, ctx, rows, 0.1, kv_scales=scales, page_size=page, **kw)
        assert torch.isfinite(got).all() and torch.equal(got, want), kw
