"""Forms of the operators for requests with images that sizes choose between: the epilogue with all rows of a token in a workgroup,
and one row a sequence on the balanced schedule, from native code and from Python."""

import pytest
import torch

from llama_lite_npu_amd import ops
from tests.test_gpu_cross import DEV, _case, _want
from tests.test_gpu_image_requests import _both
from tests.test_gpu_mrope import _check, _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,d", [("int4", 64), ("int4", 128), ("fp8", 32), ("fp8", 64), ("fp8", 128), ("fp8", 256), ("int8", 32),
                                   ("int8", 256), ("fp16", 32), ("fp16", 256)])
@pytest.mark.parametrize("hq,hkv", [(16, 8), (7, 3), (5, 1)])
def test_epilogue_with_all_rows_of_a_token_in_a_workgroup(fmt, d, hq, hkv):
    """From 256 tokens on; lanes of one wavefront then go through rows of q, K and V side by side."""
    print(f"mrope forms: {fmt} D={d} {hq}/{hkv}", flush=True)
    side = 3 * d // 16
    for t, interleaved in ((256, True), (300, False)):
        s = _inputs(t + d + hq, t, hq, hkv, d, fmt)
        live = torch.ones(t, dtype=torch.bool, device=DEV)
        s["slots"][t // 2], s["slots"][3] = -1, s["pool"].shape[0] + 5
        live[t // 2] = live[3] = False
        _check(s, (d // 2 - 2 * side, side, side), interleaved, live)


@pytest.mark.parametrize("hq,hkv,d", [(64, 8, 128), (16, 8, 128), (32, 8, 64), (33, 1, 64)])
@pytest.mark.parametrize("fmt", ["fp16", "fp8", "int8"])
def test_one_row_a_sequence_on_the_balanced_schedule(hq, hkv, d, fmt, monkeypatch):
    print(f"cross forms: balanced {hq}/{hkv} D={d} {fmt}", flush=True)
    keys = [(37 * i) % 1300 for i in range(300)]
    c = _case([1] * 300, keys, hq, hkv, d, fmt, seed=4)
    for most in (None, 1299):
        assert ops._cross_splits(c["q"], c["pool"], c["table"], 16, most) == 0
        one, two = _both(monkeypatch, lambda: ops.paged_cross_attention(c["q"], c["pool"], c["table"], c["lens"], kv_scales=c["scales"],
                                                                        max_kv_len=most))
        assert torch.equal(one, two)
        want = _want(c)
        assert ((one.double() - want).abs() <= 2e-3 + 1e-2 * want.abs()).all()          # the decode kernels' bound
