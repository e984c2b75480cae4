"""Sections of positions with several axes as a model's configuration may hold them."""

import numpy as np
import pytest

from llama_lite_npu_amd import ops


@pytest.mark.parametrize("kind", [np.int64, np.int32, np.uint8])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("sections", [(24, 20, 20), (0, 128), (40, 88)])
def test_whole_numbers_of_any_kind(kind, interleaved, sections):
    ops.axis_of_pair.cache_clear()
    got = ops.axis_of_pair(tuple(np.array(sections, dtype=kind)), 2 * sum(sections), interleaved)
    ops.axis_of_pair.cache_clear()
    assert got == ops.axis_of_pair(sections, 2 * sum(sections), interleaved)


@pytest.mark.parametrize("sections", [(True, 63), (np.float32(32), 32), ("32", 32), (None, 64), (np.int64(-1), 65)])
def test_anything_else_is_refused(sections):
    with pytest.raises(ValueError, match="sections"):
        ops.axis_of_pair(sections, 128)
