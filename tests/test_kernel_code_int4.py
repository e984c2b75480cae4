"""Registers of the kernels over 4-bit pools, as the compiler's notes in the built library state them; needs no GPU."""

import re

from tests.test_kernel_code import code_objects, metadata  # noqa: F401


def test_kernels_over_4_bit_codes_spill_nothing(metadata):  # noqa: F811
    """Nothing in scratch memory, and the wavefronts per SIMD that the kernels are written for: three of decode and of prefill at head
    dim 64 (168 registers of 512, in steps of 8), two of prefill at 128."""
    decode = {name: k for name, k in metadata.items() if "paged_decode_int4_kernel" in name}
    prefill = {name: k for name, k in metadata.items() if re.search(r"prefill_(tiled|two_group)_kernelILi1[01]E", name)}
    others = {name: k for name, k in metadata.items() if re.search(r"int4_(append|stage)_kernel|page_dequant_int4", name)}
    assert len(decode) == 4 and len(prefill) == 10 and len(others) == 6, (sorted(decode), sorted(prefill), sorted(others))
    for name, k in {**decode, **prefill, **others}.items():
        assert k[".vgpr_spill_count"] == 0 and k[".sgpr_spill_count"] == 0 and k[".private_segment_fixed_size"] == 0, name
    for name, k in decode.items():
        assert k[".vgpr_count"] <= 168, name
    for name, k in prefill.items():
        assert k[".vgpr_count"] <= (168 if "hd64" in name else 256), name
