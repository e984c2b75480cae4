"""Block tables as the launch that decodes a prefill's 4-bit keys once reads them; needs no GPU."""

import subprocess
from pathlib import Path

import torch

from llama_lite_npu_amd import build


def test_only_entries_of_pages_that_a_sequence_has_are_read(tmp_path):
    """The launch goes over max_kv_len tokens of every sequence, rounded up to 256. A row of a view of a wider table ends with its
    sequence's pages, or with the storage."""
    csrc = Path(build.CSRC)
    source = tmp_path / "entry.hip"
    source.write_text('#include <cstdio>\n#include "common.h"\n#include "kv_int4.h"\n'
                      "int main() {\n  int p, s, n;\n  long long k;\n  while (scanf(\"%d %lld %d %d\", &p, &k, &s, &n) == 4)\n"
                      "    printf(\"%d\\n\", litekv::int4_stage_entry(p, k, s, n));\n}\n")
    subprocess.run([build._hipcc(), "--offload-arch=gfx950", "--offload-host-only", "-std=c++17", f"-I{csrc}", f"-I{csrc.parents[1] / 'include'}",
                    str(source), "-o", str(tmp_path / "entry")], check=True, capture_output=True)
    wide = torch.arange(6 * 20, dtype=torch.int32).view(6, 20)
    asked = []
    for table in (wide, wide[:, 13:], wide[5:6, 17:], wide[1:3, 4:9], wide[4:, 19:]):
        for shift in (0, 2, 4):
            width = table.shape[1] << shift                     # 16-token pages that a row's entries name
            for keys in (0, 1, 16, min(17, 16 * width), 16 * width - 15, 16 * width):
                asked += [(p, keys, shift, table.stride(0), table) for p in range(-1, (max(keys, 300) + 255) // 256 * 16)]
    lines = "\n".join("%d %d %d %d" % a[:4] for a in asked)
    out = subprocess.run([str(tmp_path / "entry")], input=lines, text=True, check=True, capture_output=True).stdout.split()
    for (p, keys, shift, stride, table), entry in zip(asked, map(int, out), strict=True):
        assert entry == (p >> shift if 0 <= 16 * p < keys else -1)
        assert entry < table.shape[1]
        last = table.storage_offset() + (table.shape[0] - 1) * stride + max(entry, 0)
        assert last < table.untyped_storage().nbytes() // 4
    # lengths beyond the row: the row's last entry
    out = subprocess.run([str(tmp_path / "entry")], input="7 1000 0 5\n7 1000 1 3\n62 1000 0 5", text=True, check=True,
                         capture_output=True).stdout.split()
    assert out == ["4", "2", "4"]
