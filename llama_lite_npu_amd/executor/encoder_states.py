"""An encoder's K and V for the requests of a batch (an image's or a clip's states), in pages of their own.

The reference has no cross attention; the layout is the decoder cache's (a pool per layer, pages named by a block table), so the
same appends fill it and the same formats hold it. The states of a request do not change while it is answered: they are stored
once, and what a step needs to know about them (block table, lengths, the plan of the single-row form) is made once, too.
"""

from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import ops


class EncoderStates:
    def __init__(self, lengths: Sequence[int], num_layers: int, num_kv_heads: int, head_dim: int, page_size: int = 16,
                 dtype: torch.dtype = torch.float16, device="cuda:0",
                 kv_scales: Optional[Sequence[torch.Tensor]] = None) -> None:
        """Room for ``lengths[b]`` states of sequence b (0: it has none). ``dtype`` as for the executor's pools: float16,
        float8_e4m3fn or int8 (with ``kv_scales``, float32 [2 * Hkv] a layer) or uint4."""
        self.lengths = [int(n) for n in lengths]
        if not self.lengths or min(self.lengths) < 0:
            raise ValueError("lengths must be whole numbers of states, one a sequence")
        self.page_size, self.num_kv_heads, self.head_dim = int(page_size), int(num_kv_heads), int(head_dim)
        each = [-(-n // self.page_size) for n in self.lengths]
        pages = max(1, sum(each))
        table = torch.zeros((len(each), max(1, max(each))), dtype=torch.int32)
        slots, first = [], 0
        for b, (n, own) in enumerate(zip(self.lengths, each)):
            table[b, :own] = torch.arange(first, first + own, dtype=torch.int32)
            slots.append(torch.arange(first * self.page_size, first * self.page_size + n, dtype=torch.int32))
            first += own
        self.block_table, self.slot_mapping = table.to(device), torch.cat(slots).to(device)
        self.kv_lens = torch.tensor(self.lengths, dtype=torch.int32, device=device)
        self.max_kv_len = max(self.lengths)
        int4 = dtype is ops.INT4_DTYPE
        row = ops.int4_row_bytes(head_dim) if int4 else head_dim
        shape = (pages * self.page_size, 2 * self.num_kv_heads, row)
        self.kv_buffer = [torch.zeros(shape, dtype=torch.uint8 if int4 else dtype, device=device) for _ in range(num_layers)]
        coded = dtype in (torch.float8_e4m3fn, torch.int8)
        if coded != (kv_scales is not None) or (coded and len(kv_scales) != num_layers):
            raise ValueError("kv_scales, one a layer, belong to pools of 8-bit codes")
        self.kv_scales = list(kv_scales) if coded else [None] * num_layers
        self._dtype, self._pages, self._plans = dtype, pages, {}
        self._graph_plans: dict = {}          # head count -> (capture, its plan), of the last capture

    def store(self, layer_index: int, xk: torch.Tensor, xv: torch.Tensor) -> None:
        """K and V [sum of the lengths, Hkv, D] of all sequences' states, one sequence after another."""
        pool = self.kv_buffer[layer_index]
        if pool.dtype is torch.float16:
            ops.kv_append(xk, xv, self.slot_mapping, pool)
        else:
            ops.kv_append_quantised(xk, xv, self.slot_mapping, pool, self.kv_scales[layer_index])

    def decode_plan(self, num_q_heads: int) -> ops.DecodePlan:
        """How a step of one row a sequence reads the states: made at its first call, and the same for every layer and step. Steps
        share its workspace, so they run one after the other (one stream). A graph gets a plan of its own, shared by its layers
        and made once at each of its replays: nothing has run while it is captured, and it may run beside other steps."""
        captured = ops.capture_id()
        if captured is None:
            plan = self._plans.get(num_q_heads)
        else:
            known, plan = self._graph_plans.get(num_q_heads, (None, None))
            plan = plan if known == captured else None
        if plan is None:
            row = 2 * self.num_kv_heads * (self.kv_buffer[0].shape[2] * self.kv_buffer[0].element_size())
            plan = ops.DecodePlan(self.block_table, self.kv_lens, num_q_heads, self.num_kv_heads, self._pages,
                                  page_size=self.page_size, host_seq_lens=self.lengths, token_bytes=row, kv_dtype=self._dtype)
            if captured is None:
                self._plans[num_q_heads] = plan
            else:
                self._graph_plans[num_q_heads] = captured, plan
        return plan
