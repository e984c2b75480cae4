"""4-bit pools in use: prompts, chunks, decode steps, shared pages and captured graphs through the executor, against attention in 64
bits on the decoded pool."""

import math

import numpy as np
import pytest
import torch

from llama_lite_npu_amd import ops
from llama_lite_npu_amd.attention import Attention
from llama_lite_npu_amd.executor import ModelExecutor
from oracle import int4
from tests import test_gpu_decode_graph as dg
from tests.test_gpu_int4 import HALF, score_error

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
LOG2E = 1.4426950408889634


def rows(tokens, heads, d, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn((tokens, heads, d), generator=g, device=DEV, dtype=torch.float16)


def executor(hq, hkv, d, layers=2, page=16, num_pages=96, max_seq_len=512):
    ex = ModelExecutor(num_layers=layers, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, num_pages=num_pages * 16 // page, page_size=page,
                       max_seq_len=max_seq_len, max_requests=8, device=DEV, dtype=torch.uint4)
    for pool in ex.kv_mem_manager.gpu_kv_buffer:
        pool.fill_(255)                    # scales that are not numbers
    return ex


def close(ex, layer, hq, hkv, d, q, out, table, lens, rows_of, p_error):
    """The rows of sequence b, which see rows_of(b)[1] keys, within fp16's rounding, fp32 scores and p_error."""
    page = ex.page_size
    values, _ = int4.decode_pool(ex.kv_mem_manager.gpu_kv_buffer[layer].cpu().numpy(), hkv, d)
    q, out, table = q.cpu().numpy(), out.cpu().numpy().astype(np.float64), table.cpu().numpy()
    assert np.isfinite(out).all()
    for b, n in enumerate(lens):
        at, seen = rows_of(b)
        mine = values[int4.tokens_of(table[b], n, page)]
        k, v = mine[:, :hkv], mine[:, hkv:]
        want, size = int4.attend(q[at], k, v, 1 / math.sqrt(d), seen)
        rel = 2 * (math.expm1(score_error(q[at], k, 1 / math.sqrt(d))) + p_error) + 2.0 ** -18
        allowed = HALF * np.abs(want) + 2.0 ** -25 + rel * (size + np.abs(want)) + 2.0 ** -20 * np.abs(v).max()
        assert (np.abs(out[at] - want) <= allowed).all(), (b, n)


@pytest.mark.parametrize("hq,hkv,d,page", [(16, 8, 128, 16), (8, 2, 64, 64), (12, 1, 128, 32)])
def test_prompts_chunks_steps_and_compaction(hq, hkv, d, page):
    ex = executor(hq, hkv, d, page=page)
    assert ex.kv_mem_manager.is_int4 and ex.atten_info.kv_scales[0] is None
    attn, scale = Attention(hq, hkv, d), 1 / math.sqrt(d)
    lens = [37, 16, 90, 5]
    ids = ex.reserve_paged_requests(lens)
    ex.activate_paged_packed_prefill_batch(ids, lens)
    info = ex.atten_info
    for layer in range(2):
        q, k, v = rows(sum(lens), hq, d, 10 + layer), rows(sum(lens), hkv, d, 20 + layer), rows(sum(lens), hkv, d, 30 + layer)
        out = attn.context_forward(q, k, v, info, layer, scale * LOG2E)
        # a fresh prompt attends to its own K and V; the pool takes the definition's bytes
        cu = np.concatenate([[0], np.cumsum(lens)])
        for b, n in enumerate(lens):
            kk, vv = (x[cu[b]:cu[b + 1]].cpu().numpy().astype(np.float64) for x in (k, v))
            want, size = int4.attend(q[cu[b]:cu[b + 1]].cpu().numpy(), kk, vv, scale, np.arange(1, n + 1))
            off = np.abs(out[cu[b]:cu[b + 1]].cpu().numpy() - want)
            # probabilities as fp16, a half step each, in numerator and denominator; scores in fp32
            assert (off <= HALF * np.abs(want) + 2.0 ** -25 + (2 * HALF + 2.0 ** -16) * (size + np.abs(want))).all()
        pool = np.full(tuple(ex.kv_mem_manager.gpu_kv_buffer[layer].shape), 255, np.uint8)
        int4.store(pool, info.cur_select_index.cpu().numpy(), k.cpu().numpy(), v.cpu().numpy())
        assert np.array_equal(ex.kv_mem_manager.gpu_kv_buffer[layer].cpu().numpy(), pool)
    # a later chunk of one request over its cached history
    ex.ensure_paged_request_capacity(ids[3], 5 + 40)
    ex.activate_paged_chunk_prefill_batch((ids[3],), [5], [30])
    for layer in range(2):
        q = rows(30, hq, d, 41 + layer)
        out = attn.context_forward(q, rows(30, hkv, d, 43 + layer), rows(30, hkv, d, 45 + layer), ex.atten_info, layer, scale * LOG2E)
        close(ex, layer, hq, hkv, d, q, out, ex.atten_info.block_table, [35], lambda b: (np.arange(30), np.arange(6, 36)),
              HALF + 2.0 ** -25 * 35)
    lens[3] = 35
    for step in range(18):
        ex.extend_paged_requests(ids)
        lens = [n + 1 for n in lens]
        assert ex.atten_info.decode_plan.int4 and ex.atten_info.seq_lens_i32.tolist() == lens
        for layer in range(2):
            q = rows(4, hq, d, 100 + 2 * step + layer)
            out = attn.token_forward(q, rows(4, hkv, d, 200 + 2 * step + layer), rows(4, hkv, d, 300 + step), ex.atten_info, layer, scale)
            close(ex, layer, hq, hkv, d, q, out, ex.atten_info.block_table, lens, lambda b: ([b], [lens[b]]), 2.0 ** -19)
    # pages move as bytes: free a request, compact, the same answers bit for bit
    ex.release_paged_request_ids((ids[1],))
    keep, q = (ids[0], ids[2], ids[3]), rows(3, hq, d, 999)
    ex.activate_paged_decode_batch(keep)
    before = attn.token_forward(q, None, None, ex.atten_info, 0, scale).clone()
    assert ex.compact_kv_pool()
    ex.activate_paged_decode_batch(keep)
    assert torch.equal(before, attn.token_forward(q, None, None, ex.atten_info, 0, scale))


def test_requests_that_share_a_system_prompt():
    """Cached pages in several block tables: read by all, written by none; a step has no shared-prefix form and needs none."""
    hq, hkv, d = 16, 8, 128
    ex = executor(hq, hkv, d, layers=1)
    attn, scale = Attention(hq, hkv, d), 1 / math.sqrt(d)
    system = tuple(range(2000, 2096))               # 6 full pages
    (a,) = ex.reserve_paged_requests([96])
    ex.activate_paged_packed_prefill_batch((a,), [96])
    attn.context_forward(rows(96, hq, d, 61), rows(96, hkv, d, 62), rows(96, hkv, d, 63), ex.atten_info, 0, scale * LOG2E)
    ex.store_paged_request_prefix(system, a, first_token_id=5)
    batch, lens = [a], [96]
    for i, extra in enumerate((20, 3)):
        req, matched, _ = ex.share_paged_prefix_from_cache(system + tuple(range(3000 + 100 * i, 3000 + 100 * i + extra)))
        assert matched == 96
        ex.ensure_paged_request_capacity(req, 96 + extra + 8)
        ex.activate_paged_chunk_prefill_batch((req,), [96], [extra])
        q = rows(extra, hq, d, 70 + i)
        out = attn.context_forward(q, rows(extra, hkv, d, 80 + i), rows(extra, hkv, d, 90 + i), ex.atten_info, 0, scale * LOG2E)
        close(ex, 0, hq, hkv, d, q, out, ex.atten_info.block_table, [96 + extra],
              lambda b: (np.arange(extra), 97 + np.arange(extra)), HALF + 2.0 ** -25 * 200)  # noqa: B023
        batch.append(req)
        lens.append(96 + extra)
    shared = ex.atten_info.block_table[0, :6].long()
    slots = (shared[:, None] * 16 + torch.arange(16, device=DEV)).reshape(-1)
    before = ex.kv_mem_manager.gpu_kv_buffer[0][slots].clone()
    for step in range(3):
        ex.extend_paged_requests(tuple(batch))
        lens = [n + 1 for n in lens]
        assert ex.atten_info.decode_plan.shared_pages == 0
        q = rows(3, hq, d, 95 + step)
        out = attn.token_forward(q, rows(3, hkv, d, 96 + step), rows(3, hkv, d, 97 + step), ex.atten_info, 0, scale)
        close(ex, 0, hq, hkv, d, q, out, ex.atten_info.block_table, lens, lambda b: ([b], [lens[b]]), 2.0 ** -19)
    assert torch.equal(before, ex.kv_mem_manager.gpu_kv_buffer[0][slots])


@pytest.mark.parametrize("lens", [[1, 17, 48, 100, 31], [1017, 3, 500, 1021]])
def test_decode_steps_replay_as_graphs(lens):
    """The epilogue with its append on even layers, the append fused into the decode launch on odd ones; the second batch outgrows a
    split on the way, which needs a graph of its own."""
    def build():
        ex = ModelExecutor(num_layers=dg.LAYERS, num_q_heads=dg.HQ, num_kv_heads=dg.HKV, head_dim=dg.D, num_pages=256, max_seq_len=1100,
                           max_requests=8, device=DEV, dtype=torch.uint4)
        for pool in ex.kv_mem_manager.gpu_kv_buffer:
            pool.fill_(255)
        ids = ex.reserve_paged_requests(lens)
        ex.activate_paged_packed_prefill_batch(ids, lens)
        for layer in range(dg.LAYERS):
            ops.kv_append_quantised(rows(sum(lens), dg.HKV, dg.D, 7 + layer), rows(sum(lens), dg.HKV, dg.D, 57 + layer),
                                    ex.atten_info.cur_select_index, ex.atten_info.kv_buffer[layer])
        return ex, ids

    (host, ids_h), (dev, ids_d) = build(), build()
    model_h, model_d = dg.TinyModel(max_pos=1200), dg.TinyModel(max_pos=1200)
    dev.attach_model(model_d, "qwen3")
    batch = dev.activate_device_decode_batch(ids_d, reserve_tokens=8)
    tok_h = tok_d = torch.arange(len(lens), device=DEV).reshape(-1, 1) % dg.VOCAB
    schedules = set()
    for step in range(40):
        out_h = dg._host_step(host, model_h, ids_h, tok_h)
        dev.extend_paged_requests(ids_d)
        out_d = dev.forward(tok_d)
        torch.cuda.synchronize()
        schedules.add((host.atten_info.decode_plan.splits, batch.decode_plan.splits))
        if host.atten_info.decode_plan.splits == batch.decode_plan.splits:
            assert torch.equal(out_h, out_d), f"step {step}"
        else:
            # another number of splits: the same keys in another order of summing (fp32), three layers of outputs rounded to fp16
            assert ((out_h - out_d).abs() <= 2 * dg.LAYERS * HALF * (out_h.abs() + 4)).all(), f"step {step}"
        tok_h = tok_d = dg._next_tokens(out_h)
    assert dev.graph_runner.fallback_count == 0 and dev.graph_runner.replay_count >= 37
    batch.check()
    assert all(torch.equal(a, b) for a, b in zip(host.kv_mem_manager.gpu_kv_buffer, dev.kv_mem_manager.gpu_kv_buffer)) or len(schedules) > 1


def test_captured_calls_on_another_stream_and_a_plan_in_two_graphs():
    """Append, decode with several splits and prefill captured on a side stream; two graphs that share a plan's workspace, replayed
    in turn with eager steps between."""
    hq, hkv, d, b, cap = 8, 4, 128, 3, 2048
    g = torch.Generator(device=DEV).manual_seed(1)
    pools = [torch.full((b * cap, 2 * hkv, 66), 255, dtype=torch.uint8, device=DEV) for _ in range(2)]
    table = torch.arange(b * cap // 16, dtype=torch.int32, device=DEV).view(b, -1).flip(1).contiguous()
    lens = torch.tensor([1900, 0, 1300], dtype=torch.int32, device=DEV)
    k, v = (torch.randn((1900 * 2, hkv, d), generator=g, device=DEV, dtype=torch.float16) for _ in range(2))
    at = torch.arange(1900, device=DEV)
    slots = torch.cat([table[i].long()[at // 16] * 16 + at % 16 for i in (0, 2)]).to(torch.int32)
    for i, pool in enumerate(pools):
        ops.kv_append_quantised(k if i == 0 else v, v if i == 0 else k, slots, pool)
    plan = ops.DecodePlan(table, lens, hq, hkv, b * cap // 16, kv_dtype=torch.uint4)
    assert plan.splits > 1
    qs = [torch.randn((b, hq, d), generator=g, device=DEV, dtype=torch.float16) for _ in range(4)]
    cu = torch.tensor([0, 400, 400, 460], dtype=torch.int32, device=DEV)
    ctx = torch.tensor([1500, 0, 1240], dtype=torch.int32, device=DEV)
    qp = torch.randn((460, hq, d), generator=g, device=DEV, dtype=torch.float16)

    def work(i, q):
        pool = pools[i]
        out = ops.decode_step(q, pool, plan, None, None, 0.1)
        chunk = ops.paged_prefill(qp, pool, table, cu, ctx, 400, 0.1, max_kv_len=1900)
        many = ops.paged_prefill(qp.repeat(1, 8, 1), pool, table, cu, ctx, 400, 0.1, max_kv_len=1900)
        return out, chunk, many

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        want = {(i, j): [x.clone() for x in work(i, q)] for i in range(2) for j, q in enumerate(qs)}
    side.synchronize()
    for (i, j), outs in want.items():
        assert (outs[0][1] == 0).all() and all(torch.isfinite(x).all() for x in outs)
        assert all(torch.equal(x, y) for x, y in zip(outs, work(i, qs[j])))
    q_in, graphs, outs = torch.zeros_like(qs[0]), [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(work(i, q_in))
        graphs.append(graph)
    for j, q in enumerate(qs):
        for i in range(2):
            q_in.copy_(q)
            graphs[i].replay()
            got = [x.clone() for x in outs[i]]
            work(1 - i, qs[3 - j])
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, want[i, j])), (i, j)
