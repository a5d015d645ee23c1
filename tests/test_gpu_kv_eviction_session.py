"""Eviction next to what else touches a cache: steps that append without accumulating, the page-ID allocator, the page table
and the block bookkeeping, and rotary positions that count on behind a compaction."""
import importlib
import types

import numpy as np
import pytest

from eviction_util import attention_weights, compacted, kept_positions, page_rows, softmax_rows, to_f64
from parity_util import assert_outputs_close, importlib_workloads, oracle_step
from test_gpu_kv_eviction import LAYERS, _assert_weights, _config

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 8, 2, 128, 16
runtime = importlib.import_module("psi-dec_amd.runtime")


def _step(psi, w, seed, contexts, q_lens, requests=None):
    """A step of requests of w (its table, slots and arena) whose contexts after the append are given."""
    wl = importlib_workloads(psi)
    requests = list(range(len(w.req_slots))) if requests is None else requests
    s = wl.make_workload(seed, contexts, HQ, HKV, D, psi.Dtype.Bfloat16, PAGE, q_lens=q_lens, shuffle_slots=False,
                         host_pages=False)
    s.layout, s.layer, s.page_ids, s.pages, s.num_pages = w.layout, w.layer, w.page_ids, w.pages, w.num_pages
    s.req_slots = np.asarray(w.req_slots, np.uint32)[requests]
    return s


def _plain(psi, device, s, pages, ids):
    """The step as a framework without eviction runs it (TiledQ): appends, attends, accumulates nothing."""
    dw = importlib_workloads(psi).DeviceWorkload(device, s, partition_tokens=128, f32_output=True, pages=pages, page_ids=ids,
                                                 variant=psi.GQASplitKVVariant.TiledQ(8, 16, 8))
    dw.step()
    return dw.output_f32()


def _accumulating(psi, device, s, pages, ids, acc, decay):
    dw = importlib_workloads(psi).DeviceWorkload(device, s, partition_tokens=64, f32_output=True, balanced=True, pages=pages,
                                                 page_ids=ids, variant=psi.GQASplitKVVariant.SingleQ(16, 256, 4))
    logits, m = psi.GQASplitKVSingleQLogits(device, dw.cfg, dw.kshape, int(s.context_lens.max())), dw.meta
    device.f32_output(True)
    dw.kernels.invoke_attend_weights_bucketed(
        dw.q, pages, m.d_req_slots, m.d_flat_token_indices, ids, m.d_kv_splits, m.d_cu_kv_splits, dw.scratch, logits,
        dw.output, acc, decay, s.layer, s.num_tokens, dw.shape.num_sdpa_map_task_templates, worker_cu=m.d_worker_cu,
        num_workers=m.num_workers, flat_k=dw.flat_k, flat_v=dw.flat_v, partial_row_index=m.d_partial_row_index)
    device.f32_output(False)
    return dw.output_f32()


def _used(s, shape):
    used = np.zeros(shape, bool)
    for r in range(len(s.req_slots)):
        p = np.arange(int(s.context_lens[r]))
        used[page_rows(s, r)[p // PAGE], :, p % PAGE] = True
    return used


def _check_accumulators(s, host_pages, held, decay, before, after, what):
    exp, bound = attention_weights(s, host_pages, held, decay, before)
    used = _used(s, exp.shape)
    _assert_weights(after[used], exp[used], bound, what)
    assert np.array_equal(after[~used], before[~used], equal_nan=True), what


@pytest.mark.parametrize("route", ["observed", "cleared"])
def test_tokens_that_a_plain_step_appended(psi, oracle, device, route):
    """Prefill and verify steps accumulate nothing.  What the last owner of a page left there (NaN) is kept out by observing
    their tokens from the first of them on, or by clearing the accumulators of pages as they are issued."""
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(151, [330, 120], HQ, HKV, D, psi.Dtype.Bfloat16, PAGE, **LAYERS)
    pages, ids = device.from_numpy(w.pages.reshape(-1)), device.from_numpy(w.page_ids)
    acc = psi.page_weights(device, _config(psi, w), w.num_pages).fill_(float("nan"))
    if route == "cleared":
        for r in range(2):
            acc[torch.from_numpy(page_rows(w, r)[:-(-int(w.context_lens[r]) // PAGE)])] = 0.0
    observe, cached = psi.GQAKVObserveKernels(device, _config(psi, w)), np.array([0, 0])
    for n, (q_lens, how) in enumerate([([300, 90], "prefill"), ([4, 4], "verify"), ([1, 1], "decode"), ([4, 2], "verify"),
                                       ([1, 1], "decode")]):
        s = _step(psi, w, 152 + n, cached + q_lens, q_lens)
        s.pages = w.pages
        before = acc.cpu().numpy()
        held = [0, 0] if how == "prefill" else cached
        if how == "decode":
            out = _accumulating(psi, device, s, pages, ids, acc, 0.5)
        else:
            out = _plain(psi, device, s, pages, ids)
            if route == "observed":
                plan = observe.prepare(s.req_slots, s.token_indices, s.cu_tokens, held)
                observe.invoke(plan, device.from_numpy(s.q.reshape(-1)), pages, ids, acc, w.layer, decay=0.5)
        w.pages, exp_out = oracle_step(oracle, s)
        assert_outputs_close(out, exp_out, f"{how} {n}")
        if how == "decode" or route == "observed":
            _check_accumulators(s, w.pages, held, 0.5, before, acc.cpu().numpy(), f"{how} {n}")
        cached = cached + q_lens
    got = acc.cpu().numpy()
    assert np.isfinite(got[_used(s, got.shape)]).all()


def _cache(psi, device, slots, blocks, num_pages, seed):
    """An arena of random bytes, its accumulators, a table of two layers, and what a step's workload needs of them."""
    wl = importlib_workloads(psi)
    layout = psi.GQAPageTableLayout(4, 2, blocks, 1)
    table = psi.GQARequestPageTable(device, layout)
    rng = np.random.default_rng(seed)
    host = wl.to_storage(rng.standard_normal((num_pages, 2, HKV, PAGE, D)).astype(np.float32), psi.Dtype.Bfloat16)
    c = types.SimpleNamespace(table=table, layout=layout, num_pages=num_pages, req_slots=np.asarray(slots, np.uint32),
                              pages=host, layer=0, page_ids=None)
    c.cfg = psi.GQAKVEvictionConfig(HQ, HKV, D, D ** -0.5, 2 * HKV * PAGE * D * 2, layout, psi.Dtype.Bfloat16)
    c.d_pages = device.from_numpy(host.reshape(-1))
    c.acc = psi.page_weights(device, c.cfg, num_pages).fill_(float("nan"))
    return c


def _view(c, device, layer):
    device.sync()
    c.layer, c.page_ids = layer, c.table.page_ids.cpu().numpy().view(np.uint32)
    return c


def _cut(psi, device, c, kernels, requests, cached):
    """Selects and compacts both layers of some requests, next to the same on the host."""
    plan = kernels.prepare(c.req_slots[requests], cached)
    for layer in range(2):
        _view(c, device, layer)
        host_acc = c.acc.cpu().numpy()
        kept = kernels.invoke_select(plan, c.acc, c.table.page_ids, layer)
        kernels.invoke_compact(plan, kept, c.d_pages, c.acc, c.table.page_ids, layer)
        for r, n in zip(requests, cached):
            rows, p = page_rows(c, r), np.arange(n)
            keep = [kept_positions(host_acc[rows[p // PAGE], h, p % PAGE], n, kernels.budget, kernels.num_first,
                                   kernels.num_recent) for h in range(HKV)]
            c.pages, host_acc = compacted(c.pages, host_acc, rows, keep, PAGE)
        assert c.d_pages.cpu().numpy().tobytes() == c.pages.tobytes()
        assert c.acc.cpu().numpy().tobytes() == host_acc.tobytes()


def _prompt(psi, oracle, device, c, observe, requests, lens, seed):
    """Prefill of whole prompts by plain steps, then their last eight tokens observe."""
    for layer in range(2):
        _view(c, device, layer)
        s = _step(psi, c, seed + layer, lens, lens, requests)
        out = _plain(psi, device, s, c.d_pages, c.table.page_ids)
        c.pages, exp = oracle_step(oracle, s)
        assert_outputs_close(out, exp, "prefill")
        last = _step(psi, c, seed + layer, lens, [8] * len(lens), requests)
        last.q = np.concatenate([s.q[int(s.cu_tokens[r + 1]) - 8:int(s.cu_tokens[r + 1])] for r in range(len(lens))])
        before = c.acc.cpu().numpy()
        plan = observe.prepare(last.req_slots, last.token_indices, last.cu_tokens, [0] * len(lens))
        observe.invoke(plan, device.from_numpy(last.q.reshape(-1)), c.d_pages, c.table.page_ids, c.acc, layer)
        _check_accumulators(last, c.pages, [0] * len(lens), 1.0, before, c.acc.cpu().numpy(), "prompt")


def _decode(psi, oracle, device, c, requests, cached, seed):
    for layer in range(2):
        _view(c, device, layer)
        s = _step(psi, c, seed + layer, np.asarray(cached) + 1, 1, requests)
        before = c.acc.cpu().numpy()
        out = _accumulating(psi, device, s, c.d_pages, c.table.page_ids, c.acc, 0.75)
        c.pages, exp = oracle_step(oracle, s)
        assert_outputs_close(out, exp, "decode")
        _check_accumulators(s, c.pages, s.token_indices, 0.75, before, c.acc.cpu().numpy(), "decode")


def test_freed_pages_go_to_another_request(psi, oracle, device):
    """A cache that the caller's own table and the allocator hold: a prompt finds no pages until two requests are cut,
    then gets theirs, with the accumulators they left there; all three decode and are cut again."""
    alloc = runtime.U32IDAllocator(64)
    c = _cache(psi, device, [2, 0, 3], 24, 64, 161)
    owned = {}

    def grow(r, tokens):
        for layer in range(2):
            mine = owned.setdefault((r, layer), [])
            while len(mine) * PAGE < tokens:
                mine.append(alloc.alloc_one())
                c.table.write_page_ids(int(c.req_slots[r]), layer, len(mine) - 1, mine[-1:], c.num_pages)

    def trim(r, tokens):
        for layer in range(2):
            keep = -(-tokens // PAGE)
            alloc.free_many(owned[r, layer][keep:])
            del owned[r, layer][keep:]

    observe = psi.GQAKVObserveKernels(device, c.cfg)
    evict = psi.GQAKVEvictionKernels(device, c.cfg, 60, 4, 16)
    for r, n in ((0, 300), (1, 90)):
        grow(r, n)
    _prompt(psi, oracle, device, c, observe, [0, 1], [300, 90], 162)
    assert alloc.free() == 14  # a prompt of 200 wants 26
    before = set(owned[0, 0] + owned[0, 1] + owned[1, 0] + owned[1, 1])
    _cut(psi, device, c, evict, [0, 1], [300, 90])
    for r in (0, 1):
        trim(r, 60)
    grow(2, 200)
    assert before & set(owned[2, 0] + owned[2, 1])
    _prompt(psi, oracle, device, c, observe, [2], [200], 164)
    _cut(psi, device, c, evict, [2], [200])
    trim(2, 60)
    cached = [60, 60, 60]
    for step in range(12):
        for r in range(3):
            grow(r, cached[r] + 1)
        _decode(psi, oracle, device, c, [0, 1, 2], cached, 170 + 2 * step)
        cached = [n + 1 for n in cached]
    _cut(psi, device, c, evict, [0, 1, 2], cached)
    for r in range(3):
        trim(r, 60)
    assert alloc.used() == 3 * 2 * 4


def test_a_request_of_the_block_bookkeeping(psi, oracle, device):
    """DecoderBlocks counts the tokens of the request and owns its pages: the cut cache lives in the first of them, at
    positions less by what was evicted, and all pages go back when the request does."""
    alloc = runtime.U32IDAllocator(64)
    c = _cache(psi, device, [1], 24, 64, 181)
    blocks = runtime.DecoderBlocks(alloc, PAGE, 1, 2, range(91))

    def schedule(tokens):
        while blocks.ready_token_slots() < tokens:
            assert blocks.init_block_once() != "ResourceLimitExceeded"
        sync = blocks.prepare_blocks()
        for i, ids in enumerate(sync.kv_page_ids[0]):
            for layer in range(2):
                c.table.write_page_ids(1, layer, sync.block_index + i, ids[layer:layer + 1], c.num_pages)
        blocks.commit_blocks(sync)
        return blocks.prepare(tokens)

    query = schedule(90)
    assert query.kind == "Prefill" and query.token_index == 0
    observe = psi.GQAKVObserveKernels(device, c.cfg)
    _prompt(psi, oracle, device, c, observe, [0], [90], 182)
    blocks.commit(query, runtime.SampledTokens.prefill(query.epoch))
    _cut(psi, device, c, psi.GQAKVEvictionKernels(device, c.cfg, 40, 4, 16), [0], [90])
    evicted = 90 - 40
    for step in range(20):
        query = schedule(1)
        assert query.kind == "Decode" and query.token_index == 90 + step
        _decode(psi, oracle, device, c, [0], [query.token_index - evicted], 190 + 2 * step)
        blocks.commit(query, runtime.SampledTokens.decode(query.epoch, [], 1000 + step))
    assert len(blocks.cached_tokens()) == 110 and alloc.used() == 2 * 7
    blocks.close()
    assert alloc.used() == 0


def test_rotary_positions_count_on_behind_a_compaction(psi, device):
    """Tokens are rotated for the position they have in the text and cached where the cut cache ends, through the layer's
    split-row form; the plain cache is a list of rotated lines per head."""
    import torch

    wl = importlib_workloads(psi)
    c = _cache(psi, device, [2], 24, 24, 201)
    dev, dtype = device.torch_device, torch.bfloat16
    for block in range(12):
        for layer in range(2):
            c.table.write_page_ids(2, layer, block, [2 * block + layer], 24)
    layer, n, budget = 1, 120, 48
    core = psi.GQACore(0, HQ * D, D, HQ, HKV, D ** -0.5)
    gqa = psi.GQA.new(device, core, psi.GQAMetalConfig(c.cfg.page_bytes, 64, 1e-6, 1e4), False)
    rope = {h: psi.RMSNormRopeKernel(device, psi.RMSNormRopeConfig(h, D, 64, 1e-6, 1e4)) for h in (HQ, HKV)}
    gen = torch.Generator(device=dev).manual_seed(202)
    norm = {h: torch.rand(D, generator=gen, device=dev).add_(0.5).to(dtype) for h in (HQ, HKV)}

    def rotated(heads, rows, positions):
        x = torch.randn(rows, heads, D, generator=gen, device=dev).to(dtype)
        out = torch.empty_like(x)
        rope[heads].invoke(rows, x, norm[heads], torch.as_tensor(positions, dtype=torch.int32, device=dev), out)
        return x, out

    def record(first, rows, text_first, weights=None):
        meta = psi.GQAMetadataBuffers(device, rows, max_kv_splits=4 * rows)
        shape = gqa.prepare_fixed_partition(meta, [2], [first], [0, rows], 64,
                                            variant=psi.GQASplitKVVariant.SingleQ(16, 256, 4))
        text = list(range(text_first, text_first + rows))
        (_, q), (k_raw, k) = rotated(HQ, rows, text), rotated(HKV, rows, text)
        if text_first != first:  # (the cache position would rotate otherwise)
            other = torch.empty_like(k)
            rope[HKV].invoke(rows, k_raw, norm[HKV], torch.arange(first, first + rows, dtype=torch.int32, device=dev), other)
            assert not torch.equal(other, k)
        v = torch.randn(rows, HKV, D, generator=gen, device=dev).to(dtype)
        scratch = gqa.new_scratch(rows, shape.num_total_sdpa_map_task_templates)
        inp = psi.GQAInput(c.layout, layer, meta, psi.GQAKVCacheBindings(c.d_pages, c.table.page_ids), scratch, q=q, k=k, v=v)
        inp.output = torch.zeros(rows * HQ * D, device=dev)
        inp.kv_weights = weights
        device.f32_output(True)
        gqa.record(inp)
        device.f32_output(False)
        device.sync()
        return [t.view(torch.int16).cpu().numpy().view(np.uint16) for t in (q, k, v)] + [inp.output.cpu().numpy()]

    q, k, v, _ = record(0, n, 0)
    lines = [np.stack([k[:, h], v[:, h]], axis=1) for h in range(HKV)]  # [token][K, V][dim]
    observe = psi.GQAKVObserveKernels(device, c.cfg)
    observe.invoke(observe.prepare([2], [n - 16], [0, 16], [0]), device.from_numpy(q[-16:]), c.d_pages, c.table.page_ids,
                   c.acc, layer)
    evict = psi.GQAKVEvictionKernels(device, c.cfg, budget, 4, 8)
    plan = evict.prepare([2], [n])
    kept = evict.invoke_select(plan, c.acc, c.table.page_ids, layer)
    evict.invoke_compact(plan, kept, c.d_pages, c.acc, c.table.page_ids, layer)
    lines = [x[kept[0, h].cpu().numpy()] for h, x in enumerate(lines)]
    weights = psi.GQAKVWeights(c.acc, gqa.new_logits(1, 64))
    for step in range(8):
        q, k, v, out = record(budget + step, 1, n + step, weights)
        lines = [np.concatenate([x, np.stack([k[:, h], v[:, h]], axis=1)]) for h, x in enumerate(lines)]
        exp = np.zeros((HQ, D))
        for g in range(HQ):
            keys, values = (to_f64(lines[g // (HQ // HKV)][:, i], psi.Dtype.Bfloat16) for i in (0, 1))
            exp[g] = softmax_rows((keys @ to_f64(q[0, g], psi.Dtype.Bfloat16))[None, :] * D ** -0.5)[0] @ values
        assert_outputs_close(out, exp, f"step {step}")
    _view(c, device, layer)
    pages = c.d_pages.cpu().numpy().view(np.uint16).reshape(c.pages.shape)
    rows, p = page_rows(c, 0), np.arange(budget + 8)
    for h in range(HKV):
        assert np.array_equal(pages[rows[p // PAGE], :, h, p % PAGE], lines[h])
    acc = c.acc.cpu().numpy()[rows[p // PAGE], :, p % PAGE]
    assert np.isfinite(acc).all() and (acc > 0).all()
