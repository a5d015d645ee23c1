"""Cache eviction through the layer call, on other streams and contexts, with unaligned accumulators, and with pages whose
offsets pass 32 bits."""
import dataclasses

import numpy as np
import pytest

from eviction_util import attention_weights, page_rows
from parity_util import assert_outputs_close, importlib_workloads
from test_gpu_kv_eviction import LAYERS, _assert_weights, _config, _weights

pytestmark = pytest.mark.gpu

SINGLE_Q = (16, 256, 8)


def _layer(psi, device, w, gated):
    core = psi.GQACore(0, w.num_q_heads * w.head_dim, w.head_dim, w.num_q_heads, w.num_kv_heads, w.scale)
    return psi.GQA.new(device, core, psi.GQAMetalConfig(w.page_bytes, 64, 1e-6, 1e7, io_dtype=w.dtype), gated)


def _two_byte(device, w, array):
    import torch

    return device.from_numpy(array.reshape(-1)).view(torch.bfloat16 if int(w.dtype) == 1 else torch.float16)


def _layer_input(psi, device, w, gqa, meta, shape, pages, ids, from_rows, seed):
    """A layer's input from split rows with a gate, or from projection output."""
    import torch

    scratch = gqa.new_scratch(shape.num_total_tokens, shape.num_total_sdpa_map_task_templates)
    gen = torch.Generator(device=device.torch_device).manual_seed(seed)
    inp = psi.GQAInput(w.layout, w.layer, meta, psi.GQAKVCacheBindings(pages, ids), scratch)
    inp.output = torch.zeros(w.num_tokens * w.num_q_heads * w.head_dim, device=device.torch_device)
    if from_rows:
        inp.q, inp.k, inp.v = (_two_byte(device, w, x) for x in (w.q, w.flat_k, w.flat_v))
        inp.g = torch.randn(inp.q.shape, generator=gen, device=device.torch_device).to(inp.q.dtype)
    else:
        scratch.qgkv.copy_(torch.randn(scratch.qgkv.shape, generator=gen, device=device.torch_device))
        inp.weights = psi.GQAWeights(*(torch.rand(w.head_dim, generator=gen, device=device.torch_device)
                                       .add_(0.5).to(torch.bfloat16) for _ in range(2)))
    return inp


@pytest.mark.parametrize("from_rows,gated", [(True, True), (False, True), (False, False)])
@pytest.mark.parametrize("balanced", [False, True])
def test_layer_call_accumulates(psi, device, from_rows, gated, balanced):
    """`record` with weights: the output and the appended cache of `record` without them, and the accumulators of the
    queries and keys that the layer made."""
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(71, [700, 17, 1, 1025], 24, 4, 256, psi.Dtype.Bfloat16, 16, **LAYERS)
    gqa = _layer(psi, device, w, gated)
    meta = psi.GQAMetadataBuffers(device, 8, max_kv_splits=256)
    shape = gqa.prepare_fixed_partition(meta, w.req_slots, w.token_indices, w.cu_tokens, 256, balanced=balanced,
                                        variant=psi.GQASplitKVVariant.SingleQ(*SINGLE_Q))
    ids = device.from_numpy(w.page_ids)
    acc, out, lines = _weights(w), [], []
    for with_weights in (False, True):
        pages = _two_byte(device, w, w.pages)
        inp = _layer_input(psi, device, w, gqa, meta, shape, pages, ids, from_rows, 72)
        if with_weights:
            inp.kv_weights = psi.GQAKVWeights(device.from_numpy(acc), gqa.new_logits(4, 1025), 0.5)
            inp.kv_weights.logits.buffer.fill_(0xff)
        device.f32_output(True)
        try:
            gqa.record(inp)
        finally:
            device.f32_output(False)
        device.sync()
        out.append(inp.output.cpu().numpy())
        lines.append(pages.view(dtype=torch.int16).cpu().numpy().view(np.uint16).reshape(w.pages.shape))
    assert np.array_equal(lines[0], lines[1])
    assert_outputs_close(out[1], out[0].astype(np.float64), "output")
    q = inp.q if from_rows else inp.scratch.q_norm_rope[:w.num_tokens * 24 * 256]
    w = dataclasses.replace(w, q=q.view(torch.int16).cpu().numpy().view(np.uint16))
    exp, bound = attention_weights(w, lines[1], w.token_indices, 0.5, acc)
    got, used = inp.kv_weights.page_weights.cpu().numpy(), np.zeros(exp.shape, bool)
    for r in range(4):
        p = np.arange(int(w.context_lens[r]))
        used[page_rows(w, r)[p // 16], :, p % 16] = True
    _assert_weights(got[used], exp[used], bound, "weights")
    assert np.array_equal(got[~used], acc[~used])


def test_layer_call_refusals(psi, device):
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(73, [40, 90], 24, 4, 256, psi.Dtype.Bfloat16, 16, q_lens=2)
    gqa = _layer(psi, device, w, True)
    meta = psi.GQAMetadataBuffers(device, 8, max_kv_splits=64)
    shape = gqa.prepare_fixed_partition(meta, w.req_slots, w.token_indices, w.cu_tokens, 256)
    assert meta.split_kv_variant().is_tiled()
    pages, ids = _two_byte(device, w, w.pages), device.from_numpy(w.page_ids)
    inp = _layer_input(psi, device, w, gqa, meta, shape, pages, ids, False, 74)
    acc = device.from_numpy(_weights(w))
    inp.kv_weights = psi.GQAKVWeights(acc, gqa.new_logits(4, 90))
    with pytest.raises(psi.PsiHipError, match="SingleQ"):
        gqa.record(inp)
    with pytest.raises(ValueError, match="only `record`"):
        gqa.record_static_scratch(inp)
    inp.kv_weights = psi.GQAKVWeights(acc.half(), gqa.new_logits(4, 90))
    with pytest.raises(ValueError, match="float32"):
        gqa.record(inp)
    device.sync()
    assert np.array_equal(pages.view(dtype=torch.int16).cpu().numpy().view(np.uint16), w.pages.reshape(-1))


class _Round:
    """Observation, selection, compaction and a decode step of one small batch on a device: prepared once, run on the
    arena and accumulators it is given."""

    def __init__(self, psi, device, ids_of=lambda ids: ids, num_pages=None, seed=81):
        wl = importlib_workloads(psi)
        self.psi, self.device = psi, device
        self.w = w = wl.make_workload(seed, [400, 90, 2050], 8, 2, 128, psi.Dtype.Bfloat16, 16, q_lens=[8, 1, 5], **LAYERS)
        cfg = _config(psi, w)
        self.observe = psi.GQAKVObserveKernels(device, cfg)
        self.evict = psi.GQAKVEvictionKernels(device, cfg, 64, 4, 8)
        self.oplan = self.observe.prepare(w.req_slots, w.token_indices, w.cu_tokens, [0, 50, 0])
        self.eplan = self.evict.prepare(w.req_slots, w.context_lens)
        self.q = device.from_numpy(w.q.reshape(-1))
        self.ids = device.from_numpy(ids_of(w.page_ids))
        self.step = wl.make_workload(seed + 1, [65, 65, 65], 8, 2, 128, psi.Dtype.Bfloat16, 16, shuffle_slots=False,
                                     host_pages=False)
        s = self.step
        s.layout, s.layer, s.req_slots, s.page_ids, s.pages = w.layout, w.layer, w.req_slots, ids_of(w.page_ids), None
        s.num_pages = num_pages or w.num_pages
        self.dw = None

    def run(self, pages, acc):
        w, device = self.w, self.device
        if self.dw is None:
            self.dw = importlib_workloads(self.psi).DeviceWorkload(
                device, self.step, partition_tokens=64, f32_output=False, balanced=True, pages=pages, page_ids=self.ids,
                variant=self.psi.GQASplitKVVariant.SingleQ(16, 256, 4))
            self.logits = self.psi.GQASplitKVSingleQLogits(device, self.dw.cfg, self.dw.kshape, 65)
        dw, m = self.dw, self.dw.meta
        self.observe.invoke(self.oplan, self.q, pages, self.ids, acc, w.layer, decay=0.5)
        kept = self.evict.invoke_select(self.eplan, acc, self.ids, w.layer)
        self.evict.invoke_compact(self.eplan, kept, pages, acc, self.ids, w.layer)
        dw.kernels.invoke_attend_weights_bucketed(
            dw.q, pages, m.d_req_slots, m.d_flat_token_indices, self.ids, m.d_kv_splits, m.d_cu_kv_splits, dw.scratch,
            self.logits, dw.output, acc, 0.5, w.layer, 3, dw.shape.num_sdpa_map_task_templates, worker_cu=m.d_worker_cu,
            num_workers=m.num_workers, flat_k=dw.flat_k, flat_v=dw.flat_v)

    def results(self, pages, acc):
        import torch

        self.device.sync()
        return [t.contiguous().view(torch.uint8).cpu().numpy().copy() for t in (pages, acc, self.eplan.kept, self.dw.output)]


def _plain_round(psi, device):
    r = _Round(psi, device)
    pages, acc = device.from_numpy(r.w.pages.reshape(-1)), device.from_numpy(_weights(r.w))
    r.run(pages, acc)
    return r, r.results(pages, acc)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_accumulators_that_are_not_aligned_to_16_bytes(psi, device, offset):
    import torch

    _, exp = _plain_round(psi, device)
    r = _Round(psi, device)
    start = _weights(r.w)
    flat = torch.full((start.size + 8,), -7.0, device=device.torch_device)
    acc = flat[offset:offset + start.size].view(start.shape)
    assert acc.data_ptr() % 16 == 4 * offset
    acc.copy_(device.from_numpy(start))
    pages = device.from_numpy(r.w.pages.reshape(-1))
    r.run(pages, acc)
    for a, b in zip(r.results(pages, acc), exp):
        assert np.array_equal(a, b)
    assert (flat[:offset] == -7.0).all() and (flat[offset + start.size:] == -7.0).all()


def test_two_streams_at_once(psi, device):
    """Two contexts on streams of their own with their own arenas, plans and scratch, the default stream busy besides:
    either gets what it gets alone."""
    import torch

    _, exp = _plain_round(psi, device)
    busy = torch.randn(2048, 2048, device="cuda")
    torch.cuda.synchronize()
    rounds = []
    for _ in range(2):
        stream = torch.cuda.Stream()
        dev = psi.Device(0, stream)
        with torch.cuda.stream(stream):
            r = _Round(psi, dev)
            rounds.append((r, stream, dev.from_numpy(r.w.pages.reshape(-1)), dev.from_numpy(_weights(r.w))))
    for r, stream, pages, acc in rounds:
        with torch.cuda.stream(stream):
            r.run(pages, acc)
        busy = busy @ busy * 1e-3
    for r, stream, pages, acc in rounds:
        with torch.cuda.stream(stream):
            for a, b in zip(r.results(pages, acc), exp):
                assert np.array_equal(a, b)
        r.device.close()


def test_two_graphs_of_one_plan_replayed_in_turn(psi, device):
    """Two captured graphs that share a plan's scratch, kept positions and logits, on two arenas, replayed one after the
    other with other work between them."""
    import torch

    _, exp = _plain_round(psi, device)
    stream = torch.cuda.Stream()
    dev = psi.Device(0, stream)
    with torch.cuda.stream(stream):
        r = _Round(psi, dev)
        start = dev.from_numpy(r.w.pages.reshape(-1)), dev.from_numpy(_weights(r.w))
        arenas = [tuple(t.clone() for t in start) for _ in range(2)]
        r.run(*arenas[0])  # (builds the step's buffers)
    dev.sync()
    graphs = []
    for pages, acc in arenas:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            r.run(pages, acc)
        graphs.append(graph)
    for _ in range(3):
        with torch.cuda.stream(stream):
            for arena in arenas:
                for t, s in zip(arena, start):
                    t.copy_(s)
            for graph, (pages, acc) in zip(graphs, arenas):
                graph.replay()
                torch.randn(1 << 18, device="cuda").sum().item()
            for pages, acc in arenas:
                for a, b in zip(r.results(pages, acc), exp):
                    assert np.array_equal(a, b)
    dev.close()


def test_pages_beyond_32_bit_offsets(psi, device):
    """The same batch on pages whose elements lie beyond 2^32: the same bits as at the front of an arena."""
    import torch

    plain, exp = _plain_round(psi, device)
    elems, n = plain.w.pages[0].size, plain.w.num_pages
    first = (1 << 32) // elems + 5
    r = _Round(psi, device, ids_of=lambda ids: (ids + np.uint32(first)).astype(np.uint32), num_pages=first + n)
    pages = torch.empty((first + n) * elems, dtype=torch.int16, device=device.torch_device)
    acc = torch.zeros((first + n,) + _weights(r.w).shape[1:], device=device.torch_device)
    pages[first * elems:].copy_(device.from_numpy(r.w.pages.reshape(-1)))
    acc[first:].copy_(device.from_numpy(_weights(r.w)))
    r.run(pages, acc)
    got = r.results(pages[first * elems:], acc[first:])
    for a, b in zip(got, exp):
        assert np.array_equal(a, b)
    assert not acc[:first].any()


def test_long_selection_and_compaction_captured(psi, device):
    """The forms of several launches (a selection in chunks, a compaction in levels) in a graph, replayed."""
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(91, [20001, 17000], 1, 1, 64, psi.Dtype.Float16, 16, **LAYERS)
    stream = torch.cuda.Stream()
    dev = psi.Device(0, stream)
    evict = psi.GQAKVEvictionKernels(dev, _config(psi, w), 9000, 4, 8)
    with torch.cuda.stream(stream):
        plan = evict.prepare(w.req_slots, w.context_lens)
        ids, start = dev.from_numpy(w.page_ids), (dev.from_numpy(w.pages.reshape(-1)), dev.from_numpy(_weights(w)))
        pages, acc = (t.clone() for t in start)

    def step():
        evict.invoke_compact(plan, evict.invoke_select(plan, acc, ids, w.layer), pages, acc, ids, w.layer)

    def results():
        dev.sync()
        return [t.view(torch.uint8).cpu().numpy().copy() for t in (pages, acc, plan.kept)]

    with torch.cuda.stream(stream):
        step()
    exp = results()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(3):
        with torch.cuda.stream(stream):
            pages.copy_(start[0])
            acc.copy_(start[1])
            graph.replay()
            got = results()
            torch.randn(1 << 18, device="cuda").sum().item()
        for a, b in zip(got, exp):
            assert np.array_equal(a, b)
    # the plain form of what was kept and moved
    from eviction_util import compacted, kept_positions

    host_pages, host_acc = w.pages.copy(), _weights(w)
    for r, n in enumerate(w.context_lens):
        rows, p = page_rows(w, r), np.arange(int(n))
        keep = [kept_positions(host_acc[rows[p // 16], 0, p % 16], int(n), 9000, 4, 8)]
        assert np.array_equal(exp[2].view(np.int32).reshape(2, 9000)[r], keep[0])
        host_pages, host_acc = compacted(host_pages, host_acc, rows, keep, 16)
    assert exp[0].tobytes() == host_pages.tobytes() and exp[1].tobytes() == host_acc.tobytes()
    dev.close()
