"""Arenas that are aligned to their elements only, and lines that are no multiple of 16 bytes: the eviction operators take
the units and kernels that fit and give the same results."""
import numpy as np
import pytest

from eviction_util import attention_weights, compacted, kept_positions, page_rows
from parity_util import assert_outputs_close, importlib_workloads, oracle_step
from test_gpu_kv_eviction import LAYERS, _assert_weights, _attend, _compact, _config, _observe, _weights

pytestmark = pytest.mark.gpu


def _shifted(device, array, elements):
    """The array on the device, `elements` of its elements behind an aligned address; the tensor and its whole buffer."""
    import torch

    t = device.from_numpy(array.reshape(-1))
    room = torch.full((t.numel() + 64,), 17, dtype=t.dtype, device=t.device)
    view = room[elements:elements + t.numel()]
    view.copy_(t)
    return view, room


def _margins_untouched(room, view, elements):
    return bool((room[:elements] == 17).all()) and bool((room[elements + view.numel():] == 17).all())


@pytest.mark.parametrize("hkv,d,page,ids", [(3, 3, 5, 3), (1, 10, 16, 1), (2, 33, 8, 2), (2, 1, 7, 1)])
@pytest.mark.parametrize("dtype", ["Float32", "Bfloat16"])
@pytest.mark.parametrize("budget", [5, 640])
def test_compaction_of_lines_that_are_no_multiple_of_16_bytes(psi, device, hkv, d, page, ids, dtype, budget):
    _compact(psi, device, [0, 1, budget, budget + 1, 3 * budget + 2, 1601], hkv, d, dtype, page, ids, budget)


@pytest.mark.parametrize("dtype,d,elements", [("Float32", 64, 1), ("Float32", 64, 2), ("Bfloat16", 128, 1),
                                              ("Float16", 256, 4), ("Bfloat16", 64, 2)])
def test_compaction_in_an_arena_that_is_not_aligned_to_16_bytes(psi, device, dtype, d, elements):
    wl = importlib_workloads(psi)
    lens, budget = [40, 700, 1601], 300
    w = wl.make_workload(161, lens, 2, 2, d, getattr(psi.Dtype, dtype), 16, **LAYERS)
    acc, rng = _weights(w), np.random.default_rng(162)
    exp_pages, exp_acc, kept = w.pages.copy(), acc.copy(), np.full((3, 2, budget), -1, np.int32)
    for r, n in enumerate(lens):
        keep = [kept_positions(rng.random(n).astype(np.float32), n, budget, 2, 30) for _ in range(2)]
        for h in range(2):
            kept[r, h, :len(keep[h])] = keep[h]
        exp_pages, exp_acc = compacted(exp_pages, exp_acc, page_rows(w, r), keep, 16)
    kernels = psi.GQAKVEvictionKernels(device, _config(psi, w), budget, 2, 30)
    pages, room = _shifted(device, w.pages, elements)
    assert pages.data_ptr() % 16 != 0
    weights = device.from_numpy(acc)
    kernels.invoke_compact(kernels.prepare(w.req_slots, lens), device.from_numpy(kept), pages, weights,
                           device.from_numpy(w.page_ids), w.layer)
    device.sync()
    assert pages.cpu().numpy().tobytes() == exp_pages.tobytes() and weights.cpu().numpy().tobytes() == exp_acc.tobytes()
    assert _margins_untouched(room, pages, elements)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(12, 2, 128, "Bfloat16"), (4, 1, 256, "Float16")])
@pytest.mark.parametrize("elements", [1, 4])
def test_attention_over_an_arena_that_is_not_aligned_to_16_bytes(psi, oracle, device, hq, hkv, d, dtype, elements):
    wl = importlib_workloads(psi)
    w = wl.make_workload(163, [33, 600], hq, hkv, d, getattr(psi.Dtype, dtype), 16, q_lens=[3, 1], **LAYERS)
    acc = _weights(w)
    exp, bound = attention_weights(w, w.pages, [0, 300], 0.5, acc)
    pages, room = _shifted(device, w.pages, elements)
    _assert_weights(_observe(psi, device, w, acc, [0, 300], 0.5, pages=pages).cpu().numpy(), exp, bound, "observation")
    dw = wl.DeviceWorkload(device, w, partition_tokens=128, f32_output=True, pages=pages,
                           variant=psi.GQASplitKVVariant.SingleQ(16, 256, 8))
    _, weights = _attend(psi, device, w, acc, 0.5, dw=dw)
    device.sync()
    exp_pages, exp_out = oracle_step(oracle, w)
    assert np.array_equal(dw.pages_host().reshape(exp_pages.shape), exp_pages)
    assert_outputs_close(dw.output_f32(), exp_out, "attention")
    exp, bound = attention_weights(w, exp_pages, w.token_indices, 0.5, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound, "step")
    assert _margins_untouched(room, pages, elements)
