"""Slots beyond the page table and pages beyond the arena in a decode step that accumulates: their accumulators are left
out and reported.  (K and V come through the table unchecked, as in every decode step, so the table and the arena that
these tests hand over are whole; only the bounds that the call is told are smaller.)"""
import dataclasses

import numpy as np
import pytest

from eviction_util import attention_weights, page_rows
from parity_util import importlib_workloads
from test_gpu_kv_eviction import LAYERS, _assert_weights, _attend, _weights

pytestmark = pytest.mark.gpu

SINGLE_Q = (16, 256, 8)


def _step(psi, device, w, **kw):
    wl = importlib_workloads(psi)
    return wl.DeviceWorkload(device, w, partition_tokens=128, f32_output=True,
                             variant=psi.GQASplitKVVariant.SingleQ(*SINGLE_Q), **kw)


@pytest.mark.parametrize("q_lens", [1, [1, 1, 4, 1]], ids=str)
@pytest.mark.parametrize("generic", [False, True])
def test_a_slot_beyond_the_table_leaves_its_accumulators(psi, device, q_lens, generic):
    wl = importlib_workloads(psi)
    w = wl.make_workload(111, [300, 70, 513, 90], 12, 2, 128, psi.Dtype.Bfloat16, 16, q_lens=q_lens, shuffle_slots=False,
                         **LAYERS)
    acc = _weights(w)
    dw = _step(psi, device, w)
    # the table keeps its five slots; the call is told of two
    dw.kernels.config = dataclasses.replace(dw.cfg, page_table_layout=dataclasses.replace(w.layout, num_req_slots=2))
    device.force_generic(generic)
    try:
        _, weights = _attend(psi, device, w, acc, 0.5, dw=dw)
        assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    finally:
        device.force_generic(False)
    exp, bound = attention_weights(w, dw.pages_host().reshape(w.pages.shape), w.token_indices, 0.5, acc)
    for r in (2, 3):
        rows, p = page_rows(w, r), np.arange(int(w.context_lens[r]))
        exp[rows[p // 16], :, p % 16] = acc[rows[p // 16], :, p % 16]
    _assert_weights(weights.cpu().numpy(), exp, bound)


def test_pages_beyond_the_arena_leave_their_accumulators(psi, device):
    wl = importlib_workloads(psi)
    w = wl.make_workload(112, [300, 513], 12, 2, 128, psi.Dtype.Bfloat16, 16, **LAYERS)
    acc, told = _weights(w), w.num_pages // 2
    dw = _step(psi, device, w)
    arena = dw.pages
    dw.pages = arena[:told * (arena.numel() // w.num_pages)]  # (the tensor behind it holds every page)
    _, weights = _attend(psi, device, w, acc, 1.0, dw=dw)
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    dw.pages = arena
    exp, bound = attention_weights(w, dw.pages_host().reshape(w.pages.shape), w.token_indices, 1.0, acc)
    exp[told:] = acc[told:]
    _assert_weights(weights.cpu().numpy(), exp, bound)
