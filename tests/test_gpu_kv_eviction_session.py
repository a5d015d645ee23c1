"""Eviction next to what else touches a cache: steps that append without accumulating."""
import numpy as np
import pytest

from eviction_util import attention_weights, page_rows
from parity_util import assert_outputs_close, importlib_workloads, oracle_step
from test_gpu_kv_eviction import LAYERS, _assert_weights, _config

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE = 8, 2, 128, 16


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
