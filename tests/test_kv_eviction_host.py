"""Cache eviction on the host: plans and what the entry points refuse, through the C ABI, without a GPU."""
import ctypes

import numpy as np
import pytest

from eviction_util import kept_positions


def _config(psi, hq=24, hkv=4, d=256, page=16, dtype=None, slots=8, layers=2, blocks=64, ids=1):
    dtype = psi.Dtype.Bfloat16 if dtype is None else dtype
    layout = psi.GQAPageTableLayout(slots, layers, blocks, ids)
    return psi.GQAKVEvictionConfig(hq, hkv, d, d ** -0.5, 2 * hkv * page * d * dtype.item_size(), layout, dtype)


def _p(a):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32)) if a is not None else None


def _observe_plan(psi, cfg, slots, firsts, cu, held=None, capacity=None):
    L = psi._lib
    slots, firsts, cu = (np.asarray(x, np.uint32) for x in (slots, firsts, cu))
    held = np.asarray(held, np.uint32) if held is not None else None
    capacity = 512 + len(slots) if capacity is None else capacity
    windows, rows = np.zeros((len(slots), 8), np.uint32), np.zeros((max(capacity, 1), 3), np.uint32)
    n, most, scratch = ctypes.c_uint32(), ctypes.c_uint32(), ctypes.c_uint64()
    c, lay = cfg.struct(), cfg.page_table_layout.struct()
    L.check(L.load().psi_hip_kv_observe_plan(ctypes.byref(c), ctypes.byref(lay), _p(slots), _p(firsts), _p(cu), _p(held),
                                             len(slots), _p(windows), _p(rows), capacity, ctypes.byref(n),
                                             ctypes.byref(most), ctypes.byref(scratch)))
    return windows, rows[:n.value], most.value, scratch.value


def test_page_weights_bytes(psi):
    L, cfg, out = psi._lib, _config(psi).struct(), ctypes.c_uint64()
    L.check(L.load().psi_hip_kv_page_weights_bytes(ctypes.byref(cfg), 10, ctypes.byref(out)))
    assert out.value == 10 * 4 * 16 * 4
    for pages in (0, 1 << 32):
        with pytest.raises(psi.PsiHipError, match="number of pages"):
            L.check(L.load().psi_hip_kv_page_weights_bytes(ctypes.byref(cfg), pages, ctypes.byref(out)))


def test_logits_bytes_round_the_context_up_to_a_block(psi):
    L, cfg, out = psi._lib, _config(psi).struct(), ctypes.c_uint64()
    L.check(L.load().psi_hip_split_kv_single_q_logits_bytes(ctypes.byref(cfg), 3, 17, ctypes.byref(out)))
    assert out.value == 3 * 24 * 64 * 4
    with pytest.raises(psi.PsiHipError, match="need tokens and a context"):
        L.check(L.load().psi_hip_split_kv_single_q_logits_bytes(ctypes.byref(cfg), 3, 0, ctypes.byref(out)))


@pytest.mark.parametrize("blocks,reqs", [(64, [(0, 1)]), (64, [(0, 9), (1000, 24), (333, 1), (15, 17)]),
                                         (8192, [(131000, 72), (5, 3), (65536, 64)])])
def test_observe_plan_rows_tile_every_window(psi, blocks, reqs):
    cfg = _config(psi, blocks=blocks)
    firsts, sizes = [a for a, _ in reqs], [b for _, b in reqs]
    cu = np.concatenate([[0], np.cumsum(sizes)])
    windows, rows, most, scratch = _observe_plan(psi, cfg, range(len(reqs)), firsts, cu)
    assert most == max(sizes)
    assert scratch >= (len(rows) * most * 2 + cu[-1]) * 24 * 4
    at = 0
    for r, (first, size) in enumerate(reqs):
        assert windows[r].tolist()[:5] == [r, cu[r], size, first, first]
        begin, end = windows[r][5:7]
        assert begin == at and end > begin
        at = end
        mine = rows[begin:end]
        assert (mine[:, 0] == r).all() and mine[0, 1] == 0 and mine[-1, 2] == first + size
        assert (mine[1:, 1] == mine[:-1, 2]).all() and (mine[:, 2] > mine[:, 1]).all()
    assert at == len(rows) <= 512 + len(reqs)


def test_observe_plan_takes_held_counts(psi):
    windows, _, _, _ = _observe_plan(psi, _config(psi), [3, 1], [10, 20], [0, 4, 5], held=[0, 7])
    assert windows[:, 4].tolist() == [0, 7]


@pytest.mark.parametrize("slots,firsts,cu,match", [
    ([0, 0], [1, 1], [0, 1, 2], "named twice"),
    ([8], [1], [0, 1], "req_slot out of range"),
    ([0], [1020], [0, 5], "exceed the page table"),
    ([0], [1], [0, 0], "needs a query token"),
    ([0, 1], [1, 1], [0, 2, 1], "needs a query token"),
    ([0], [1], [1, 2], "start at zero"),
    ([], [], [0], "needs requests"),
])
def test_observe_plan_refusals(psi, slots, firsts, cu, match):
    with pytest.raises(psi.PsiHipError, match=match):
        _observe_plan(psi, _config(psi), slots, firsts, cu)


def test_observe_plan_refuses_too_few_rows(psi):
    with pytest.raises(psi.PsiHipError, match="rows are not enough"):
        _observe_plan(psi, _config(psi), [0, 1], [700, 700], [0, 1, 2], capacity=1)


def _evict_plan(psi, cfg, slots, cached):
    L = psi._lib
    slots, cached = np.asarray(slots, np.uint32), np.asarray(cached, np.uint32)
    requests, most = np.zeros((max(len(slots), 1), 2), np.uint32), ctypes.c_uint32()
    c, lay = cfg.struct(), cfg.page_table_layout.struct()
    L.check(L.load().psi_hip_kv_evict_plan(ctypes.byref(c), ctypes.byref(lay), _p(slots), _p(cached), len(slots),
                                           _p(requests), ctypes.byref(most)))
    return requests, most.value


def test_evict_plan(psi):
    requests, most = _evict_plan(psi, _config(psi), [5, 0, 2], [1024, 0, 7])
    assert requests.tolist() == [[5, 1024], [0, 0], [2, 7]] and most == 1024


@pytest.mark.parametrize("slots,cached,match", [
    ([0, 3, 0], [1, 1, 1], "named twice"),
    ([9], [1], "req_slot out of range"),
    ([0], [1025], "exceed the page table"),
    ([], [], "needs requests"),
])
def test_evict_plan_refusals(psi, slots, cached, match):
    with pytest.raises(psi.PsiHipError, match=match):
        _evict_plan(psi, _config(psi), slots, cached)


def test_positions_stay_below_two_to_the_31(psi):
    with pytest.raises(psi.PsiHipError, match="below 2\\^31"):
        _evict_plan(psi, _config(psi, blocks=1 << 28), [0], [1])


def test_null_arguments_are_refused_before_a_gpu_is_touched(psi):
    L, lib = psi._lib, psi.load()
    cfg, lay = _config(psi).struct(), _config(psi).page_table_layout.struct()
    c, y = ctypes.byref(cfg), ctypes.byref(lay)
    assert lib.psi_hip_split_kv_single_q_attend_weights(None, c, y, *[None] * 2, 0, *[None] * 8, 0, None, None, 0, None,
                                                        None, None, 0, 1, 1, 1, 1) == L.ERR_INVALID_ARGUMENT
    assert lib.psi_hip_kv_observe_weights(None, c, y, None, 1, None, 0, None, None, 1, 1, None, 1, None, 0, None, 0, 1.0,
                                          0) == L.ERR_INVALID_ARGUMENT
    assert lib.psi_hip_kv_select_kept(None, c, y, None, 0, None, None, 1, 1, 1, 0, 0, None, None, 0,
                                      0) == L.ERR_INVALID_ARGUMENT
    assert lib.psi_hip_kv_compact(None, c, y, None, 0, None, 0, None, None, 1, 1, 1, None, 0) == L.ERR_INVALID_ARGUMENT
    assert b"must not be null" in lib.psi_hip_last_error()


def test_layer_call_refuses_missing_weights_and_contexts(psi):
    lib, L = psi.load(), psi._lib
    cfg, inp, weights = L.LayerConfigStruct(), L.LayerInputStruct(), L.KVWeightsStruct()
    assert lib.psi_hip_gqa_layer_record_weights(None, ctypes.byref(cfg), ctypes.byref(inp), None) == L.ERR_INVALID_ARGUMENT
    assert b"weights must not be null" in lib.psi_hip_last_error()
    assert lib.psi_hip_gqa_layer_record_weights(None, ctypes.byref(cfg), ctypes.byref(inp),
                                                ctypes.byref(weights)) == L.ERR_INVALID_ARGUMENT
    assert b"ctx must not be null" in lib.psi_hip_last_error()


def test_kernel_classes_refuse_budgets_that_do_not_hold_what_is_always_kept(psi):
    for budget, first, recent in ((0, 0, 0), (4, 3, 2), (4, -1, 0)):
        with pytest.raises(ValueError, match="budget"):
            psi.GQAKVEvictionKernels(None, _config(psi), budget, first, recent)


def test_plain_rule_of_the_selection():
    """The oracle itself on a case worked by hand: ties to the lower index, NaN below everything, -0 equal to 0."""
    w = np.array([0.0, 5.0, np.nan, -0.0, 5.0, 0.0, 1.0, 0.0], np.float32)
    assert kept_positions(w, 8, 4, 0, 0).tolist() == [0, 1, 4, 6]
    assert kept_positions(w, 8, 5, 0, 0).tolist() == [0, 1, 3, 4, 6]
    assert kept_positions(w, 8, 4, 3, 1).tolist() == [0, 1, 2, 7]
    assert kept_positions(w, 8, 8, 3, 1).tolist() == list(range(8))
    assert kept_positions(w, 3, 2, 0, 0).tolist() == [0, 1]


def test_device_error_bit_matches_the_header(psi):
    import os
    import re

    text = open(os.path.join(os.path.dirname(psi.__file__), "..", "include", "psi_hip.h")).read()
    assert int(re.search(r"#define PSI_HIP_DEVICE_ERR_CACHE_RANGE\s+(\d+)u", text).group(1)) == \
        psi._lib.DEVICE_ERR_CACHE_RANGE
