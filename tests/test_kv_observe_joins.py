"""Where the statistics of an observation's windows are joined: inside the second pass, or in a launch of their own when a
window has many rows.  The longest window decides, however short the others are."""
import numpy as np
import pytest

from test_kv_eviction_host import _config


@pytest.mark.parametrize("firsts,sizes", [([100], [9]), ([100, 5, 900], [9, 1, 64]), ([99968] + [32] * 31, [32] * 32)])
def test_plans_know_their_longest_window(psi, firsts, sizes):
    import types

    import torch

    host = types.SimpleNamespace(lib=psi.load(), ctx=None, torch_device=torch.device("cpu"), stream=None)
    kernels = psi.GQAKVObserveKernels(host, _config(psi, hq=8, hkv=1, slots=32, blocks=8192))
    plan = kernels.prepare(range(len(firsts)), firsts, np.concatenate([[0], np.cumsum(sizes)]))
    rows = plan.rows.numpy().reshape(-1, 3)
    assert plan.max_window_rows == np.bincount(rows[:, 0]).max()
    if len(firsts) == 32:  # 1792 states by the average, 57344 in the long window
        assert plan.max_window_rows > 25 * len(rows) // len(firsts)


def test_null_context_is_refused(psi):
    import ctypes

    L, lib, cfg = psi._lib, psi.load(), _config(psi)
    c, lay = cfg.struct(), cfg.page_table_layout.struct()
    assert lib.psi_hip_kv_observe_weights_rows(None, ctypes.byref(c), ctypes.byref(lay), None, 1, None, 0, None, None, 1,
                                               1, None, 1, 1, None, 0, None, 0, 1.0, 0) == L.ERR_INVALID_ARGUMENT


@pytest.mark.gpu
@pytest.mark.parametrize("hq,hkv,d,window", [(8, 1, 128, 32), (24, 4, 256, 16), (6, 1, 256, 3)])
@pytest.mark.parametrize("told", ["planned", "unknown", "one"])
def test_one_long_prompt_among_short_ones(psi, device, hq, hkv, d, window, told):
    """Either form gives the weights, whichever the launch takes for what it is told."""
    from eviction_util import attention_weights
    from parity_util import importlib_workloads
    from test_gpu_kv_eviction import LAYERS, _assert_weights, _weights

    wl = importlib_workloads(psi)
    lens = [16500] + [64] * 9
    w = wl.make_workload(131, lens, hq, hkv, d, psi.Dtype.Bfloat16, 16, q_lens=[window] * 10, **LAYERS)
    cfg = psi.GQAKVEvictionConfig(hq, hkv, d, w.scale, w.page_bytes, w.layout, w.dtype)
    kernels = psi.GQAKVObserveKernels(device, cfg)
    held = [9000] + [0] * 9
    plan = kernels.prepare(w.req_slots, w.token_indices, w.cu_tokens, held)
    plan.scratch.fill_(0xff)
    plan.max_window_rows = {"planned": plan.max_window_rows, "unknown": 0, "one": 1}[told]
    acc = _weights(w)
    weights = device.from_numpy(acc)
    kernels.invoke(plan, device.from_numpy(w.q.reshape(-1)), device.from_numpy(w.pages.reshape(-1)),
                   device.from_numpy(w.page_ids), weights, w.layer, decay=0.5)
    exp, bound = attention_weights(w, w.pages, held, 0.5, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound)
