"""Rows longer than the planners of small batches make them, against 64 bits: observation over several turns of a
workgroup, decode attention whose logits overflow their room in LDS, whose rows take several turns of the accumulating
launch, and whose steps bring more (token, head) pairs than it holds normalisers for."""
import numpy as np
import pytest

from eviction_util import attention_weights, page_rows, softmax_rows, to_f64
from parity_util import assert_outputs_close, importlib_workloads, oracle_step
from test_gpu_kv_eviction import LAYERS, _assert_weights, _attend, _config, _weights

pytestmark = pytest.mark.gpu


def _observe_rows(psi, device, w, acc, held, decay, cuts):
    """An observation whose windows are cut at `cuts(context)` (ascending, without the ends)."""
    import torch

    kernels = psi.GQAKVObserveKernels(device, _config(psi, w))
    plan = kernels.prepare(w.req_slots, w.token_indices, w.cu_tokens, held)
    windows = plan.windows.cpu().numpy().view(np.uint32).reshape(-1, 8).copy()
    rows = []
    for r, n in enumerate(int(c) for c in w.context_lens):
        at = [0, *cuts(n), n]
        windows[r, 5:7] = len(rows), len(rows) + len(at) - 1
        rows += [(r, a, b) for a, b in zip(at, at[1:])]
    plan.windows = device.from_numpy(windows.reshape(-1))
    plan.rows, plan.num_rows = device.from_numpy(np.asarray(rows, np.uint32).reshape(-1)), len(rows)
    plan.scratch = torch.full((4 * (4 * len(rows) * plan.max_window + 2 * w.num_tokens) * w.num_q_heads,), 0xff,
                              dtype=torch.uint8, device=device.torch_device)
    weights = device.from_numpy(acc)
    kernels.invoke(plan, device.from_numpy(w.q.reshape(-1)), device.from_numpy(w.pages.reshape(-1)),
                   device.from_numpy(w.page_ids), weights, w.layer, decay=decay)
    return weights


CONTEXTS = [385, 769, 1153, 2500, 40]
CUTS = {"one row": lambda n: [], "two rows": lambda n: [n // 3] if n > 64 else [],
        "ragged rows": lambda n: [c for c in (17, 1000, 1003) if c < n]}


@pytest.mark.parametrize("hq,hkv,d,dtype,page", [(12, 2, 256, "Bfloat16", 16), (10, 2, 128, "Float16", 8),
                                                 (7, 1, 256, "Float16", 5), (16, 2, 128, "Bfloat16", 12),
                                                 (3, 3, 128, "Bfloat16", 32)])
@pytest.mark.parametrize("window", ["narrow", "wide"])
@pytest.mark.parametrize("cuts", CUTS)
def test_observation_in_rows_of_several_turns(psi, device, hq, hkv, d, dtype, page, window, cuts):
    wl = importlib_workloads(psi)
    q_lens = [5, 1, 8, 7, 2] if window == "narrow" else [33, 64, 1, 40, 40]
    w = wl.make_workload(101, CONTEXTS, hq, hkv, d, getattr(psi.Dtype, dtype), page, q_lens=q_lens, **LAYERS)
    acc, held = _weights(w), [0, 500, 1153, 2400, 10]
    got = _observe_rows(psi, device, w, acc, held, 0.75, CUTS[cuts])
    exp, bound = attention_weights(w, w.pages, held, 0.75, acc)
    _assert_weights(got.cpu().numpy(), exp, bound)


@pytest.mark.parametrize("hq,hkv,d,window", [(12, 2, 256, 5), (12, 2, 256, 40), (10, 2, 128, 64), (4, 2, 128, 3)])
@pytest.mark.parametrize("bad", [3, 70, 150, 156])
def test_a_page_beyond_the_arena_in_a_later_turn(psi, device, hq, hkv, d, window, bad):
    """The keys of that page take no part: the others' weights are a softmax without them, its accumulators stay."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(102, [2500], hq, hkv, d, psi.Dtype.Bfloat16, 16, q_lens=[window], **LAYERS)
    acc, rows = _weights(w), page_rows(w, 0)
    _, bound = attention_weights(w, w.pages, [2000], 0.5, acc)
    p = np.array([q for q in range(2500) if q // 16 != bad])
    values, q = to_f64(w.pages, w.dtype), to_f64(w.q, w.dtype).reshape(window, hq, d)
    exp = acc.astype(np.float64)
    hidden = p[None, :] > (2500 - window + np.arange(window))[:, None]
    for h in range(hkv):
        k, at = values[rows[p // 16], 0, h, p % 16], (rows[p // 16], h, p % 16)
        total = sum(softmax_rows(np.where(hidden, -np.inf, q[:, g] @ k.T * w.scale)).sum(axis=0)
                    for g in range(h * hq // hkv, (h + 1) * hq // hkv))
        exp[at] = np.where(p < 2000, 0.5 * exp[at], 0.0) + total
    w.page_ids = w.page_ids.copy()
    w.page_ids[(int(w.req_slots[0]) * w.layout.num_gqa_layers + w.layer) * w.layout.num_blocks + bad] = w.num_pages
    got = _observe_rows(psi, device, w, acc, [2000], 0.5, CUTS["one row"])
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    _assert_weights(got.cpu().numpy(), exp, bound)


@pytest.mark.parametrize("hq,hkv,d,dtype,page", [(2, 2, 256, "Bfloat16", 16), (12, 2, 256, "Bfloat16", 16),
                                                 (8, 1, 256, "Float16", 16), (1, 1, 128, "Float16", 8),
                                                 (6, 1, 128, "Bfloat16", 32), (16, 2, 128, "Bfloat16", 8),
                                                 (10, 2, 256, "Bfloat16", 8)])
@pytest.mark.parametrize("workers", [None, 1, 5])
def test_decode_rows_longer_than_the_logits_room(psi, oracle, device, hq, hkv, d, dtype, page, workers):
    """Rows of up to 9001 keys: a row to a workgroup (workers None), or shares of the balanced plan."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(103, [1153, 2049, 3713, 9001], hq, hkv, d, getattr(psi.Dtype, dtype), page, **LAYERS)
    acc = _weights(w)
    dw = wl.DeviceWorkload(device, w, partition_tokens=1 << 14, f32_output=True, balanced=workers is not None,
                           num_workers=workers, variant=psi.GQASplitKVVariant.SingleQ(16, 256, 8))
    _, first = _attend(psi, device, w, acc, 0.75, dw=dw)
    device.sync()
    out = dw.output_f32()
    exp_pages, exp_out = oracle_step(oracle, w)
    assert_outputs_close(out, exp_out, "attention next to the weights")
    exp, bound = attention_weights(w, exp_pages, w.token_indices, 0.75, acc)
    _assert_weights(first.cpu().numpy(), exp, bound)
    _, second = _attend(psi, device, w, acc, 0.75, dw=dw)
    device.sync()
    assert np.array_equal(dw.output_f32(), out) and np.array_equal(first.cpu().numpy(), second.cpu().numpy())


@pytest.mark.parametrize("hq,hkv,d,tokens", [(16, 2, 256, 65), (8, 1, 128, 150), (12, 2, 256, 90), (7, 1, 128, 147),
                                             (12, 1, 64, 43)])
@pytest.mark.parametrize("decay", [1.0, 0.25])
def test_steps_of_more_pairs_than_normalisers_are_held(psi, oracle, device, hq, hkv, d, tokens, decay):
    """More than 512 (token, head) pairs of one request: the decay is applied once, and also where a block of
    normalisers ends inside a token's heads."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(104, [tokens, 40 + tokens, 5, 2100], hq, hkv, d, psi.Dtype.Bfloat16, 16,
                         q_lens=[tokens, tokens - 1, 2, tokens], **LAYERS)
    acc = _weights(w)
    dw, weights = _attend(psi, device, w, acc, decay)
    exp_pages, exp_out = oracle_step(oracle, w)
    assert_outputs_close(dw.output_f32(), exp_out, "attention")
    exp, bound = attention_weights(w, exp_pages, w.token_indices, decay, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound)
