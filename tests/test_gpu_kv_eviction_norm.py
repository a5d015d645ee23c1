"""Weights of keys that are all alike: with keys of zero every logit is 0 and every key of n gets 1 / n.  The maximum (0),
the sum (n ones) and the exponentials are exact in f32, so one division is the only rounding of a query's weight."""
import numpy as np
import pytest

from eviction_util import HALF_ULP32, page_rows
from parity_util import importlib_workloads
from test_gpu_kv_eviction import LAYERS, _attend, _observe

pytestmark = pytest.mark.gpu


def _alike(psi, lens, hq, hkv, d, dtype):
    wl = importlib_workloads(psi)
    w = wl.make_workload(121, lens, hq, hkv, d, getattr(psi.Dtype, dtype), 16, **LAYERS)
    w.pages[:, 0] = 0
    w.flat_k[:] = 0
    return w, np.zeros((w.num_pages, hkv, 16), np.float32)


def _assert_equal_weights(w, weights):
    weights = weights.cpu().numpy().astype(np.float64)
    for r, n in enumerate(int(c) for c in w.context_lens):
        rows, p = page_rows(w, r), np.arange(n)
        off = np.abs(weights[rows[p // 16], :, p % 16] * n - 1.0).max()
        # (2^-24 relative to the rounded value is a little more relative to 1 / n)
        assert off <= HALF_ULP32 * (1 + 2 * HALF_ULP32), f"{n} keys: {off:.3e}"


@pytest.mark.parametrize("hq,hkv,d,dtype", [(2, 2, 256, "Bfloat16"), (1, 1, 128, "Float16"), (2, 2, 64, "Bfloat16"),
                                            (1, 1, 20, "Float32")])
@pytest.mark.parametrize("lens", [[1, 2, 3, 7, 777, 1283, 5000], [40001]], ids=str)
def test_equal_keys_weigh_one_nth_each(psi, device, hq, hkv, d, dtype, lens):
    w, acc = _alike(psi, lens, hq, hkv, d, dtype)
    _assert_equal_weights(w, _observe(psi, device, w, acc, [0] * len(lens), 1.0))
    _, weights = _attend(psi, device, w, acc, 1.0)
    device.sync()
    _assert_equal_weights(w, weights)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(12, 2, 256, "Bfloat16"), (8, 1, 128, "Bfloat16"), (4, 2, 64, "Bfloat16")])
@pytest.mark.parametrize("tokens", [1, 3])
def test_a_step_over_keys_that_nothing_can_attend_to(psi, device, hq, hkv, d, dtype, tokens):
    """Keys with an element of -inf under queries that are all positive: their weights are 0, and the others' sum to one
    per query, also where a whole row of the plan holds such keys only."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(122, [400, 30], hq, hkv, d, getattr(psi.Dtype, dtype), 16, q_lens=[tokens, 1], **LAYERS)
    w.q = np.where((w.q & 0x7fff) == 0, 0x3f80, w.q & 0x7fff).astype(np.uint16)
    rows, dead = page_rows(w, 0), np.r_[5, 64:128, 390]
    w.pages[rows[dead // 16], 0, :, dead % 16, d - 1] = 0xff80
    acc = np.full((w.num_pages, hkv, 16), 3.0, np.float32)
    _, weights = _attend(psi, device, w, acc, 0.0, partition=64, balanced=False)
    device.sync()
    p, group = np.arange(400), hq // hkv
    mine = weights.cpu().numpy()[rows[p // 16], :, p % 16]
    assert np.isfinite(mine).all() and (mine[dead] == 0.0).all()
    # 400 weights of a few queries, each a few roundings of exp2 and of a normaliser of 400 terms
    assert np.abs(mine.sum(axis=0) / (tokens * group) - 1.0).max() <= HALF_ULP32 * (2 * 400 + tokens * group + 64)
