"""The scratch of a long selection: sized once for a capacity, it serves every smaller batch."""
import ctypes

import numpy as np
import pytest

from test_kv_eviction_host import _config

CHUNK_BYTES = 3 * 2048 * 2 + 16  # three digits' counters of 16 bits, and what a chunk knows between the launches


def _bytes(psi, cfg, reqs, cached):
    out, c = ctypes.c_uint64(), cfg.struct()
    psi._lib.check(psi.load().psi_hip_kv_select_scratch_bytes(ctypes.byref(c), reqs, cached, ctypes.byref(out)))
    return out.value


@pytest.mark.parametrize("hkv", [1, 2, 3, 8])
def test_scratch_never_falls_with_a_larger_capacity(psi, hkv):
    cfg = _config(psi, hq=hkv, hkv=hkv)
    cached = [0, 1, 4096, 16384, 16385, 24576, 24577, 32768, 32769, 65536, 100000, 131072, 140000, 262144, 524288, 1 << 20,
              (1 << 20) + 1, 1 << 24, 1 << 30]
    reqs = [1, 2, 3, 4, 5, 6, 7, 8, 9, 13, 16, 17, 31, 32, 33, 64, 128, 1000]
    table = np.array([[_bytes(psi, cfg, r, n) for n in cached] for r in reqs], object)
    assert (table[1:] >= table[:-1]).all() and (table[:, 1:] >= table[:, :-1]).all()
    assert (table[:, :4] == 0).all()
    # what a launch of either chunk size goes through is there (whichever of them this size takes)
    for i, r in enumerate(reqs):
        for j, n in enumerate(cached[4:], 4):
            small, large = r * hkv * -(-n // 4096), r * hkv * -(-n // 8192)
            assert table[i, j] >= CHUNK_BYTES * (small if large <= 128 else large)
            assert table[i, j] <= CHUNK_BYTES * max(large, 256)


@pytest.mark.parametrize("hkv", [1, 3, 8, 300])
def test_observation_scratch_has_a_bound_over_all_batches(psi, hkv):
    from test_kv_eviction_host import _observe_plan

    cfg, rng = _config(psi, hq=2 * hkv, hkv=hkv, d=8, slots=80, blocks=8192), np.random.default_rng(37)
    for reqs in (1, 2, 7, 40, 80):
        firsts, sizes = rng.integers(0, 120000, reqs), rng.integers(1, 65, reqs)
        cu = np.concatenate([[0], np.cumsum(sizes)])
        _, rows, most, scratch = _observe_plan(psi, cfg, range(reqs), firsts, cu)
        assert scratch <= (max(256 // hkv, reqs, 1) * most + int(cu[-1])) * 2 * hkv * 8


@pytest.mark.gpu
@pytest.mark.parametrize("hkv,large,small", [(8, [32768] * 5, [32768, 17001, 30000, 32768]),
                                             (2, [140000, 16], [131072]), (1, [600000], [524288])])
def test_scratch_of_a_larger_batch_serves_a_smaller_one(psi, device, hkv, large, small):
    """The larger batch takes chunks of 8192 positions, the smaller one twice as many of 4096."""
    import torch

    from eviction_util import kept_positions, page_rows
    from parity_util import importlib_workloads

    wl = importlib_workloads(psi)
    w = wl.make_workload(35, small, hkv, hkv, 8, psi.Dtype.Float32, 16, host_pages=False)
    cfg = psi.GQAKVEvictionConfig(hkv, hkv, 8, 1.0, w.page_bytes, w.layout, w.dtype)
    acc = np.random.default_rng(36).integers(0, 1000, (w.num_pages, hkv, 16)).astype(np.float32)
    kernels = psi.GQAKVEvictionKernels(device, cfg, 5000, 4, 32)
    plan = kernels.prepare(w.req_slots, small)
    capacity = _bytes(psi, cfg, len(large), max(large))
    plan.scratch = torch.full((capacity // 4,), float("nan"), device=device.torch_device)
    kept = kernels.invoke_select(plan, device.from_numpy(acc), device.from_numpy(w.page_ids), w.layer).cpu().numpy()
    for r, n in enumerate(small):
        rows, p = page_rows(w, r), np.arange(n)
        for h in range(hkv):
            assert np.array_equal(kept[r, h], kept_positions(acc[rows[p // 16], h, p % 16], n, 5000, 4, 32)), (r, h)
