"""What the cache-eviction classes refuse before anything is launched, without a GPU: the checks run against a device whose
context is null, so that a call which passes them ends with the library's own refusal."""
import types

import pytest

from test_kv_eviction_host import _config


@pytest.fixture
def host(psi):
    import torch

    return types.SimpleNamespace(lib=psi.load(), ctx=None, torch_device=torch.device("cpu"), stream=None)


def _weights(device, pages=64, hkv=4, page=16):
    import torch

    return torch.zeros(pages, hkv, page, device=device.torch_device)


@pytest.mark.parametrize("budget,hkv", [(64, 4), (16, 4), (32, 8), (32, 2), (64, 2)])
def test_a_plan_is_refused_by_kernels_of_another_budget_or_head_count(psi, host, budget, hkv):
    """A larger budget would write behind the plan's kept positions, and a budget and head count of the same product
    would read them in another order."""
    import torch

    ids = torch.zeros(8 * 2 * 64, dtype=torch.int32)
    plan = psi.GQAKVEvictionKernels(host, _config(psi), 32, 4, 8).prepare([1, 5], [100, 200])
    other = psi.GQAKVEvictionKernels(host, _config(psi, hq=24, hkv=hkv), budget, 4, 8)
    kept = torch.zeros(2, hkv, budget, dtype=torch.int32)
    with pytest.raises(ValueError, match="plan: one prepared by kernels of this budget"):
        other.invoke_select(plan, _weights(host, hkv=hkv), ids, 0)
    for k in (kept, plan.kept):
        with pytest.raises(ValueError, match="plan: one prepared by kernels of this budget"):
            other.invoke_compact(plan, k, torch.zeros(64), None, ids, 0)


def test_a_plan_serves_kernels_of_the_same_budget_and_head_count(psi, host):
    import torch

    ids = torch.zeros(8 * 2 * 64, dtype=torch.int32)
    plan = psi.GQAKVEvictionKernels(host, _config(psi), 32, 4, 8).prepare([1, 5], [100, 200])
    other = psi.GQAKVEvictionKernels(host, _config(psi), 32, 0, 16)
    with pytest.raises(psi.PsiHipError, match="ctx must not be null"):
        other.invoke_select(plan, _weights(host), ids, 0)
    with pytest.raises(psi.PsiHipError, match="ctx must not be null"):
        other.invoke_compact(plan, plan.kept.clone(), torch.zeros(64), None, ids, 0)
    with pytest.raises(ValueError, match="kept"):
        other.invoke_compact(plan, plan.kept[:1].contiguous(), torch.zeros(64), None, ids, 0)
