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


def _pages():
    import torch

    return torch.zeros(64 * 2 * 4 * 16 * 256, dtype=torch.bfloat16)


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
            other.invoke_compact(plan, k, _pages(), None, ids, 0)


def test_a_plan_serves_kernels_of_the_same_budget_and_head_count(psi, host):
    import torch

    ids = torch.zeros(8 * 2 * 64, dtype=torch.int32)
    plan = psi.GQAKVEvictionKernels(host, _config(psi), 32, 4, 8).prepare([1, 5], [100, 200])
    other = psi.GQAKVEvictionKernels(host, _config(psi), 32, 0, 16)
    with pytest.raises(psi.PsiHipError, match="ctx must not be null"):
        other.invoke_select(plan, _weights(host), ids, 0)
    with pytest.raises(psi.PsiHipError, match="ctx must not be null"):
        other.invoke_compact(plan, plan.kept.clone(), _pages(), None, ids, 0)
    with pytest.raises(ValueError, match="kept"):
        other.invoke_compact(plan, plan.kept[:1].contiguous(), _pages(), None, ids, 0)


@pytest.mark.parametrize("dtype,other", [("Bfloat16", "float16"), ("Float16", "bfloat16"), ("Float32", "bfloat16"),
                                         ("Bfloat16", "float32"), ("Float32", "float64"), ("Float16", "float32")])
def test_queries_and_pages_of_another_type_are_refused(psi, host, dtype, other):
    import torch

    dtype, other, ids = getattr(psi.Dtype, dtype), getattr(torch, other), torch.zeros(1024, dtype=torch.int32)
    observe = psi.GQAKVObserveKernels(host, _config(psi, dtype=dtype))
    plan = observe.prepare([3], [100], [0, 4])
    q = torch.zeros(4 * 24 * 256)
    pages = torch.zeros(64 * 2 * 4 * 16 * 256)
    with pytest.raises(ValueError, match="q: contiguous rows of the cache's type"):
        observe.invoke(plan, q.to(other), pages.to(dtype.torch()), ids, _weights(host), 0)
    with pytest.raises(ValueError, match="kv_pages: a contiguous arena of the configured type"):
        observe.invoke(plan, q.to(dtype.torch()), pages.to(other), ids, _weights(host), 0)
    evict = psi.GQAKVEvictionKernels(host, _config(psi, dtype=dtype), 32)
    plan = evict.prepare([1], [100])
    with pytest.raises(ValueError, match="kv_pages: a contiguous arena of the configured type"):
        evict.invoke_compact(plan, plan.kept, pages.to(other), None, ids, 0)


@pytest.mark.parametrize("dtype,bits", [("Bfloat16", "int16"), ("Float16", "int16"), ("Float32", "int32")])
def test_queries_may_come_as_bit_patterns_and_pages_as_bytes(psi, host, dtype, bits):
    import torch

    dtype, ids = getattr(psi.Dtype, dtype), torch.zeros(1024, dtype=torch.int32)
    observe = psi.GQAKVObserveKernels(host, _config(psi, dtype=dtype))
    plan = observe.prepare([3], [100], [0, 4])
    for t in (dtype.torch(), getattr(torch, bits)):
        q, pages = torch.zeros(4 * 24 * 256, dtype=t), torch.zeros(64 * 2 * 4 * 16 * 256, dtype=t)
        for arena in (pages, pages.view(torch.uint8)):
            with pytest.raises(psi.PsiHipError, match="ctx must not be null"):
                observe.invoke(plan, q, arena, ids, _weights(host), 0)
    with pytest.raises(ValueError, match="q: contiguous rows of the cache's type"):
        observe.invoke(plan, q.view(torch.uint8), pages, ids, _weights(host), 0)


def test_strided_queries_and_pages_are_refused(psi, host):
    import torch

    ids = torch.zeros(1024, dtype=torch.int32)
    observe = psi.GQAKVObserveKernels(host, _config(psi))
    plan = observe.prepare([3], [100], [0, 4])
    wide = torch.zeros(4, 2 * 24 * 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="q: contiguous"):
        observe.invoke(plan, wide[:, :24 * 256], _pages(), ids, _weights(host), 0)
    with pytest.raises(ValueError, match="kv_pages: a contiguous"):
        observe.invoke(plan, wide, _pages().view(64, -1)[:, ::2], ids, _weights(host), 0)


def test_logits_on_another_device_are_refused(psi, host):
    import torch

    logits = types.SimpleNamespace(buffer=torch.empty(64, device="meta"), bytes=256, max_context_tokens=64)
    with pytest.raises(ValueError, match="logits: room on the kernels' device"):
        psi.GQAKVWeights(_weights(host), logits).struct(host)


def test_missing_pages_are_refused(psi, host):
    import torch

    ids = torch.zeros(1024, dtype=torch.int32)
    observe = psi.GQAKVObserveKernels(host, _config(psi))
    q = torch.zeros(4 * 24 * 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="kv_pages: a contiguous"):
        observe.invoke(observe.prepare([3], [100], [0, 4]), q, None, ids, _weights(host), 0)
    evict = psi.GQAKVEvictionKernels(host, _config(psi), 32)
    plan = evict.prepare([1], [100])
    with pytest.raises(ValueError, match="kv_pages: a contiguous"):
        evict.invoke_compact(plan, plan.kept, None, None, ids, 0)
