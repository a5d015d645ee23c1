"""A layer step that is refused for its accumulators leaves the cache as it was: nothing is appended before the check."""
import types

import numpy as np
import pytest

from parity_util import importlib_workloads
from test_gpu_kv_eviction import _weights
from test_gpu_kv_eviction_layer import SINGLE_Q, _layer, _layer_input, _two_byte

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("from_rows", [False, True])
@pytest.mark.parametrize("what,match", [("decay", "decay"), ("logits", "logits buffer too small"),
                                        ("aligned", "16-byte aligned"), ("accumulators", "smaller than one page")])
def test_refused_steps_append_nothing(psi, device, from_rows, what, match):
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(141, [40, 90], 24, 4, 256, psi.Dtype.Bfloat16, 16)
    gqa = _layer(psi, device, w, True)
    meta = psi.GQAMetadataBuffers(device, 8, max_kv_splits=64)
    shape = gqa.prepare_fixed_partition(meta, w.req_slots, w.token_indices, w.cu_tokens, 256,
                                        variant=psi.GQASplitKVVariant.SingleQ(*SINGLE_Q))
    pages, acc = _two_byte(device, w, w.pages), device.from_numpy(_weights(w))
    inp = _layer_input(psi, device, w, gqa, meta, shape, pages, device.from_numpy(w.page_ids), from_rows, 142)
    logits, decay = gqa.new_logits(2, 90), 0.5
    if what == "decay":
        decay = 1.5
    elif what == "logits":
        logits = types.SimpleNamespace(buffer=logits.buffer, bytes=logits.bytes - 64, max_context_tokens=90)
    elif what == "aligned":
        room = torch.empty(logits.bytes + 4, dtype=torch.uint8, device=device.torch_device)
        logits = types.SimpleNamespace(buffer=room[4:], bytes=logits.bytes, max_context_tokens=90)
    else:
        acc = acc.reshape(-1)[:63]
    inp.kv_weights = psi.GQAKVWeights(acc, logits, decay)
    before = acc.clone()
    with pytest.raises(psi.PsiHipError, match=match):
        gqa.record(inp)
    device.sync()
    assert np.array_equal(pages.view(dtype=torch.int16).cpu().numpy().view(np.uint16), w.pages.reshape(-1))
    assert torch.equal(acc, before)
