"""Cache eviction on the GPU against its plain 64-bit forms: what decode steps and prompts accumulate, which positions
are kept, what a compaction moves, and the four together over several steps."""
import numpy as np
import pytest

from eviction_util import HALF_ULP32, attention_weights, compacted, kept_positions, page_rows
from parity_util import assert_outputs_close, importlib_workloads, oracle_step

pytestmark = pytest.mark.gpu

LAYERS = dict(num_gqa_layers=2, layer=1)


def _config(psi, w):
    return psi.GQAKVEvictionConfig(w.num_q_heads, w.num_kv_heads, w.head_dim, w.scale, w.page_bytes, w.layout, w.dtype)


def _weights(w, seed=5):
    """Accumulators before a step: positive, none of them what a step leaves."""
    rng = np.random.default_rng(seed)
    return rng.uniform(0.5, 2.0, (w.num_pages, w.num_kv_heads, w.tokens_per_page)).astype(np.float32)


def _assert_weights(got, exp, bound, what=""):
    got = np.asarray(got, np.float64)
    assert got.shape == exp.shape and np.isfinite(got).all(), what
    off = np.abs(got - exp) / exp
    assert off.max() <= bound + 4 * HALF_ULP32, f"{what}: {off.max():.3e} > {bound:.3e}"


def _attend(psi, device, w, acc, decay, partition=None, balanced=True, fused=True, longest_first=False, max_context=None,
            dw=None):
    """One decode step through the component entry: (workload on the device, accumulators after)."""
    wl = importlib_workloads(psi)
    if dw is None:
        dw = wl.DeviceWorkload(device, w, partition_tokens=partition or 512, f32_output=True, balanced=balanced,
                               longest_first=longest_first, variant=psi.GQASplitKVVariant.SingleQ(16, 256, 8))
    m, s = dw.meta, dw.shape
    logits = psi.GQASplitKVSingleQLogits(device, dw.cfg, dw.kshape, max_context or int(w.context_lens.max()))
    logits.buffer.fill_(0xff)  # NaN wherever a logit is read that was not stored
    weights = device.from_numpy(acc)
    if not fused:
        dw.append()
    device.f32_output(True)
    dw.kernels.invoke_attend_weights_bucketed(
        dw.q, dw.pages, m.d_req_slots, m.d_flat_token_indices, dw.page_ids, m.d_kv_splits, m.d_cu_kv_splits, dw.scratch,
        logits, dw.output, weights, decay, w.layer, s.num_tokens, s.num_sdpa_map_task_templates,
        worker_cu=m.d_worker_cu if dw.balanced else None, num_workers=m.num_workers if dw.balanced else 0,
        flat_k=dw.flat_k if fused else None, flat_v=dw.flat_v if fused else None,
        partial_row_index=m.d_partial_row_index)
    device.f32_output(False)
    return dw, weights


SHAPES = [  # hq, hkv, d, tokens per page, page IDs per block, type
    (24, 4, 256, 16, 1, "Bfloat16"), (16, 2, 256, 16, 1, "Float16"), (40, 8, 128, 8, 2, "Float16"),
    (7, 1, 128, 32, 1, "Bfloat16"), (3, 3, 256, 8, 1, "Bfloat16"), (4, 2, 64, 16, 1, "Bfloat16"),
    (6, 2, 20, 5, 3, "Float32"), (12, 1, 128, 16, 1, "Float16"),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("decay", [1.0, 0.75])
def test_decode_step_accumulates(psi, oracle, device, shape, decay):
    hq, hkv, d, page, ids, dtype = shape
    wl = importlib_workloads(psi)
    w = wl.make_workload(11, [1, 2, 16, 17, 255, 600, 1283], hq, hkv, d, getattr(psi.Dtype, dtype), page,
                         num_page_ids_per_block=ids, **LAYERS)
    acc = _weights(w)
    dw, weights = _attend(psi, device, w, acc, decay)
    exp_pages, exp_out = oracle_step(oracle, w)
    assert np.array_equal(dw.pages_host().reshape(exp_pages.shape).view(np.uint8), exp_pages.view(np.uint8))
    assert_outputs_close(dw.output_f32(), exp_out, "attention next to the weights")
    exp, bound = attention_weights(w, exp_pages, w.token_indices, decay, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound)


@pytest.mark.parametrize("how", [dict(balanced=False), dict(balanced=False, longest_first=True), dict(fused=False),
                                 dict(balanced=False, fused=False, partition=16), dict(partition=64)],
                         ids=["rows", "longest-first", "append-apart", "rows-of-16", "balanced-64"])
def test_every_plan_accumulates_the_same(psi, oracle, device, how):
    wl = importlib_workloads(psi)
    w = wl.make_workload(12, [700, 1, 333, 2049], 24, 4, 256, psi.Dtype.Bfloat16, 16, **LAYERS)
    acc = _weights(w)
    dw, weights = _attend(psi, device, w, acc, 1.0, **how)
    exp_pages, exp_out = oracle_step(oracle, w)
    assert_outputs_close(dw.output_f32(), exp_out, "attention")
    exp, bound = attention_weights(w, exp_pages, w.token_indices, 1.0, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound)


@pytest.mark.parametrize("generic", [False, True])
def test_several_tokens_of_a_request_in_one_step(psi, oracle, device, generic):
    """Verify steps through the decode plan: the last token's rows own the positions, earlier tokens' weights are in."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(13, [400, 90, 9, 1030], 16, 2, 256, psi.Dtype.Bfloat16, 16, q_lens=[3, 1, 9, 40], **LAYERS)
    acc = _weights(w)
    device.force_generic(generic)
    try:
        dw, weights = _attend(psi, device, w, acc, 0.5)
        device.sync()
    finally:
        device.force_generic(False)
    exp_pages, exp_out = oracle_step(oracle, w)
    assert_outputs_close(dw.output_f32(), exp_out, "attention")
    exp, bound = attention_weights(w, exp_pages, w.token_indices, 0.5, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound)


def test_same_bits_on_every_run(psi, device):
    wl = importlib_workloads(psi)
    w = wl.make_workload(14, [900, 77, 2000], 24, 4, 256, psi.Dtype.Bfloat16, 16, **LAYERS)
    acc = _weights(w)
    dw, first = _attend(psi, device, w, acc, 1.0)
    _, second = _attend(psi, device, w, acc, 1.0, dw=dw)
    device.sync()
    assert np.array_equal(first.cpu().numpy(), second.cpu().numpy())


def test_contexts_beyond_the_logits_and_pages_beyond_the_accumulators_are_reported(psi, device):
    wl = importlib_workloads(psi)
    w = wl.make_workload(15, [300, 100], 24, 4, 256, psi.Dtype.Bfloat16, 16, **LAYERS)
    acc = _weights(w)
    dw, weights = _attend(psi, device, w, acc, 1.0, max_context=200)
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    exp, bound = attention_weights(w, dw.pages_host().reshape(w.pages.shape), w.token_indices, 1.0, acc)
    rows, p = page_rows(w, 0), np.arange(200, 300)
    exp[rows[p // 16], :, p % 16] = acc[rows[p // 16], :, p % 16]  # left as they were
    _assert_weights(weights.cpu().numpy(), exp, bound)
    short = acc[:w.num_pages // 2]
    _, weights = _attend(psi, device, w, short, 1.0, dw=dw)
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    exp, bound = attention_weights(w, dw.pages_host().reshape(w.pages.shape), w.token_indices, 1.0, acc)
    _assert_weights(weights.cpu().numpy(), exp[:len(short)], bound)
    device.sync()  # nothing is reported any more


def test_attend_weights_refusals(psi, device):
    wl = importlib_workloads(psi)
    w = wl.make_workload(16, [40], 24, 4, 256, psi.Dtype.Bfloat16, 16)
    for kw, match in ((dict(decay=1.5), "decay"), (dict(decay=float("nan")), "decay"), (dict(decay=-0.1), "decay")):
        with pytest.raises(psi.PsiHipError, match=match):
            _attend(psi, device, w, _weights(w), **kw)
    with pytest.raises(psi.PsiHipError, match="smaller than one page"):
        _attend(psi, device, w, np.zeros((1, 1, 16), np.float32), 1.0)


def test_bound_counts_limit_what_a_step_accumulates(psi, oracle, device):
    """Device-side counts: a launch cut for four tokens serves two; the other requests' accumulators keep their bytes."""
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(17, [500, 64, 33, 200], 24, 4, 256, psi.Dtype.Bfloat16, 16, **LAYERS)
    acc = _weights(w)
    dw = wl.DeviceWorkload(device, w, partition_tokens=64, f32_output=True,
                           variant=psi.GQASplitKVVariant.SingleQ(16, 256, 8))
    rows = int(np.count_nonzero(dw.meta.h_kv_splits.reshape(-1, 3)[:dw.shape.num_sdpa_map_task_templates, 0] < 2))
    counts = torch.tensor([2, 2, rows, 0], dtype=torch.int32, device=device.torch_device)
    device.bind_replay_counts(counts)
    try:
        _, weights = _attend(psi, device, w, acc, 1.0, dw=dw)
        device.sync()
    finally:
        device.bind_replay_counts(None)
    exp_pages, _ = oracle_step(oracle, w)
    exp, bound = attention_weights(w, exp_pages, w.token_indices, 1.0, acc)
    got = weights.cpu().numpy()
    for r in range(4):
        used = page_rows(w, r)[:-(-int(w.context_lens[r]) // 16)]
        if r < 2:
            _assert_weights(got[used], exp[used], bound, f"request {r}")
        else:
            assert np.array_equal(got[used], acc[used])


# ------------------------------------------------------------------ observation


def _observe(psi, device, w, acc, held, decay, pages=None):
    kernels = psi.GQAKVObserveKernels(device, _config(psi, w))
    plan = kernels.prepare(w.req_slots, w.token_indices, w.cu_tokens, held)
    plan.scratch.fill_(0xff)
    weights = device.from_numpy(acc)
    pages = device.from_numpy(w.pages.reshape(-1)) if pages is None else pages
    kernels.invoke(plan, device.from_numpy(w.q.reshape(-1)), pages, device.from_numpy(w.page_ids), weights, w.layer,
                   decay=decay)
    return weights


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("windows", [(1, 1, 1, 1, 1), (8, 3, 1, 5, 2), (9, 33, 1, 17, 64)], ids=str)
def test_observation_accumulates(psi, device, shape, windows):
    hq, hkv, d, page, ids, dtype = shape
    wl = importlib_workloads(psi)
    w = wl.make_workload(21, [9, 33, 1, 500, 1283], hq, hkv, d, getattr(psi.Dtype, dtype), page, q_lens=windows,
                         num_page_ids_per_block=ids, **LAYERS)
    acc, held = _weights(w), [0, 4, 1, 250, 1283]
    weights = _observe(psi, device, w, acc, held, 0.9)
    exp, bound = attention_weights(w, w.pages, held, 0.9, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound)


@pytest.mark.parametrize("hq,hkv,d", [(24, 4, 256), (8, 1, 128)])
def test_observation_of_a_whole_prompt(psi, device, hq, hkv, d):
    """Every token of a prompt observes: many query columns, and rows of keys that the first tokens do not reach."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(22, [300, 777], hq, hkv, d, psi.Dtype.Bfloat16, 16, q_lens=[300, 700], **LAYERS)
    acc = _weights(w)
    weights = _observe(psi, device, w, acc, [0, 0], 1.0)
    exp, bound = attention_weights(w, w.pages, [0, 0], 1.0, acc)
    _assert_weights(weights.cpu().numpy(), exp, bound)
    total = weights.cpu().numpy()[page_rows(w, 0)[:19]].sum()
    pad = acc[page_rows(w, 0)[18], :, 300 % 16:].sum()  # places behind the prompt's end keep what they had
    assert abs(total - pad - 300 * hq) <= 300 * hq * bound


def test_observation_ignores_what_lies_behind_the_context(psi, device):
    """NaN in the places behind a prompt's end and in pages that are not its own reach no accumulator."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(23, [37, 129], 24, 4, 256, psi.Dtype.Bfloat16, 16, q_lens=[5, 20], **LAYERS)
    acc = _weights(w)
    exp, bound = attention_weights(w, w.pages, [0, 0], 1.0, acc)
    pages = w.pages.copy()
    used = np.zeros(pages.shape[:1] + pages.shape[3:4], bool)
    for r in range(2):
        p = np.arange(int(w.context_lens[r]))
        used[page_rows(w, r)[p // 16], p % 16] = True
    pages.swapaxes(1, 3)[~used] = 0x7fc0
    w.pages = pages
    _assert_weights(_observe(psi, device, w, acc, [0, 0], 1.0).cpu().numpy(), exp, bound)


@pytest.mark.parametrize("hq,hkv,d", [(3, 3, 256), (10, 2, 128), (4, 2, 64)])
def test_observation_of_a_key_that_nothing_can_attend_to(psi, device, hq, hkv, d):
    """A key whose logits are -inf for every query (an infinite element, all queries positive) receives nothing; the
    weights of the others sum to one per query, also where the queries do not fill a block of columns."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(27, [150], hq, hkv, d, psi.Dtype.Bfloat16, 16, q_lens=[5], **LAYERS)
    w.q = np.where((w.q & 0x7fff) == 0, 0x3f80, w.q & 0x7fff).astype(np.uint16)
    rows = page_rows(w, 0)
    w.pages[rows[33 // 16], 0, :, 33 % 16, 7] = 0xff80
    acc = np.full((w.num_pages, hkv, 16), 3.0, np.float32)
    got = _observe(psi, device, w, acc, [0], 1.0).cpu().numpy()
    p = np.arange(150)
    mine = got[rows[p // 16], :, p % 16]
    assert np.isfinite(mine).all() and (mine[33] == 0.0).all()
    # 150 weights of 5 * group queries, each a few roundings of exp2 and of a normaliser of 150 terms
    assert np.abs(mine.sum(axis=0) / (5 * hq // hkv) - 1.0).max() <= 2.0 ** -24 * (2 * 150 + 5 * (hq // hkv) + 64)


def test_observation_leaves_out_pages_beyond_the_arena(psi, device):
    wl = importlib_workloads(psi)
    w = wl.make_workload(24, [64, 48], 24, 4, 256, psi.Dtype.Bfloat16, 16, q_lens=4, **LAYERS)
    acc = _weights(w)
    lay = w.layout
    bad = (int(w.req_slots[0]) * lay.num_gqa_layers + w.layer) * lay.num_blocks + 1
    exp, bound = attention_weights(w, w.pages, [0, 0], 1.0, acc)
    w.page_ids = w.page_ids.copy()
    w.page_ids[bad] = w.num_pages + 7
    weights = _observe(psi, device, w, acc, [0, 0], 1.0)
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    mine = page_rows(w, 1)[:3]
    _assert_weights(weights.cpu().numpy()[mine], exp[mine], bound)


@pytest.mark.parametrize("hq,hkv,d", [(40, 8, 128), (16, 2, 256)])
def test_observation_of_many_columns_over_few_keys(psi, device, hq, hkv, d):
    """Rows whose waves share the columns; a page beyond the arena in one prompt leaves its positions as they were and
    the other prompt untouched."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(28, [200, 330], hq, hkv, d, psi.Dtype.Bfloat16, 16, q_lens=[61, 64], **LAYERS)
    acc = _weights(w)
    exp, bound = attention_weights(w, w.pages, [150, 0], 0.5, acc)
    got = _observe(psi, device, w, acc, [150, 0], 0.5).cpu().numpy()
    for r in range(2):
        p = np.arange(int(w.context_lens[r]))
        at = (page_rows(w, r)[p // 16], slice(None), p % 16)
        _assert_weights(got[at], exp[at], bound, f"prompt {r}")
    rows, lay = page_rows(w, 0), w.layout
    w.page_ids = w.page_ids.copy()
    w.page_ids[(int(w.req_slots[0]) * lay.num_gqa_layers + w.layer) * lay.num_blocks + 2] = w.num_pages + 7
    got = _observe(psi, device, w, acc, [150, 0], 0.5)
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    got, mine = got.cpu().numpy(), page_rows(w, 1)[:-(-330 // 16)]
    p = np.arange(330)
    _assert_weights(got[mine[p // 16], :, p % 16], exp[mine[p // 16], :, p % 16], bound, "the other prompt")
    assert np.array_equal(got[rows[2]], acc[rows[2]])
    p = np.array([q for q in range(200) if q // 16 != 2])
    mine = got[rows[p // 16], :, p % 16]
    base = np.where(p < 150, 0.5, 0.0)[:, None] * acc[rows[p // 16], :, p % 16]
    # (weights of the keys that are left sum to one per query)
    assert np.abs((mine - base).sum(axis=0) / (61 * hq // hkv) - 1.0).max() <= 2.0 ** -24 * (4 * 200 + 61 * hq // hkv + 64)


def test_observation_refusals(psi, device):
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(25, [64], 24, 4, 256, psi.Dtype.Bfloat16, 16, q_lens=4)
    with pytest.raises(psi.PsiHipError, match="decay"):
        _observe(psi, device, w, _weights(w), [0], 2.0)
    counts = torch.zeros(4, dtype=torch.int32, device=device.torch_device)
    device.bind_replay_counts(counts)
    try:
        with pytest.raises(psi.PsiHipError, match="unbind") as err:
            _observe(psi, device, w, _weights(w), [0], 1.0)
        assert err.value.code == psi._lib.ERR_UNSUPPORTED
    finally:
        device.bind_replay_counts(None)
    kernels = psi.GQAKVObserveKernels(device, _config(psi, w))
    plan = kernels.prepare(w.req_slots, w.token_indices, w.cu_tokens)
    acc = device.from_numpy(_weights(w))
    with pytest.raises(ValueError, match="contiguous rows"):
        kernels.invoke(plan, torch.zeros(3, 24, 256, dtype=torch.bfloat16, device=device.torch_device), None, None, acc, 0)
    with pytest.raises(ValueError, match="float32"):
        kernels.invoke(plan, acc, None, None, acc.double(), 0)


# ------------------------------------------------------------------ selection


def _select(psi, device, lens, values, budget, first, recent, hkv=2, page=16, ids=1, seed=31):
    """(kept, expected) for requests of the given lengths with accumulators drawn by `values(rng, shape)`."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(seed, np.maximum(lens, 1), hkv, hkv, 8, psi.Dtype.Float32, page, num_page_ids_per_block=ids,
                         host_pages=False, **LAYERS)
    rng = np.random.default_rng(seed)
    acc = values(rng, (w.num_pages, hkv, page)).astype(np.float32)
    kernels = psi.GQAKVEvictionKernels(device, _config(psi, w), budget, first, recent)
    plan = kernels.prepare(w.req_slots, lens)
    plan.kept.fill_(77)
    kept = kernels.invoke_select(plan, device.from_numpy(acc), device.from_numpy(w.page_ids), w.layer)
    exp = np.full((len(lens), hkv, budget), -1, np.int64)
    for r, n in enumerate(lens):
        rows, p = page_rows(w, r), np.arange(n)
        for h in range(hkv):
            keep = kept_positions(acc[rows[p // page], h, p % page], n, budget, first, recent)
            exp[r, h, :len(keep)] = keep
    return kept.cpu().numpy(), exp


VALUES = {
    "softmax": lambda rng, s: np.exp(2 * rng.standard_normal(s)) * (rng.random(s) > 0.1),
    "ties": lambda rng, s: rng.integers(0, 3, s),
    "equal": lambda rng, s: np.full(s, 0.25),
    "signed zeros": lambda rng, s: np.where(rng.random(s) < 0.5, 0.0, -0.0),
    "specials": lambda rng, s: rng.choice([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-42, -1e-42, 1.0, -3.0], s),
    "negative": lambda rng, s: -np.exp(rng.standard_normal(s)),
    "one bit apart": lambda rng, s: (0x3f800000 + rng.integers(0, 40, s)).astype(np.uint32).view(np.float32),
}


@pytest.mark.parametrize("values", VALUES, ids=str)
@pytest.mark.parametrize("budget,first,recent", [(1, 0, 0), (48, 4, 17), (48, 20, 28), (300, 0, 1)])
def test_selection(psi, device, values, budget, first, recent):
    lens = [0, 1, budget - 1, budget, budget + 1, 2 * budget + 3, 1023, 1024, 1025, 4096, 5001]
    got, exp = _select(psi, device, lens, VALUES[values], budget, first, recent)
    assert np.array_equal(got, exp)


@pytest.mark.parametrize("lens,hkv,page,ids", [([70001, 65536, 300], 2, 16, 1), ([40000], 8, 8, 4), ([9000, 33], 3, 5, 2),
                                              ([16384, 4097, 8192], 2, 16, 1), (range(17000, 19000, 300), 8, 16, 1),
                                              ([16385, 24576, 24577, 8193, 5], 2, 16, 1),
                                              ([20011, 12289], 2, 7, 1)])
@pytest.mark.parametrize("values", ["softmax", "ties", "equal"])
def test_selection_of_long_requests(psi, device, lens, hkv, page, ids, values):
    for budget, first, recent in ((256, 4, 32), (max(lens) // 2, 16, 100), (max(lens) - 1, 0, 0)):
        got, exp = _select(psi, device, lens, VALUES[values], budget, first, recent, hkv, page, ids)
        assert np.array_equal(got, exp), (budget, first, recent)


def test_selection_counts_unreachable_accumulators_as_lightest(psi, device):
    wl = importlib_workloads(psi)
    w = wl.make_workload(33, [64], 2, 2, 8, psi.Dtype.Float32, 16, host_pages=False, **LAYERS)
    lay = w.layout
    w.page_ids = w.page_ids.copy()
    w.page_ids[(int(w.req_slots[0]) * lay.num_gqa_layers + w.layer) * lay.num_blocks + 1] = 0xfffffff0
    kernels = psi.GQAKVEvictionKernels(device, _config(psi, w), 40, 0, 0)
    plan = kernels.prepare(w.req_slots, [64])
    acc = np.ones((w.num_pages, 2, 16), np.float32)
    kept = kernels.invoke_select(plan, device.from_numpy(acc), device.from_numpy(w.page_ids), w.layer)
    exp = list(range(16)) + list(range(32, 56))
    assert kept.cpu().numpy().tolist() == [[exp, exp]]
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE


# ------------------------------------------------------------------ compaction


def _compact(psi, device, lens, hkv, d, dtype, page, ids, budget, first=1, recent=3, with_weights=True, seed=41, choose=None):
    wl = importlib_workloads(psi)
    w = wl.make_workload(seed, np.maximum(lens, 1), hkv, hkv, d, getattr(psi.Dtype, dtype), page,
                         num_page_ids_per_block=ids, **LAYERS)
    rng = np.random.default_rng(seed)
    acc = _weights(w)
    exp_pages, exp_acc = w.pages.copy(), acc.copy()
    kept = np.full((len(lens), hkv, budget), -1, np.int32)
    for r, n in enumerate(lens):
        keep = []
        for h in range(hkv):
            mine = (choose(rng, n) if choose is not None and n > budget else
                    kept_positions(rng.random(n).astype(np.float32), n, budget, first, recent))
            kept[r, h, :len(mine)] = mine
            keep.append(np.asarray(mine))
        exp_pages, exp_acc = compacted(exp_pages, exp_acc, page_rows(w, r), keep, page)
    kernels = psi.GQAKVEvictionKernels(device, _config(psi, w), budget, first, recent)
    plan = kernels.prepare(w.req_slots, lens)
    pages, weights = device.from_numpy(w.pages.reshape(-1)), device.from_numpy(acc) if with_weights else None
    kernels.invoke_compact(plan, device.from_numpy(kept), pages, weights, device.from_numpy(w.page_ids), w.layer)
    device.sync()
    got = pages.cpu().numpy()
    assert got.tobytes() == exp_pages.tobytes()
    if with_weights:
        assert weights.cpu().numpy().tobytes() == exp_acc.tobytes()
    return w


@pytest.mark.parametrize("hkv,d,dtype,page,ids", [(4, 256, "Bfloat16", 16, 1), (8, 128, "Float16", 8, 2),
                                                  (2, 256, "Float32", 32, 1), (3, 20, "Float32", 5, 3),
                                                  (2, 10, "Bfloat16", 7, 1), (1, 72, "Float16", 16, 1)])
@pytest.mark.parametrize("budget", [1, 47, 640])
def test_compaction(psi, device, hkv, d, dtype, page, ids, budget):
    first, recent = (0, 0) if budget == 1 else (1, 3)
    _compact(psi, device, [0, 1, budget, budget + 1, 3 * budget + 2, 1000, 1601], hkv, d, dtype, page, ids, budget, first,
             recent)


@pytest.mark.parametrize("choose", [lambda rng, n: np.arange(n - 900, n), lambda rng, n: np.arange(900),
                                    lambda rng, n: np.arange(1, 901),
                                    lambda rng, n: np.concatenate([np.arange(450), np.arange(n - 450, n)])],
                         ids=["tail", "front", "one-on", "both-ends"])
@pytest.mark.parametrize("with_weights", [True, False])
def test_compaction_where_source_and_target_overlap(psi, device, choose, with_weights):
    _compact(psi, device, [4001, 901], 2, 256, "Bfloat16", 16, 1, 900, with_weights=with_weights, choose=choose)


def test_compaction_of_a_long_request(psi, device):
    _compact(psi, device, [40000], 1, 128, "Bfloat16", 16, 1, 20000)


@pytest.mark.parametrize("choose", [None, lambda rng, n: np.arange(n - 20000, n), lambda rng, n: np.arange(1, 20001),
                                    lambda rng, n: np.arange(20000) if n % 2 else np.arange(20000) * 2 % n,
                                    lambda rng, n: np.concatenate([np.arange(9001), np.arange(n - 10999, n)]),
                                    lambda rng, n: np.sort(rng.permutation(np.arange(min(3, n - 20000), n))[:20000])],
                         ids=["random", "tail", "one-on", "doubled", "both-ends", "sparse"])
@pytest.mark.parametrize("d,page,ids,with_weights", [(64, 16, 1, True), (32, 5, 3, True), (128, 8, 2, False)])
def test_compaction_of_few_long_requests(psi, device, choose, d, page, ids, with_weights):
    """Entries that only wait for each other in a few steps, and chains of thousands of them."""
    _compact(psi, device, [40000, 20000, 20001, 31111], 1, d, "Float16", page, ids, 20000, with_weights=with_weights,
             choose=choose)


def test_compaction_leaves_out_what_is_no_ascending_choice(psi, device):
    """Entries beyond the cached tokens, below their own index or on pages beyond the arena move nothing; the rest does."""
    wl = importlib_workloads(psi)
    w = wl.make_workload(43, [64], 1, 1, 128, psi.Dtype.Bfloat16, 16, **LAYERS)
    acc = _weights(w)
    kept = np.array([[[3, 0, 5, 64, -1, 9, 10, 40]]], np.int32)
    rows = page_rows(w, 0)
    exp_pages, exp_acc = w.pages.copy(), acc.copy()
    for i, src in ((0, 3), (2, 5), (5, 9), (6, 10)):
        exp_pages[rows[0], :, 0, i] = w.pages[rows[src // 16], :, 0, src % 16]
        exp_acc[rows[0], 0, i] = acc[rows[src // 16], 0, src % 16]
    w.page_ids = w.page_ids.copy()
    w.page_ids[(int(w.req_slots[0]) * 2 + 1) * w.layout.num_blocks + 2] = w.num_pages  # position 40's page
    kernels = psi.GQAKVEvictionKernels(device, _config(psi, w), 8, 0, 0)
    plan = kernels.prepare(w.req_slots, [64])
    pages, weights = device.from_numpy(w.pages.reshape(-1)), device.from_numpy(acc)
    kernels.invoke_compact(plan, device.from_numpy(kept), pages, weights, device.from_numpy(w.page_ids), w.layer)
    assert device.take_device_error() == psi._lib.DEVICE_ERR_CACHE_RANGE
    assert pages.cpu().numpy().tobytes() == exp_pages.tobytes()
    assert weights.cpu().numpy().tobytes() == exp_acc.tobytes()


def test_eviction_refusals(psi, device):
    wl = importlib_workloads(psi)
    w = wl.make_workload(44, [64], 2, 2, 128, psi.Dtype.Bfloat16, 16)
    kernels = psi.GQAKVEvictionKernels(device, _config(psi, w), 8, 0, 0)
    plan = kernels.prepare(w.req_slots, [64])
    pages, acc, ids = device.from_numpy(w.pages.reshape(-1)), device.from_numpy(_weights(w)), device.from_numpy(w.page_ids)
    with pytest.raises(ValueError, match="kept"):
        kernels.invoke_compact(plan, plan.kept[:, :, :4], pages, acc, ids, 0)
    with pytest.raises(ValueError, match="float32"):
        kernels.invoke_select(plan, acc.half(), ids, 0)
    with pytest.raises(psi.PsiHipError, match="layer count"):
        kernels.invoke_select(plan, acc, ids, 1)
    import torch

    counts = torch.zeros(4, dtype=torch.int32, device=device.torch_device)
    device.bind_replay_counts(counts)
    try:
        for call in (lambda: kernels.invoke_select(plan, acc, ids, 0),
                     lambda: kernels.invoke_compact(plan, plan.kept, pages, acc, ids, 0)):
            with pytest.raises(psi.PsiHipError, match="unbind"):
                call()
    finally:
        device.bind_replay_counts(None)


# ------------------------------------------------------------------ together


def test_prompt_to_decode_under_a_budget(psi, oracle, device):
    """As a server uses them: a prompt is observed and cut, then decode steps accumulate and the cache is cut again when
    it has grown.  A plain cache (lists of lines per head) goes through the same; lines and positions are compared bit
    for bit, outputs and accumulators within their bounds."""
    wl = importlib_workloads(psi)
    hq, hkv, d, page, budget, grown = 8, 2, 128, 16, 64, 80
    dtype = psi.Dtype.Bfloat16
    w = wl.make_workload(51, [300, 131, 90], hq, hkv, d, dtype, page, q_lens=[16, 16, 16], **LAYERS)
    pages, acc = device.from_numpy(w.pages.reshape(-1)), psi.page_weights(device, _config(psi, w), w.num_pages)
    ids = device.from_numpy(w.page_ids)
    observe = psi.GQAKVObserveKernels(device, _config(psi, w))
    evict = psi.GQAKVEvictionKernels(device, _config(psi, w), budget, 4, 16)
    cached = w.context_lens.astype(np.int64)
    observe.invoke(observe.prepare(w.req_slots, w.token_indices, w.cu_tokens, [0, 0, 0]),
                   device.from_numpy(w.q.reshape(-1)), pages, ids, acc, w.layer)
    host_pages, host_acc = w.pages.copy(), acc.cpu().numpy()
    exp, bound = attention_weights(w, host_pages, [0, 0, 0], 1.0, np.ones_like(host_acc))
    used = exp != 1.0
    _assert_weights(host_acc[used], exp[used], bound, "prompt")
    for step in range(40):
        if step == 0 or cached.max() >= grown:
            plan = evict.prepare(w.req_slots, cached)
            kept = evict.invoke_select(plan, acc, ids, w.layer)
            evict.invoke_compact(plan, kept, pages, acc, ids, w.layer)
            got = kept.cpu().numpy()
            host_acc = host_acc if step == 0 else before
            for r in range(3):
                rows, p = page_rows(w, r), np.arange(int(cached[r]))
                keep = [kept_positions(host_acc[rows[p // page], h, p % page], int(cached[r]), budget, 4, 16)
                        for h in range(hkv)]
                for h in range(hkv):
                    assert np.array_equal(got[r, h][got[r, h] >= 0], keep[h])
                host_pages, host_acc = compacted(host_pages, host_acc, rows, keep, page)
            assert pages.cpu().numpy().tobytes() == host_pages.tobytes()
            assert acc.cpu().numpy().tobytes() == host_acc.tobytes()
            cached = np.minimum(cached, budget)
        s = wl.make_workload(100 + step, cached + 1, hq, hkv, d, dtype, page, shuffle_slots=False, host_pages=False)
        s.layout, s.layer, s.req_slots, s.page_ids, s.pages = w.layout, w.layer, w.req_slots, w.page_ids, host_pages
        s.num_pages = w.num_pages
        dw = wl.DeviceWorkload(device, s, partition_tokens=64, f32_output=True, balanced=True, pages=pages, page_ids=ids,
                               variant=psi.GQASplitKVVariant.SingleQ(16, 256, 4))
        start = acc.cpu().numpy()
        logits = psi.GQASplitKVSingleQLogits(device, dw.cfg, dw.kshape, grown + 1)
        m = dw.meta
        device.f32_output(True)
        dw.kernels.invoke_attend_weights_bucketed(
            dw.q, pages, m.d_req_slots, m.d_flat_token_indices, ids, m.d_kv_splits, m.d_cu_kv_splits, dw.scratch, logits,
            dw.output, acc, 1.0, w.layer, 3, dw.shape.num_sdpa_map_task_templates, worker_cu=m.d_worker_cu,
            num_workers=m.num_workers, flat_k=dw.flat_k, flat_v=dw.flat_v)
        device.f32_output(False)
        out = dw.output_f32()
        host_pages, exp_out = oracle_step(oracle, s)
        assert_outputs_close(out, exp_out, f"step {step}")
        before = acc.cpu().numpy()
        exp, bound = attention_weights(s, host_pages, s.token_indices, 1.0, start)
        used = np.zeros(exp.shape, bool)
        for r in range(3):
            p = np.arange(int(cached[r]) + 1)
            used[page_rows(w, r)[p // page], :, p % page] = True
        _assert_weights(before[used], exp[used], bound, f"step {step}")
        assert np.array_equal(before[~used], start[~used])
        cached = cached + 1


def test_captured_and_replayed(psi, device):
    """Observe, select, compact and a decode step in one graph, replayed with other work between the replays."""
    import torch

    wl = importlib_workloads(psi)
    w = wl.make_workload(61, [400, 90], 8, 2, 128, psi.Dtype.Bfloat16, 16, q_lens=[8, 8], **LAYERS)
    stream = torch.cuda.Stream()
    dev = psi.Device(0, stream)
    observe = psi.GQAKVObserveKernels(dev, _config(psi, w))
    evict = psi.GQAKVEvictionKernels(dev, _config(psi, w), 64, 4, 8)
    with torch.cuda.stream(stream):
        oplan, eplan = observe.prepare(w.req_slots, w.token_indices, w.cu_tokens, [0, 0]), evict.prepare(w.req_slots, [400, 90])
        q, ids = dev.from_numpy(w.q.reshape(-1)), dev.from_numpy(w.page_ids)
        pages0, pages = dev.from_numpy(w.pages.reshape(-1)), dev.from_numpy(w.pages.reshape(-1))
        acc0 = dev.from_numpy(_weights(w))
        acc = acc0.clone()
        s = wl.make_workload(62, [65, 65], 8, 2, 128, psi.Dtype.Bfloat16, 16, shuffle_slots=False, host_pages=False)
        s.layout, s.layer, s.req_slots, s.page_ids, s.pages, s.num_pages = w.layout, w.layer, w.req_slots, w.page_ids, None, w.num_pages
        dw = wl.DeviceWorkload(dev, s, partition_tokens=64, f32_output=False, balanced=True, pages=pages, page_ids=ids,
                               variant=psi.GQASplitKVVariant.SingleQ(16, 256, 4))
        logits = psi.GQASplitKVSingleQLogits(dev, dw.cfg, dw.kshape, 65)
    m = dw.meta

    def step():
        observe.invoke(oplan, q, pages, ids, acc, w.layer, decay=0.5)
        kept = evict.invoke_select(eplan, acc, ids, w.layer)
        evict.invoke_compact(eplan, kept, pages, acc, ids, w.layer)
        dw.kernels.invoke_attend_weights_bucketed(
            dw.q, pages, m.d_req_slots, m.d_flat_token_indices, ids, m.d_kv_splits, m.d_cu_kv_splits, dw.scratch, logits,
            dw.output, acc, 0.5, w.layer, 2, dw.shape.num_sdpa_map_task_templates, worker_cu=m.d_worker_cu,
            num_workers=m.num_workers, flat_k=dw.flat_k, flat_v=dw.flat_v)

    def state():
        dev.sync()
        return [t.view(torch.uint8).cpu().numpy().copy() for t in (pages, acc, eplan.kept, dw.output)]

    def start():
        with torch.cuda.stream(stream):
            pages.copy_(pages0)
            acc.copy_(acc0)

    start()
    step()
    exp = state()
    graph = torch.cuda.CUDAGraph()
    start()
    dev.sync()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for _ in range(3):
        start()
        with torch.cuda.stream(stream):
            graph.replay()
            got = state()
            torch.randn(1 << 20, device="cuda").sum().item()  # the program's own work between replays
        for a, b in zip(got, exp):
            assert np.array_equal(a, b)
    dev.close()
