"""Cases of the operators that bound a paged KV cache by what its tokens are attended with.

  attend    decode attention over the paged cache, one new token per sequence, that also adds to every cached token the
            attention weight it received: acc[h][p] = decay * acc[h][p] + sum over the query heads g of KV head h of
            softmax_p(scale * q_g . k_p); tokens appended in the step start from zero
  observe   the same sums for the last tokens of a prompt (causal among them), without the attention's output
  select    per (sequence, KV head) the `budget` tokens to keep: the first `first`, the last `recent`, and of the others
            those with the largest accumulated weight (ties: the lowest index), as ascending indices padded with -1
  compact   moves the kept tokens' K and V lines and accumulators to the front of the sequence's pages, in order

Pages are [K|V][KV heads][tokens per page][head_dim], accumulators f32 [page][KV head][token in page].
"""
import functools
import importlib
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LAYERS, LAYER = 2, 1  # page tables of two layers, of which the second is worked on


def listed():
    return [
        # the lone interactive sequence: 512 cached tokens, where launches and round trips are what counts
        dict(name="attend one of 512 f16", op="attend", batch=1, lo=512, hi=512, hq=16, hkv=2, d=256, page=16,
             dtype="f16", decay=1.0),
        # a handful of short chats of odd lengths on narrow heads and small pages
        dict(name="attend 7 short d128", op="attend", batch=7, lo=101, hi=2903, hq=40, hkv=8, d=128, page=8,
             dtype="f16", decay=0.98),
        # the ordinary serving step: 32 ragged sequences
        dict(name="attend 32 of 1k-8k", op="attend", batch=32, lo=1024, hi=8192, hq=24, hkv=4, d=256, page=16,
             dtype="bf16", decay=1.0),
        # few sequences with very long contexts: the split over the cache's length is all there is to share out
        dict(name="attend 4 of 131072", op="attend", batch=4, lo=131072, hi=131072, hq=16, hkv=2, d=256, page=16,
             dtype="bf16", decay=1.0),
        # a short prompt whose last 8 tokens are taken as the observation
        dict(name="observe 8 of 777 f16", op="observe", batch=1, lo=777, hi=777, window=8, hq=16, hkv=2, d=256, page=16,
             dtype="f16", decay=1.0),
        # a batch of prompts after prefill, 32 tokens observing each
        dict(name="observe 32 of 1k-8k", op="observe", batch=8, lo=1024, hi=8192, window=32, hq=24, hkv=4, d=256,
             page=16, dtype="bf16", decay=1.0),
        # one long document on narrow heads, 64 tokens observing
        dict(name="observe 64 of 65536 d128", op="observe", batch=1, lo=65536, hi=65536, window=64, hq=40, hkv=8, d=128,
             page=16, dtype="bf16", decay=0.9),
        # one short sequence over a small budget
        dict(name="select 256 of 601", op="select", batch=1, lo=601, hi=601, budget=256, first=4, recent=32, hkv=2,
             page=16),
        # the serving batch, cut to 1024 tokens a sequence; the shortest sequences keep everything
        dict(name="select 1024 of 1k-8k", op="select", batch=32, lo=1000, hi=8192, budget=1024, first=4, recent=64,
             hkv=4, page=16),
        # long sequences cut to an eighth
        dict(name="select 16384 of 131072", op="select", batch=4, lo=131072, hi=131072, budget=16384, first=16,
             recent=512, hkv=2, page=16),
        # one sequence cut to a third, small pages
        dict(name="compact 256 of 777 f16", op="compact", batch=1, lo=777, hi=777, budget=256, first=4, recent=32, hkv=8,
             d=128, page=8, dtype="f16"),
        # the serving batch's eviction step
        dict(name="compact 1024 of 1k-8k", op="compact", batch=32, lo=1024, hi=8192, budget=1024, first=4, recent=64,
             hkv=4, d=256, page=16, dtype="bf16"),
    ]


def _spread(rng, lo, hi):
    """A whole number, spread over the logarithm of lo .. hi."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 1e15)


def draw(rng):
    op = rng.choice(["attend", "observe", "select", "compact"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        hkv = rng.choice([1, 2, 4, 8])
        case = dict(op=op, batch=_spread(rng, 1, 64), page=rng.choice([8, 16, 32]), hkv=hkv)
        case["hi"] = _spread(rng, 96, 131072)
        case["lo"] = max(80, case["hi"] // rng.choice([1, 2, 8]))
        if op in ("attend", "observe", "compact"):
            case.update(d=rng.choice([128, 256]), dtype=rng.choice(["bf16", "f16"]))
        if op in ("attend", "observe"):
            case.update(hq=hkv * rng.randint(1, 8), decay=rng.choice([1.0, 0.9, 0.99]))
        if op == "observe":
            case["window"] = _spread(rng, 1, 80)
        if op in ("select", "compact"):
            case.update(first=rng.choice([0, 1, 4, 16]), recent=rng.choice([0, 1, 17, 33]))
            case["budget"] = max(case["first"] + case["recent"] + 1, int(case["hi"] * rng.uniform(0.05, 0.9)))
        padded = case["batch"] * case["hi"] * hkv * case.get("d", 1)
        if _cost(case) <= most and padded <= 4 * 131072 * 2 * 256 and case["batch"] * case["hi"] <= 4 * 131072:
            if op == "observe" and padded // case["d"] * case["window"] * case["hq"] // hkv > 65536 * 64 * 40:
                continue
            return case


def _lengths(case):
    """Cached tokens of each sequence: from lo to hi in equal steps, in a shuffled order."""
    n = np.rint(np.linspace(case["lo"], case["hi"], case["batch"])).astype(np.int64)
    return n[np.random.RandomState(case["batch"]).permutation(case["batch"])]


def _windows(case):
    """Observing tokens of each sequence: the window, some of them a little shorter."""
    return np.maximum(1, case["window"] - np.arange(case["batch"]) % 3)


def work(case):
    n = _lengths(case)
    total, hkv = float(n.sum()), case["hkv"]
    if case["op"] == "select":
        kept = float(np.minimum(n, case["budget"]).sum())
        return {"bytes": hkv * 4 * (total + kept), "flops": hkv * total}
    line = case["d"] * torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "compact":
        # what stands at the front already needs no moving: the first tokens, and all of a sequence under the budget
        moved = float(np.maximum(np.minimum(n, case["budget"]) - case["first"], 0)[n > case["budget"]].sum())
        return {"bytes": moved * hkv * (2 * 2 * line + 2 * 4 + 4), "flops": 0.0}
    if case["op"] == "attend":
        rows = case["batch"] * case["hq"]
        return {"bytes": total * hkv * (2 * line + 8) + 2 * rows * line, "flops": 4.0 * total * case["hq"] * case["d"]}
    w = _windows(case)
    return {"bytes": total * hkv * (line + 8) + float(w.sum()) * case["hq"] * line,
            "flops": 2.0 * float((n * w).sum()) * case["hq"] * case["d"]}


class _State:
    pass


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = np.random.default_rng(seed)
    st = _State()
    st.case, st.n = case, _lengths(case)
    batch, hkv, page, longest = case["batch"], case["hkv"], case["page"], int(st.n.max())
    counts = -(-st.n // page)
    st.num_pages, st.blocks = int(counts.sum()), -(-longest // page)
    st.slots = host.permutation(batch)
    table = np.zeros((batch, LAYERS, st.blocks), np.int32)
    pool, at = host.permutation(st.num_pages).astype(np.int32), 0
    for r in range(batch):
        table[st.slots[r], LAYER, :counts[r]] = pool[at:at + counts[r]]
        at += counts[r]
    st.page_ids = torch.from_numpy(table).to(dev)
    st.slots_t = torch.from_numpy(st.slots).to(dev)
    st.n_t = torch.from_numpy(st.n).to(dev)
    # accumulators as some steps of attention leave them: a few heavy tokens, many light ones, some that underflowed
    acc = torch.randn(st.num_pages, hkv, page, generator=gen, device=dev).mul_(2.0).exp_().mul_(1.0 / longest)
    acc.mul_(torch.rand(acc.shape, generator=gen, device=dev) > 0.05)
    st.page_weights = acc
    if case["op"] != "select":
        dtype = DTYPES[case["dtype"]]
        st.pages = torch.empty(st.num_pages, 2, hkv, page, case["d"], dtype=dtype, device=dev)
        for part in st.pages.split(max(1, (1 << 26) // st.pages[0].numel())):
            part.copy_(torch.randn(part.shape, generator=gen, device=dev))
    if case["op"] in ("attend", "observe"):
        st.scale = 1.0 / math.sqrt(case["d"])
        rows = batch if case["op"] == "attend" else int(_windows(case).sum())
        # queries a little longer than the keys, so that some tokens are attended with much more than others
        st.q = torch.randn(rows, case["hq"], case["d"], generator=gen, device=dev).mul_(1.5).to(dtype)
    if case["op"] == "attend":
        st.output = torch.zeros(batch, case["hq"], case["d"], dtype=dtype, device=dev)
    if case["op"] == "observe":
        st.windows = _windows(case)
        st.first_pos = st.n - st.windows
        # a first pass over a prompt starts from zero, a continued one from what was accumulated before
        st.held = np.where(np.arange(batch) % 2 == 0, 0, st.n // 2)
        st.windows_t, st.held_t = torch.from_numpy(st.windows).to(dev), torch.from_numpy(st.held).to(dev)
    if case["op"] == "compact":
        # a random choice of the shape that `select` gives
        score = torch.rand(batch, hkv, longest, generator=gen, device=dev)
        p = torch.arange(longest, device=dev)
        score[(p < case["first"]).expand_as(score)] = 2.0
        score[(p >= st.n_t[:, None, None] - case["recent"]).expand_as(score)] = 2.0
        score[(p >= st.n_t[:, None, None]).expand_as(score)] = -1.0
        kept = torch.full((batch, hkv, case["budget"]), longest, dtype=torch.int64, device=dev)
        most = min(case["budget"], longest)
        value, index = score.topk(most, dim=2)
        kept[:, :, :most] = torch.where(value >= 0, index, longest)
        kept = kept.sort(dim=2).values
        st.kept = torch.where(kept < longest, kept, -1).to(torch.int32)
    if own:
        _prepare_own(st)
    return st


@functools.lru_cache(maxsize=1)
def _device():
    return importlib.import_module("psi-dec_amd").Device(0)


def _prepare_own(st):
    psi, device, case = importlib.import_module("psi-dec_amd"), _device(), st.case
    dtype = {"bf16": psi.Dtype.Bfloat16, "f16": psi.Dtype.Float16, "f32": psi.Dtype.Float32}[case.get("dtype", "f32")]
    hq, d, batch = case.get("hq", case["hkv"]), case.get("d", 1), case["batch"]
    page_bytes = 2 * case["hkv"] * case["page"] * d * dtype.item_size()
    layout = psi.GQAPageTableLayout(batch, LAYERS, st.blocks, 1)
    if case["op"] == "attend":
        split = psi.GQASplitKVConfig(dtype, page_bytes, hq, case["hkv"], d)
        st.meta = psi.GQAMetadataBuffers(device, batch, max_kv_splits=int((-(-st.n // 512)).sum()))
        st.meta.update_fixed_partition(st.slots, st.n - 1, np.arange(batch + 1), psi.GQASplitKVVariant.SingleQ(16, 256, 8), 512)
        shape = st.meta.balance(psi.balanced_workers(split))
        config = psi.GQASplitKVSingleQConfig(hq, case["hkv"], d, st.scale, page_bytes, layout, 16, 256, 8, dtype)
        kshape = psi.GQASplitKVSingleQShape(batch, shape.num_total_sdpa_map_task_templates)
        st.kernels = psi.GQASplitKVSingleQKernels(device, config, kshape)
        st.scratch = psi.GQASplitKVSingleQScratch(device, config, kshape)
        st.logits = psi.GQASplitKVSingleQLogits(device, config, kshape, int(st.n.max()))
        st.rows = shape.num_sdpa_map_task_templates
        return
    config = psi.GQAKVEvictionConfig(hq, case["hkv"], d, getattr(st, "scale", 1.0), page_bytes, layout, dtype)
    if case["op"] == "observe":
        st.kernels = psi.GQAKVObserveKernels(device, config)
        st.plan = st.kernels.prepare(st.slots, st.first_pos, np.concatenate([[0], np.cumsum(st.windows)]), st.held)
    else:
        st.kernels = psi.GQAKVEvictionKernels(device, config, case["budget"], case["first"], case["recent"])
        st.plan = st.kernels.prepare(st.slots, st.n)


def run(st):
    return {"attend": _attend, "observe": _observe, "select": _select, "compact": _compact}[st.case["op"]](st)


def _positions(st):
    """Page and place in it of every position up to the longest sequence's: [sequence][position], and which exist."""
    p = torch.arange(st.blocks * st.case["page"], device=st.page_ids.device)
    pages = st.page_ids[st.slots_t, LAYER].long().repeat_interleave(st.case["page"], dim=1)
    return pages, (p % st.case["page"]).expand_as(pages), p[None, :] < st.n_t[:, None]


def _lines(st, kind):
    """K (0) or V (1) of every position, [sequence][KV head][position][dim] in 32 bits."""
    x = st.pages[st.page_ids[st.slots_t, LAYER].long(), kind]  # [sequence][page][head][token][dim]
    return x.permute(0, 2, 1, 3, 4).reshape(st.case["batch"], st.case["hkv"], -1, st.case["d"]).float()


def _accumulate(st, weight, held):
    """page_weights at every position: `weight` [sequence][KV head][position] on top of what the first `held` have."""
    pages, places, there = _positions(st)
    p = torch.arange(pages.shape[1], device=pages.device)
    old = st.page_weights[pages, :, places]  # [sequence][position][head]
    new = torch.where((p[None, :] < held[:, None])[:, :, None], st.case["decay"] * old, 0.0) + weight.transpose(1, 2)
    st.page_weights[pages[there], :, places[there]] = new[there]


def _attend(st):
    case = st.case
    if own:
        m = st.meta
        st.kernels.invoke_attend_weights_bucketed(
            st.q, st.pages, m.d_req_slots, m.d_flat_token_indices, st.page_ids, m.d_kv_splits, m.d_cu_kv_splits,
            st.scratch, st.logits, st.output, st.page_weights, case["decay"], LAYER, case["batch"], st.rows,
            worker_cu=m.d_worker_cu, num_workers=m.num_workers)
        return {"output": st.output, "weights": st.page_weights}
    q = st.q.float().view(case["batch"], case["hkv"], -1, case["d"])
    logits = torch.matmul(q, _lines(st, 0).transpose(2, 3)) * st.scale
    there = _positions(st)[2][:, None, None, :]
    logits = logits.masked_fill(~there, -math.inf)
    e = (logits - logits.amax(dim=3, keepdim=True)).exp()
    weight = e / e.sum(dim=3, keepdim=True)
    out = torch.matmul(weight, _lines(st, 1)).view(st.q.shape).to(st.q.dtype)
    _accumulate(st, weight.sum(dim=2), st.n_t - 1)
    return {"output": out, "weights": st.page_weights}


def _observe(st):
    case = st.case
    if own:
        st.kernels.invoke(st.plan, st.q, st.pages, st.page_ids, st.page_weights, LAYER, decay=case["decay"])
        return {"weights": st.page_weights}
    batch, hkv, d, most = case["batch"], case["hkv"], case["d"], int(st.windows.max())
    t = torch.arange(most, device=st.q.device)
    starts = torch.cumsum(st.windows_t, 0) - st.windows_t
    inside = t[None, :] < st.windows_t[:, None]
    q = st.q[(starts[:, None] + t[None, :]).clamp(max=st.q.shape[0] - 1)].float()  # [sequence][token][head][dim]
    q = q.view(batch, most, hkv, -1, d).transpose(1, 2).reshape(batch, hkv, -1, d)
    logits = torch.matmul(q, _lines(st, 0).transpose(2, 3)) * st.scale
    logits = logits.view(batch, hkv, most, -1, logits.shape[-1])
    p = torch.arange(logits.shape[-1], device=st.q.device)
    last = (st.n_t - st.windows_t)[:, None] + t[None, :]
    seen = (p[None, None, :] <= last[:, :, None]) & inside[:, :, None]
    logits = logits.masked_fill(~seen[:, None, :, None, :], -math.inf)
    top = logits.amax(dim=4, keepdim=True)
    e = (logits - torch.where(top.isinf(), 0.0, top)).exp()
    weight = e / e.sum(dim=4, keepdim=True).clamp(min=1e-30)
    _accumulate(st, weight.sum(dim=(2, 3)), st.held_t)
    return {"weights": st.page_weights}


def _select(st):
    case = st.case
    if own:
        return {"kept": st.kernels.invoke_select(st.plan, st.page_weights, st.page_ids, LAYER)}
    pages, places, there = _positions(st)
    score = st.page_weights[pages, :, places].transpose(1, 2)  # [sequence][head][position]
    p = torch.arange(pages.shape[1], device=pages.device)
    always = (p[None, :] < case["first"]) | (p[None, :] >= st.n_t[:, None] - case["recent"])
    score = torch.where(always[:, None, :], math.inf, score)
    score = torch.where(there[:, None, :], score, -math.inf)
    order = score.sort(dim=2, descending=True, stable=True).indices[:, :, :case["budget"]]
    order = torch.where(order < st.n_t[:, None, None], order, len(p)).sort(dim=2).values
    kept = torch.full((case["batch"], case["hkv"], case["budget"]), -1, dtype=torch.int32, device=p.device)
    kept[:, :, :order.shape[2]] = torch.where(order < len(p), order, -1)
    return {"kept": kept}


def _compact(st):
    case = st.case
    if own:
        st.kernels.invoke_compact(st.plan, st.kept, st.pages, st.page_weights, st.page_ids, LAYER)
        return {"pages": st.pages, "weights": st.page_weights}
    r, h, i = torch.nonzero(st.kept >= 0, as_tuple=True)
    src = st.kept[r, h, i].long()
    row = st.page_ids[st.slots_t, LAYER].long()
    from_page, to_page = row[r, src // case["page"]], row[r, i // case["page"]]
    from_place, to_place = src % case["page"], i % case["page"]
    lines = st.pages[from_page, :, h, from_place]
    weights = st.page_weights[from_page, h, from_place]
    st.pages[to_page, :, h, to_place] = lines
    st.page_weights[to_page, h, to_place] = weights
    return {"pages": st.pages, "weights": st.page_weights}


def exact(case, seed):
    st = prepare(case, seed)
    page = case["page"]
    if case["op"] == "select":
        kept = np.full((case["batch"], case["hkv"], case["budget"]), -1, np.int64)
        acc, ids = st.page_weights.double().cpu().numpy(), st.page_ids.cpu().numpy()
        for r, n in enumerate(st.n):
            p = np.arange(n)
            rest = p[(p >= case["first"]) & (p < n - case["recent"])]
            for h in range(case["hkv"]):
                w = acc[ids[st.slots[r], LAYER, p // page], h, p % page]
                best = rest[np.lexsort((rest, -w[rest]))][:max(0, case["budget"] - (n - len(rest)))]
                keep = np.sort(np.concatenate([np.setdiff1d(p, rest), best]))
                kept[r, h, :len(keep)] = keep
        return {"kept": kept.astype(np.int32)}
    ids = st.page_ids.cpu().numpy()
    if case["op"] == "compact":
        kept = st.kept.cpu().numpy()
        pages, acc = st.pages.clone(), st.page_weights.double()
        first = acc.clone()
        for r in range(case["batch"]):
            row = ids[st.slots[r], LAYER].astype(np.int64)
            for h in range(case["hkv"]):
                src = kept[r, h][kept[r, h] >= 0].astype(np.int64)
                dst = np.arange(len(src))
                a, b = torch.from_numpy(row[src // page]).to(acc.device), torch.from_numpy(row[dst // page]).to(acc.device)
                x, y = torch.from_numpy(src % page).to(acc.device), torch.from_numpy(dst % page).to(acc.device)
                pages[b, 0, h, y], pages[b, 1, h, y] = st.pages[a, 0, h, x], st.pages[a, 1, h, x]
                acc[b, h, y] = first[a, h, x]
        return {"pages": pages, "weights": acc}
    # attention weights of one KV head's queries at a time
    acc = st.page_weights.double()
    group, per = case["hq"] // case["hkv"], [1] * case["batch"] if case["op"] == "attend" else list(st.windows)
    out = torch.zeros(st.q.shape, dtype=torch.float64, device=acc.device)
    at = 0
    for r, n in enumerate(int(v) for v in st.n):
        t, held = int(per[r]), n - 1 if case["op"] == "attend" else int(st.held[r])
        p = np.arange(n)
        rows = torch.from_numpy(ids[st.slots[r], LAYER, p // page].astype(np.int64)).to(acc.device)
        place = torch.from_numpy(p % page).to(acc.device)
        where = torch.arange(n, device=acc.device)
        limit = n - t + torch.arange(t, device=acc.device)
        for h in range(case["hkv"]):
            k, v = (st.pages[rows, kind, h, place].double() for kind in (0, 1))
            total = torch.zeros(n, dtype=torch.float64, device=acc.device)
            for g in range(h * group, (h + 1) * group):
                s = st.q[at:at + t, g].double() @ k.T * st.scale
                w = torch.softmax(s.masked_fill(where[None, :] > limit[:, None], -math.inf), dim=1)
                total += w.sum(dim=0)
                if case["op"] == "attend":
                    out[at:at + t, g] = w @ v
            acc[rows, h, place] = torch.where(where < held, case["decay"] * acc[rows, h, place], 0.0) + total
        at += t
    return {"output": out, "weights": acc} if case["op"] == "attend" else {"weights": acc}
