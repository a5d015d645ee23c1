"""Plain 64-bit forms of the cache-eviction operators and the bounds their f32 results have to keep."""
import numpy as np

HALF_ULP32 = 2.0 ** -24  # largest relative error of one rounding to f32


def to_f64(stored, dtype):
    """Stored elements (f32, or bf16 / f16 bit patterns) as float64."""
    a = np.asarray(stored)
    if int(dtype) == 0:
        return a.astype(np.float64)
    if int(dtype) == 1:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.view(np.float16).astype(np.float64)


def page_rows(w, r):
    """Page IDs of request r of a workload, layer by its own, as the flat table holds them."""
    lay = w.layout
    per_layer = lay.num_blocks * lay.num_page_ids_per_block
    start = (int(w.req_slots[r]) * lay.num_gqa_layers + w.layer) * per_layer
    return w.page_ids[start:start + per_layer].astype(np.int64)


def softmax_rows(logits):
    m = logits.max(axis=1, keepdims=True)
    e = np.exp(logits - m)
    return e / e.sum(axis=1, keepdims=True)


def attention_weights(w, pages, held, decay, acc):
    """(accumulators after, relative bound per element) of a step or observation whose query rows are w.q at the
    positions of w; pages: storage [pages][2][Hkv][P][D] with the step's own tokens in place; acc: f32 before.

    The bound: a logit sums head_dim exact products in f32, so it is off by at most head_dim half-ulps of
    sum |q_i k_i| (times the scale; the natural exponent's error is the weight's relative error), twice over for the
    normaliser, which also sums up to n terms; the accumulator's product and sums round a few times more."""
    group, page = w.num_q_heads // w.num_kv_heads, w.tokens_per_page
    values = to_f64(pages, w.dtype)
    q = to_f64(w.q, w.dtype).reshape(w.num_tokens, w.num_q_heads, w.head_dim)
    out, bound = acc.astype(np.float64).copy(), 0.0
    for r in range(len(w.req_slots)):
        rows = page_rows(w, r)
        t0, t1 = int(w.cu_tokens[r]), int(w.cu_tokens[r + 1])
        n = int(w.token_indices[r]) + t1 - t0
        p = np.arange(n)
        hidden = p[None, :] > (int(w.token_indices[r]) + np.arange(t1 - t0))[:, None]
        for h in range(w.num_kv_heads):
            k = values[rows[p // page], 0, h, p % page]
            total = np.zeros(n)
            for g in range(h * group, (h + 1) * group):
                s = q[t0:t1, g] @ k.T * w.scale
                total += softmax_rows(np.where(hidden, -np.inf, s)).sum(axis=0)
                size = (np.abs(q[t0:t1, g]) @ np.abs(k).T * w.scale).max()
                bound = max(bound, HALF_ULP32 * (2 * (w.head_dim + 8) * size + n + group * (t1 - t0) + 64))
            at = (rows[p // page], h, p % page)
            out[at] = np.where(p < held[r], decay * out[at], 0.0) + total
    return out, bound


def kept_positions(weights, n, budget, first, recent):
    """Positions kept of n by the rule, ascending: weights f32 [n]."""
    if n <= budget:
        return np.arange(n)
    order = np.where(np.isnan(weights[:n]), -np.inf, weights[:n].astype(np.float64)) + 0.0
    p = np.arange(n)
    always = (p < first) | (p >= n - recent)
    rest = p[~always]
    best = rest[np.lexsort((rest, -order[rest]))][:budget - int(always.sum())]
    return np.sort(np.concatenate([p[always], best]))


def compacted(pages, acc, rows, kept, page):
    """Copies of pages and accumulators after a compaction of one request: kept[h] ascending positions."""
    pages, acc = pages.copy(), acc.copy()
    before_p, before_a = pages.copy(), acc.copy()
    for h, src in enumerate(kept):
        dst = np.arange(len(src))
        pages[rows[dst // page], :, h, dst % page] = before_p[rows[src // page], :, h, src % page]
        acc[rows[dst // page], h, dst % page] = before_a[rows[src // page], h, src % page]
    return pages, acc
