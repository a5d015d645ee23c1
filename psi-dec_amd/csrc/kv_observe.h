// Shared declarations of the observation kernels: attention weights of a window of query tokens over its request's
// cached keys, summed per key and KV head and added to the accumulators, without the attention's output:
//     w[h][p] = sum over the window's tokens t with p <= position(t), and over the query heads g of KV head h, of
//               exp2(l[t][g][p] - m[t][g]) / s[t][g],   l = scale * log2(e) * q . k,   m = max_p l,   s = sum_p exp2(l - m).
// The normaliser must be known before a weight is, so the keys are walked twice: a pass for the maximum and sum of every
// (row, column), and a pass that joins those of a window's rows, recomputes the logits and sums the weights.  A row is a
// range of keys of one window (psi_hip_kv_observe_plan), a column a (token of the window, query head of the KV head).  A
// workgroup owns the accumulators of its row, so nothing is added atomically and the result does not depend on the order
// of workgroups.
#pragma once
#include "kv_eviction.h"
#include "split_kv.h"

namespace psi {

struct ObserveArgs {
    CacheView v;
    const void* q;
    const void* pages;
    const uint32_t* windows;
    const uint32_t* rows;
    uint32_t num_windows, num_rows, max_window, num_q_tokens;
    uint32_t hq, group;
    float scale_log2, decay;
    float2* stats;  // [row][kv head][token in window][head of the group]: maximum (log2 domain) and sum
    float2* norm;   // [query row][q head]: maximum and reciprocal sum; null in the second pass: joined there
    float* page_weights;
    uint32_t* status;
};

// A maximum that no key contributes to: finite, so that no difference of two infinities arises.
constexpr float kEmptyMax = -3.0e38f;

// A window's row with every value that a wrong table could hold brought back into range.
struct ObserveRow {
    uint32_t slot, q_begin, num_q, position, held, begin, end, row_begin, row_end;
    bool live;
};
__device__ __forceinline__ ObserveRow load_row(const ObserveArgs& a, uint32_t row) {
    ObserveRow r;
    const uint32_t w = a.rows[(uint64_t)row * 3];
    r.live = w < a.num_windows && a.windows[(uint64_t)w * kWindowWords] < a.v.num_slots;
    const uint32_t* win = a.windows + (uint64_t)(r.live ? w : 0) * kWindowWords;
    r.slot = win[0];
    r.q_begin = min(win[1], a.num_q_tokens);
    r.num_q = min(min(win[2], a.max_window), a.num_q_tokens - r.q_begin);
    r.position = min(win[3], a.v.positions);
    r.held = win[4];
    r.row_begin = win[5];
    r.row_end = min(win[6], a.num_rows);
    r.begin = a.rows[(uint64_t)row * 3 + 1];
    r.end = min(min(a.rows[(uint64_t)row * 3 + 2], r.position + r.num_q), a.v.positions);
    return r;
}

__device__ __forceinline__ uint64_t stat_index(const ObserveArgs& a, uint32_t row, uint32_t kv_head, uint32_t column) {
    return ((uint64_t)row * a.v.hkv + kv_head) * a.max_window * a.group + column;
}

// (m, s) joined with another state of the same column.
__device__ __forceinline__ void join_states(float2 part, float* m, float* s) {
    const float next = fmaxf(*m, part.x);
    *s = *s * exp2f(*m - next) + part.y * exp2f(part.x - next);
    *m = next;
}
// What a weight is made of: exp2(l - x) * y.  +inf and 0 where no key contributes, so that the column's weights are zero.
// (The sum stays out of the exponent: half an ulp of its log2 would be an error of all the column's weights alike.)
__device__ __forceinline__ float2 norm_of_state(float m, float s) {
    return s == 0.0f ? make_float2(INFINITY, 0.0f) : make_float2(m, 1.0f / s);
}
// The states of one column over rows first, first + step, ... before row_end.
__device__ __forceinline__ void join_rows(const ObserveArgs& a, uint32_t first, uint32_t row_end, uint32_t step,
                                          uint32_t kv_head, uint32_t column, float* m, float* s) {
    constexpr uint32_t kAhead = 8;
    for (uint32_t row = first; row < row_end; row += kAhead * step) {
        float2 part[kAhead];
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u)
            part[u] = row + u * step < row_end ? a.stats[stat_index(a, row + u * step, kv_head, column)]
                                               : make_float2(kEmptyMax, 0.0f);
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) join_states(part[u], m, s);
    }
}
// The same by `parts` adjacent lanes (a power of two), each of which gets the normaliser of the column.
__device__ __forceinline__ float2 join_column(const ObserveArgs& a, const ObserveRow& r, uint32_t kv_head, uint32_t column,
                                             uint32_t part, uint32_t parts) {
    float m = kEmptyMax, s = 0.0f;
    join_rows(a, r.row_begin + part, r.row_end, parts, kv_head, column, &m, &s);
    for (uint32_t off = parts / 2; off > 0; off /= 2) {
        const float2 other = make_float2(__shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
        join_states(other, &m, &s);
    }
    return norm_of_state(m, s);
}

// First weights of a position in this call: on top of what counts already.  Later ones: on top of the first.
__device__ __forceinline__ void add_weight(const ObserveArgs& a, const ObserveRow& r, const uint32_t* table,
                                           uint32_t kv_head, uint32_t p, float sum, bool first) {
    const uint32_t page = page_of(a.v, table, p, a.v.num_weight_pages);
    if (page == kNoPage) {
        report_cache_range(a.status);
        return;
    }
    float* acc = a.page_weights + weight_index(a.v, page, kv_head, page_place(a.v, p));
    *acc = (!first ? *acc : p < r.held ? a.decay * *acc : 0.0f) + sum;
}

// The normalisers of all query rows and heads into a.norm, between the two passes.
void launch_observe_join(psi_hip_ctx* ctx, const ObserveArgs& a);

// Matrix-core kernels (kv_observe_kernel.h), one translation unit per element type; head_dim 128 or 256.  window_rows: the
// most rows that one window has.
void launch_observe_bf16(psi_hip_ctx* ctx, const ObserveArgs& a, uint32_t window_rows);
void launch_observe_f16(psi_hip_ctx* ctx, const ObserveArgs& a, uint32_t window_rows);

}  // namespace psi
