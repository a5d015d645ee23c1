// Attention weights of a window of query tokens over its request's cached keys, summed per key and KV head and added to
// the accumulators -- the observation from which a prompt's cache is cut, without the attention's output:
//     w[h][p] = sum over the window's tokens t with p <= position(t), and over the query heads g of KV head h, of
//               exp2(l[t][g][p] - lse[t][g]),   l = scale * log2(e) * q . k,   lse = log2 sum_p exp2(l).
// The normaliser must be known before a weight is, so the keys are walked twice: a pass for the maximum and sum of every
// (row, token, head), a small join over a window's rows, and a pass that recomputes the logits and sums the weights.  A
// row is a range of keys of one window (psi_hip_kv_observe_plan); a workgroup owns the accumulators of its row, so
// nothing is added atomically and the result does not depend on the order of workgroups.
#include "kv_eviction.h"
#include "split_kv.h"

namespace psi {

constexpr float kLog2eObserve = 1.4426950408889634f;

struct ObserveArgs {
    CacheView v;
    const void* q;
    const void* pages;
    const uint32_t* windows;
    const uint32_t* rows;
    uint32_t num_windows, num_rows, max_window, num_q_tokens;
    uint32_t hq, group;
    float scale_log2, decay;
    float* stat_max;  // [row][token in window][q head], log2 domain
    float* stat_sum;
    float* lse;       // [query row][q head]
    float* page_weights;
    uint32_t* status;
};

// A window's row with every value that a wrong table could hold brought back into range.
struct ObserveRow {
    uint32_t slot, q_begin, num_q, position, held, begin, end;
    bool live;
};
__device__ __forceinline__ ObserveRow load_row(const ObserveArgs& a, uint32_t row) {
    ObserveRow r;
    const uint32_t w = a.rows[row * 3];
    r.live = w < a.num_windows && a.windows[(uint64_t)w * kWindowWords] < a.v.num_slots;
    const uint32_t* win = a.windows + (uint64_t)(r.live ? w : 0) * kWindowWords;
    r.slot = win[0];
    r.q_begin = min(win[1], a.num_q_tokens);
    r.num_q = min(min(win[2], a.max_window), a.num_q_tokens - r.q_begin);
    r.position = win[3];
    r.held = win[4];
    r.begin = a.rows[row * 3 + 1];
    r.end = min(min(a.rows[row * 3 + 2], r.position + r.num_q), a.v.positions);
    return r;
}

template <typename Tag>
__device__ __forceinline__ float dot_line(const ObserveArgs& a, uint64_t q_off, uint64_t k_off) {
    float dot = 0.0f;
    for (uint32_t i = 0; i < a.v.d; ++i)
        dot += load_as_f32<Tag>(a.q, q_off + i) * load_as_f32<Tag>(a.pages, k_off + i);
    return dot;
}

// Any head_dim, page size and type.  One wave per (row, query head); lane = key.
template <typename Tag>
__global__ __launch_bounds__(64) void observe_stats_generic(ObserveArgs a) {
    const uint32_t row = blockIdx.x / a.hq, head = blockIdx.x % a.hq, kv_head = head / a.group, lane = threadIdx.x;
    const ObserveRow r = load_row(a, row);
    if (!r.live) return;
    const uint32_t* table = table_row(a.v, r.slot, a.v.layer);
    for (uint32_t t = 0; t < r.num_q; ++t) {
        const uint64_t q_off = ((uint64_t)(r.q_begin + t) * a.hq + head) * a.v.d;
        const uint32_t end = min(r.end, r.position + t + 1);
        float m = -INFINITY, s = 0.0f;
        for (uint32_t p = r.begin + lane; p < end; p += 64) {
            const uint32_t page = page_of(a.v, table, p, a.v.num_pages);
            if (page == kNoPage) {
                report_cache_range(a.status);
                continue;
            }
            const float l = dot_line<Tag>(a, q_off, line_index(a.v, page, 0, kv_head, page_place(a.v, p))) * a.scale_log2;
            const float next = fmaxf(m, l);
            s = (m > -INFINITY ? s * exp2f(m - next) : 0.0f) + (l == -INFINITY ? 0.0f : exp2f(l - next));
            m = next;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const float om = __shfl_xor(m, off, 64), os = __shfl_xor(s, off, 64), next = fmaxf(m, om);
            s = (m > -INFINITY ? s * exp2f(m - next) : s) + (om > -INFINITY ? os * exp2f(om - next) : os);
            m = next;
        }
        if (lane == 0) {
            const uint64_t at = ((uint64_t)row * a.max_window + t) * a.hq + head;
            a.stat_max[at] = m;
            a.stat_sum[at] = s;
        }
    }
}

// lse of every query row and head from its window's rows; +inf where no key contributes, so that its weights are zero.
__global__ __launch_bounds__(256) void observe_join(ObserveArgs a) {
    const uint32_t* win = a.windows + (uint64_t)blockIdx.y * kWindowWords;
    const uint32_t q_begin = min(win[1], a.num_q_tokens), num_q = min(min(win[2], a.max_window), a.num_q_tokens - q_begin);
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;
    if (item >= num_q * a.hq) return;
    const uint32_t row_end = min(win[6], a.num_rows);
    float m = -INFINITY, s = 0.0f;
    for (uint32_t row = win[5]; row < row_end; ++row) {
        const uint64_t at = (uint64_t)row * a.max_window * a.hq + item;
        const float rm = a.stat_max[at], rs = a.stat_sum[at], next = fmaxf(m, rm);
        s = (m > -INFINITY ? s * exp2f(m - next) : s) + (rm > -INFINITY ? rs * exp2f(rm - next) : rs);
        m = next;
    }
    a.lse[(uint64_t)q_begin * a.hq + item] = m > -INFINITY || s != s ? m + log2f(s) : INFINITY;
}

__device__ __forceinline__ void add_weight(const ObserveArgs& a, const ObserveRow& r, const uint32_t* table,
                                           uint32_t kv_head, uint32_t p, float sum) {
    const uint32_t page = page_of(a.v, table, p, a.v.num_weight_pages);
    if (page == kNoPage) {
        report_cache_range(a.status);
        return;
    }
    float* acc = a.page_weights + weight_index(a.v, page, kv_head, page_place(a.v, p));
    *acc = (p < r.held ? a.decay * *acc : 0.0f) + sum;
}

// One workgroup per (row, KV head); thread = key.  The sum of one token's heads is added to the total as one number, so
// that a window of T tokens and G heads loses about T + G roundings and not T * G.
template <typename Tag>
__global__ __launch_bounds__(256) void observe_sum_generic(ObserveArgs a) {
    const uint32_t row = blockIdx.x / a.v.hkv, kv_head = blockIdx.x % a.v.hkv;
    const ObserveRow r = load_row(a, row);
    if (!r.live) return;
    const uint32_t* table = table_row(a.v, r.slot, a.v.layer);
    for (uint32_t p = r.begin + threadIdx.x; p < r.end; p += 256) {
        const uint32_t page = page_of(a.v, table, p, a.v.num_pages);
        if (page == kNoPage) continue;
        const uint64_t k_off = line_index(a.v, page, 0, kv_head, page_place(a.v, p));
        float total = 0.0f;
        for (uint32_t t = p > r.position ? p - r.position : 0; t < r.num_q; ++t) {
            float sum = 0.0f;
            for (uint32_t g = 0; g < a.group; ++g) {
                const uint64_t at = (uint64_t)(r.q_begin + t) * a.hq + kv_head * a.group + g;
                sum += exp2f(dot_line<Tag>(a, at * a.v.d, k_off) * a.scale_log2 - a.lse[at]);
            }
            total += sum;
        }
        add_weight(a, r, table, kv_head, p, total);
    }
}

}  // namespace psi

using namespace psi;

extern "C" int psi_hip_kv_observe_weights(psi_hip_ctx* ctx, const psi_hip_gqa_config* cfg,
                                          const psi_hip_page_table_layout* layout, const void* q, uint32_t num_q_tokens,
                                          const void* kv_pages, uint64_t kv_pages_bytes, const uint32_t* page_ids,
                                          const uint32_t* windows, uint32_t num_windows, uint32_t max_window,
                                          const uint32_t* rows, uint32_t num_rows, void* scratch, uint64_t scratch_bytes,
                                          float* page_weights, uint64_t page_weights_bytes, float decay,
                                          uint32_t gqa_layer_index) {
    PSI_REQUIRE(ctx != nullptr, "ctx must not be null");
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    rc = check_no_replay_counts(ctx);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(g.scale > 0.0f, "GQA attention scale must be positive");
    PSI_REQUIRE(q && kv_pages && windows && rows && scratch && page_weights, "observation buffers must not be null");
    PSI_REQUIRE(num_q_tokens > 0 && num_windows > 0 && num_rows > 0 && max_window > 0, "an observation needs query tokens");
    PSI_REQUIRE(max_window <= num_q_tokens, "the longest window exceeds the query rows");
    PSI_REQUIRE(decay >= 0.0f && decay <= 1.0f, "the decay must lie in [0, 1]");
    ObserveArgs a;
    rc = make_cache_view(g, layout, page_ids, gqa_layer_index, kv_pages_bytes, page_weights_bytes, &a.v);
    if (rc != PSI_HIP_OK) return rc;
    const uint64_t stats = (uint64_t)num_rows * max_window * g.hq;
    const uint64_t needed = (2 * stats + (uint64_t)num_q_tokens * g.hq) * 4;
    PSI_REQUIRE(scratch_bytes >= needed, "observation scratch too small: %llu < %llu", (unsigned long long)scratch_bytes,
                (unsigned long long)needed);
    PSI_REQUIRE((uint64_t)num_rows * g.hq <= 0x7fffffffull && num_windows <= 65535 &&
                    (uint64_t)max_window * g.hq <= 0x7fffffffull,
                "an observation of this size exceeds the launch grid");
    a.q = q;
    a.pages = kv_pages;
    a.windows = windows;
    a.rows = rows;
    a.num_windows = num_windows;
    a.num_rows = num_rows;
    a.max_window = max_window;
    a.num_q_tokens = num_q_tokens;
    a.hq = g.hq;
    a.group = g.group;
    a.scale_log2 = g.scale * kLog2eObserve;
    a.decay = decay;
    a.stat_max = static_cast<float*>(scratch);
    a.stat_sum = a.stat_max + stats;
    a.lse = a.stat_sum + stats;
    a.page_weights = page_weights;
    a.status = ctx->status_device;

    DeviceGuard guard(ctx->device);
    LaunchScope scope(ctx, "kv_observe");
    const dim3 stats_grid(num_rows * g.hq), sum_grid(num_rows * g.hkv), join_grid((max_window * g.hq + 255) / 256, num_windows);
#define PSI_OBSERVE(TAG)                                                                                   \
    do {                                                                                                   \
        hipLaunchKernelGGL(observe_stats_generic<TAG>, stats_grid, dim3(64), 0, ctx->stream, a);           \
        hipLaunchKernelGGL(observe_join, join_grid, dim3(256), 0, ctx->stream, a);                         \
        hipLaunchKernelGGL(observe_sum_generic<TAG>, sum_grid, dim3(256), 0, ctx->stream, a);              \
    } while (0)
    if (g.dtype == PSI_HIP_F32) PSI_OBSERVE(F32Tag);
    else if (g.dtype == PSI_HIP_BF16) PSI_OBSERVE(BF16Tag);
    else PSI_OBSERVE(F16Tag);
#undef PSI_OBSERVE
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
