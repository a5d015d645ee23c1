// Observation: the shape-generic kernels and the entry point; what is computed and how it is shared out: kv_observe.h.
#include "kv_observe.h"

namespace psi {

constexpr float kLog2eObserve = 1.4426950408889634f;

template <typename Tag>
__device__ __forceinline__ float dot_line(const ObserveArgs& a, uint64_t q_off, uint64_t k_off) {
    float dot = 0.0f;
    for (uint32_t i = 0; i < a.v.d; ++i)
        dot += load_as_f32<Tag>(a.q, q_off + i) * load_as_f32<Tag>(a.pages, k_off + i);
    return dot;
}

// Any head_dim, page size and type.  One wave per (row, query head); lane = key.  Bound by the scalar products: 8 prompts of
// 1k-8k, 32 tokens, 24 heads over 4, take 13 ms with bf16 and D 64, 47 ms with f32 and D 256 (the matrix-core kernels 0.06
// ms with bf16 and D 256).
template <typename Tag>
__global__ __launch_bounds__(64) void observe_stats_generic(ObserveArgs a) {
    const uint32_t row = blockIdx.x / a.hq, head = blockIdx.x % a.hq, kv_head = head / a.group, lane = threadIdx.x;
    const ObserveRow r = load_row(a, row);
    if (!r.live) return;
    const uint32_t* table = table_row(a.v, r.slot, a.v.layer);
    for (uint32_t t = 0; t < r.num_q; ++t) {
        const uint64_t q_off = ((uint64_t)(r.q_begin + t) * a.hq + head) * a.v.d;
        const uint32_t end = min(r.end, r.position + t + 1);
        float m = kEmptyMax, s = 0.0f;
        for (uint32_t p = r.begin + lane; p < end; p += 64) {
            const uint32_t page = page_of(a.v, table, p, a.v.num_pages);
            if (page == kNoPage) {
                report_cache_range(a.status);
                continue;
            }
            const float l = dot_line<Tag>(a, q_off, line_index(a.v, page, 0, kv_head, page_place(a.v, p))) * a.scale_log2;
            const float next = fmaxf(m, l);
            s = s * exp2f(m - next) + exp2f(l - next);
            m = next;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const float om = __shfl_xor(m, off, 64), os = __shfl_xor(s, off, 64), next = fmaxf(m, om);
            s = s * exp2f(m - next) + os * exp2f(om - next);
            m = next;
        }
        if (lane == 0) a.stats[stat_index(a, row, kv_head, t * a.group + head % a.group)] = make_float2(m, s);
    }
}

// One workgroup per (window, 32 (query row, head) items): eight threads share the rows of an item.
constexpr uint32_t kJoinItems = 32, kJoinParts = 8;
__global__ __launch_bounds__(kJoinItems * kJoinParts) void observe_join(ObserveArgs a) {
    const uint32_t* win = a.windows + (uint64_t)blockIdx.y * kWindowWords;
    const uint32_t q_begin = min(win[1], a.num_q_tokens), num_q = min(min(win[2], a.max_window), a.num_q_tokens - q_begin);
    const uint32_t row_begin = win[5], row_end = min(win[6], a.num_rows);
    const uint32_t item = blockIdx.x * kJoinItems + threadIdx.x % kJoinItems, part = threadIdx.x / kJoinItems;
    __shared__ float2 parts[kJoinParts][kJoinItems];
    // items in the order of the statistics: KV head, token, head of the group
    const uint32_t columns = num_q * a.group, kv_head = item / max(columns, 1u), column = item % max(columns, 1u);
    const bool live = item < columns * a.v.hkv;
    float m = kEmptyMax, s = 0.0f;
    if (live) join_rows(a, row_begin + part, row_end, kJoinParts, kv_head, column, &m, &s);
    parts[part][threadIdx.x % kJoinItems] = make_float2(m, s);
    __syncthreads();
    if (part != 0 || !live) return;
    for (uint32_t i = 1; i < kJoinParts; ++i) join_states(parts[i][threadIdx.x], &m, &s);
    a.norm[(uint64_t)(q_begin + column / a.group) * a.hq + kv_head * a.group + column % a.group] = norm_of_state(m, s);
}

void launch_observe_join(psi_hip_ctx* ctx, const ObserveArgs& a) {
    const dim3 grid((a.max_window * a.hq + kJoinItems - 1) / kJoinItems, a.num_windows);
    hipLaunchKernelGGL(observe_join, grid, dim3(kJoinItems * kJoinParts), 0, ctx->stream, a);
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
                const float2 norm = a.norm[at];
                sum += exp2f(dot_line<Tag>(a, at * a.v.d, k_off) * a.scale_log2 - norm.x) * norm.y;
            }
            total += sum;
        }
        add_weight(a, r, table, kv_head, p, total, true);
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
    return psi_hip_kv_observe_weights_rows(ctx, cfg, layout, q, num_q_tokens, kv_pages, kv_pages_bytes, page_ids, windows,
                                           num_windows, max_window, rows, num_rows, 0, scratch, scratch_bytes,
                                           page_weights, page_weights_bytes, decay, gqa_layer_index);
}

extern "C" int psi_hip_kv_observe_weights_rows(psi_hip_ctx* ctx, const psi_hip_gqa_config* cfg,
                                               const psi_hip_page_table_layout* layout, const void* q,
                                               uint32_t num_q_tokens, const void* kv_pages, uint64_t kv_pages_bytes,
                                               const uint32_t* page_ids, const uint32_t* windows, uint32_t num_windows,
                                               uint32_t max_window, const uint32_t* rows, uint32_t num_rows,
                                               uint32_t max_window_rows, void* scratch, uint64_t scratch_bytes,
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
    const uint64_t needed = (stats + (uint64_t)num_q_tokens * g.hq) * sizeof(float2);
    PSI_REQUIRE(scratch_bytes >= needed, "observation scratch too small: %llu < %llu", (unsigned long long)scratch_bytes,
                (unsigned long long)needed);
    PSI_REQUIRE(reinterpret_cast<uintptr_t>(scratch) % 8 == 0, "the observation scratch must be 8-byte aligned");
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
    a.stats = static_cast<float2*>(scratch);
    a.norm = a.stats + stats;
    a.page_weights = page_weights;
    a.status = ctx->status_device;

    DeviceGuard guard(ctx->device);
    LaunchScope scope(ctx, "kv_observe");
    auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool two_byte = g.dtype == PSI_HIP_BF16 || g.dtype == PSI_HIP_F16;
    if (!ctx->force_generic && two_byte && (g.d == 128 || g.d == 256) && aligned(q) && aligned(kv_pages)) {
        // not told: as many as there can be, if every window has one at least
        const uint32_t most = num_rows > num_windows ? num_rows - num_windows + 1 : 1;
        const uint32_t window_rows = max_window_rows != 0 ? max_window_rows : most;
        if (g.dtype == PSI_HIP_BF16) launch_observe_bf16(ctx, a, window_rows);
        else launch_observe_f16(ctx, a, window_rows);
        PSI_HIP_CHECK(hipGetLastError());
        return PSI_HIP_OK;
    }
    const dim3 stats_grid(num_rows * g.hq), sum_grid(num_rows * g.hkv);
#define PSI_OBSERVE(TAG)                                                                                   \
    do {                                                                                                   \
        hipLaunchKernelGGL(observe_stats_generic<TAG>, stats_grid, dim3(64), 0, ctx->stream, a);           \
        launch_observe_join(ctx, a);                                                                       \
        hipLaunchKernelGGL(observe_sum_generic<TAG>, sum_grid, dim3(256), 0, ctx->stream, a);              \
    } while (0)
    if (g.dtype == PSI_HIP_F32) PSI_OBSERVE(F32Tag);
    else if (g.dtype == PSI_HIP_BF16) PSI_OBSERVE(BF16Tag);
    else PSI_OBSERVE(F16Tag);
#undef PSI_OBSERVE
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
