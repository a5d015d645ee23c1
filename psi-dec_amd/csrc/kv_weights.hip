// Decode attention that also says what its keys were attended with: the split-KV map stores its logits beside the
// partial states (split_kv_decode_kernel.h, kLogits), the combine gives every (token, head) row its maximum and sum,
// and the kernel below turns the logits into weights,
//     w[h][p] = sum over the step's tokens t of the request, p <= position(t), and over the query heads g of KV head h of
//               exp2(logit[t][g][p] - max[t][g]) / sum[t][g],
// and adds them to the accumulators:  acc = (p appended before this step ? decay * acc : 0) + w.
#include "kv_eviction.h"
#include "split_kv.h"

namespace psi {

struct WeightsArgs {
    CacheView v;
    const float* logits;
    uint64_t logits_stride;
    const float* part_max;
    const float* part_sum;
    const uint32_t* cu_kv_splits;
    const uint32_t* row_index;
    const uint32_t* kv_splits;
    const uint32_t* req_slots;
    const uint32_t* flat_token_indices;
    float* page_weights;
    float decay;
    uint32_t hq, group, max_context, num_active_tokens, num_active_kv_splits;
    const uint32_t* replay_counts;
    uint32_t* status;
};

constexpr uint32_t kLseEntries = 512;  // (token, head) normalisers held in LDS at a time

// One workgroup per (kv_split row, KV head).  The rows of a request's last token of the step tile all its positions, so
// those rows' workgroups own the accumulators they cover and the others have nothing to do: no two workgroups meet.
__global__ __launch_bounds__(256) void accumulate_weights_kernel(WeightsArgs a) {
    const uint32_t num_tokens = active_count(a.replay_counts, kReplayTokens, a.num_active_tokens);
    const uint32_t num_splits = active_count(a.replay_counts, kReplaySplits, a.num_active_kv_splits);
    const uint32_t layer = active_layer(a.replay_counts, a.v.layer, a.v.num_layers);
    const uint32_t split = blockIdx.x / a.v.hkv, kv_head = blockIdx.x % a.v.hkv;
    if (split >= num_splits) return;
    const uint32_t token = a.kv_splits[split * 3];
    if (token >= num_tokens) return;
    const uint32_t slot = a.req_slots[token];
    if (token + 1 < num_tokens && a.req_slots[token + 1] == slot) return;
    uint32_t first = token;
    while (first > 0 && a.req_slots[first - 1] == slot) --first;
    const uint32_t held = a.flat_token_indices[first];
    const uint32_t begin = a.kv_splits[split * 3 + 1];
    const uint32_t row_end = a.kv_splits[split * 3 + 2], end = min(row_end, a.max_context);
    if (threadIdx.x == 0 && row_end > end) report_cache_range(a.status);
    const uint32_t* row = table_row(a.v, slot, layer);

    __shared__ float lse[kLseEntries];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t entries = (token - first + 1) * a.group;
    for (uint32_t base = 0; base < entries; base += kLseEntries) {
        const uint32_t count = min(kLseEntries, entries - base);
        for (uint32_t e = wave; e < count; e += 4) {
            const uint32_t t = first + (base + e) / a.group, head = kv_head * a.group + (base + e) % a.group;
            const uint32_t p0 = a.cu_kv_splits[t], p1 = a.cu_kv_splits[t + 1];
            float m = -INFINITY, s = 0.0f;
            for (uint32_t p = p0 + lane; p < p1; p += 64) {
                const uint64_t r = (uint64_t)(a.row_index ? a.row_index[p] : p) * a.hq + head;
                const float pm = a.part_max[r], next = fmaxf(m, pm);
                if (pm > -INFINITY) s = s * exp2f(m - next) + a.part_sum[r] * exp2f(pm - next);
                m = next;
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) {
                const float om = __shfl_xor(m, off, 64), os = __shfl_xor(s, off, 64), next = fmaxf(m, om);
                if (next > -INFINITY) s = s * exp2f(m - next) + os * exp2f(om - next);
                m = next;
            }
            // a row that nothing contributes to has weights of zero
            if (lane == 0) lse[e] = m > -INFINITY ? m + log2f(s) : INFINITY;
        }
        __syncthreads();
        for (uint32_t p = begin + threadIdx.x; p < end; p += 256) {
            float sum = 0.0f;
            for (uint32_t e = 0; e < count; ++e) {
                const uint32_t t = first + (base + e) / a.group, head = kv_head * a.group + (base + e) % a.group;
                if (p <= a.flat_token_indices[t])
                    sum += exp2f(a.logits[((uint64_t)t * a.hq + head) * a.logits_stride + p] - lse[e]);
            }
            const uint32_t page = page_of(a.v, row, p, a.v.num_weight_pages);
            if (page == kNoPage) {
                report_cache_range(a.status);
                continue;
            }
            float* acc = a.page_weights + weight_index(a.v, page, kv_head, page_place(a.v, p));
            const float old = base > 0 ? *acc : p < held ? a.decay * *acc : 0.0f;
            *acc = old + sum;
        }
        __syncthreads();
    }
}

static uint64_t logits_stride(uint32_t max_context_tokens) { return ((uint64_t)max_context_tokens + 15) / 16 * 16; }

}  // namespace psi

using namespace psi;

extern "C" int psi_hip_split_kv_single_q_logits_bytes(const psi_hip_gqa_config* cfg, uint32_t num_total_tokens,
                                                      uint32_t max_context_tokens, uint64_t* out_bytes) {
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(out_bytes != nullptr, "out pointer must not be null");
    PSI_REQUIRE(num_total_tokens > 0 && max_context_tokens > 0, "logits need tokens and a context");
    *out_bytes = (uint64_t)num_total_tokens * g.hq * logits_stride(max_context_tokens) * 4;
    return PSI_HIP_OK;
}

extern "C" int psi_hip_split_kv_single_q_attend_weights(
    psi_hip_ctx* ctx, const psi_hip_gqa_config* cfg, const psi_hip_page_table_layout* layout, const void* q,
    void* kv_pages, uint64_t kv_pages_bytes, const void* flat_k, const void* flat_v, const uint32_t* req_slots,
    const uint32_t* flat_token_indices, const uint32_t* page_ids, const uint32_t* kv_splits,
    const uint32_t* cu_kv_splits, const uint32_t* worker_cu, uint32_t num_workers, const uint32_t* partial_row_index,
    void* scratch, uint64_t scratch_bytes, void* output, const psi_hip_output_gate* gate,
    const psi_hip_kv_weights* weights, uint32_t gqa_layer_index, uint32_t num_total_tokens,
    uint32_t num_total_kv_splits, uint32_t num_active_tokens, uint32_t num_active_kv_splits) {
    PSI_REQUIRE(ctx != nullptr && weights != nullptr, "ctx and weights must not be null");
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE((worker_cu == nullptr) == (num_workers == 0), "a worker table needs its worker count and vice versa");
    PSI_REQUIRE((flat_k == nullptr) == (flat_v == nullptr), "GQA KV page write needs K and V rows or neither");
    PSI_REQUIRE(flat_token_indices && weights->page_weights && weights->logits && cu_kv_splits && output,
                "weight accumulation buffers must not be null");
    PSI_REQUIRE(weights->decay >= 0.0f && weights->decay <= 1.0f, "the decay must lie in [0, 1]");
    PSI_REQUIRE(num_total_tokens > 0 && weights->max_context_tokens > 0, "logits need tokens and a context");
    PSI_REQUIRE(reinterpret_cast<uintptr_t>(weights->logits) % 16 == 0, "the logits must be 16-byte aligned");
    uint64_t needed = 0;
    rc = psi_hip_split_kv_single_q_logits_bytes(cfg, num_total_tokens, weights->max_context_tokens, &needed);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(weights->logits_bytes >= needed, "logits buffer too small: %llu < %llu",
                (unsigned long long)weights->logits_bytes, (unsigned long long)needed);
    WeightsArgs a;
    rc = make_cache_view(g, layout, page_ids, gqa_layer_index, kv_pages_bytes, weights->page_weights_bytes, &a.v);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE((uint64_t)num_total_kv_splits * g.hkv <= 0x7fffffffull, "too many KV splits");

    DeviceGuard guard(ctx->device);
    float* logits = static_cast<float*>(weights->logits);
    const uint64_t stride = logits_stride(weights->max_context_tokens);
    rc = single_q_map_impl(ctx, cfg, layout, q, kv_pages, kv_pages_bytes, req_slots, page_ids, kv_splits, worker_cu,
                           num_workers, scratch, scratch_bytes, gqa_layer_index, num_total_tokens, num_total_kv_splits,
                           num_active_tokens, num_active_kv_splits, flat_k, flat_v, flat_token_indices, logits, stride);
    if (rc != PSI_HIP_OK) return rc;
    rc = psi_hip_split_kv_single_q_reduce(ctx, cfg, scratch, scratch_bytes, cu_kv_splits, output, num_total_tokens,
                                          num_total_kv_splits, num_active_tokens, partial_row_index, gate);
    if (rc != PSI_HIP_OK) return rc;

    const PartialLayout pl = partial_layout(num_total_kv_splits, g.hq, g.d, 1);
    a.logits = logits;
    a.logits_stride = stride;
    a.part_max = reinterpret_cast<const float*>(static_cast<const char*>(scratch) + pl.max_offset);
    a.part_sum = reinterpret_cast<const float*>(static_cast<const char*>(scratch) + pl.sum_offset);
    a.cu_kv_splits = cu_kv_splits;
    a.row_index = partial_row_index;
    a.kv_splits = kv_splits;
    a.req_slots = req_slots;
    a.flat_token_indices = flat_token_indices;
    a.page_weights = weights->page_weights;
    a.decay = weights->decay;
    a.hq = g.hq;
    a.group = g.group;
    a.max_context = weights->max_context_tokens < a.v.positions ? weights->max_context_tokens : a.v.positions;
    a.num_active_tokens = num_active_tokens;
    a.num_active_kv_splits = num_active_kv_splits;
    a.replay_counts = ctx->replay_counts;
    a.status = ctx->status_device;
    LaunchScope scope(ctx, "kv_weights");
    hipLaunchKernelGGL(accumulate_weights_kernel, dim3(num_active_kv_splits * g.hkv), dim3(256), 0, ctx->stream, a);
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
