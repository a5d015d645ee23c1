// Decode attention that also says what its keys were attended with: the split-KV map stores its logits beside the
// partial states (split_kv_decode_kernel.h, kLogits), the combine gives every (token, head) row its maximum and sum,
// and the kernel below turns the logits into weights,
//     w[h][p] = sum over the step's tokens t of the request, p <= position(t), and over the query heads g of KV head h of
//               exp2(logit[t][g][p] - max[t][g]) / sum[t][g],
// and adds them to the accumulators:  acc = (p appended before this step ? decay * acc : 0) + w.
#include <algorithm>

#include "kv_eviction.h"
#include "split_kv_reduce_kernel.h"

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

constexpr uint32_t kFinishThreads = 512, kFinishWaves = kFinishThreads / 64;
constexpr uint32_t kNormEntries = 512;  // (token, head) normalisers held in LDS at a time
constexpr uint32_t kFewEntries = 8;    // up to this many (a decode step's heads) a thread holds the logits of all

// Maximum and reciprocal sum of one (token, head) over its partial states p0 .. p1, in every lane of the wave; +inf and 0
// where nothing contributes, so that the row's weights are zero.  The sum stays out of the exponent: half an ulp of its
// log2 would be an error of all the row's weights alike.
__device__ __forceinline__ float2 norm_of(const WeightsArgs& a, uint32_t p0, uint32_t p1, uint32_t head, uint32_t lane) {
    float m = -INFINITY, s = 0.0f;
    for (uint32_t p = p0 + lane; p < p1; p += 64) {
        const uint64_t r = (uint64_t)(a.row_index ? a.row_index[p] : p) * a.hq + head;
        const float pm = a.part_max[r], ps = a.part_sum[r], next = fmaxf(m, pm);
        if (pm > -INFINITY) s = s * exp2f(m - next) + ps * exp2f(pm - next);
        m = next;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float om = __shfl_xor(m, off, 64), os = __shfl_xor(s, off, 64), next = fmaxf(m, om);
        if (next > -INFINITY) s = s * exp2f(m - next) + os * exp2f(om - next);
        m = next;
    }
    return m > -INFINITY ? make_float2(m, 1.0f / s) : make_float2(INFINITY, 0.0f);
}

// The accumulators of one (kv_split row, KV head), by a workgroup.  The rows of a request's last token of the step tile
// all its positions, so those rows' workgroups own the accumulators they cover and the others have nothing to do: no two
// workgroups meet.  A thread takes four adjacent positions at a time: logits, accumulators and stores of 16 bytes a lane
// where a page holds a multiple of four tokens, and a whole row in one turn if it has up to 2048 keys.
// The chain of dependent reads is what bounds it (table row -> tokens -> partial states -> logits -> accumulators, each a
// round trip), so the first turn's logits and page IDs are asked for before the normalisers are.  With the combine beside
// it: 12.1 us for 25 MB at 32 requests of 1k-8k (the combine alone takes 6), 13.2 us for 49 MB (3.7 TB/s) at four of
// 131072; two to four workgroups a row repeat the chain and take longer (an earlier form: 22 us for 15).
__device__ __forceinline__ void accumulate_row(const WeightsArgs& a, uint32_t split, uint32_t kv_head, float2* norm) {
    const uint32_t num_tokens = active_count(a.replay_counts, kReplayTokens, a.num_active_tokens);
    const uint32_t num_splits = active_count(a.replay_counts, kReplaySplits, a.num_active_kv_splits);
    const uint32_t layer = active_layer(a.replay_counts, a.v.layer, a.v.num_layers);
    if (split >= num_splits) return;
    const uint32_t token = a.kv_splits[split * 3], begin = a.kv_splits[split * 3 + 1], row_end = a.kv_splits[split * 3 + 2];
    if (token >= num_tokens) return;
    // asked for together: whatever depends on the token alone
    const uint32_t before = token > 0 ? token - 1 : 0, after = min(token + 1, num_tokens - 1);
    const uint32_t slot = a.req_slots[token], slot_before = a.req_slots[before], slot_after = a.req_slots[after];
    const uint32_t own = a.flat_token_indices[token], p0 = a.cu_kv_splits[token], p1 = a.cu_kv_splits[token + 1];
    if (after != token && slot_after == slot) return;
    if (slot >= a.v.num_slots) {
        report_cache_range(a.status);
        return;
    }
    uint32_t first = token, held = own;
    if (before != token && slot_before == slot) {
        for (first = before; first > 0 && a.req_slots[first - 1] == slot;) --first;
        held = a.flat_token_indices[first];
    }
    const uint32_t end = min(row_end, a.max_context);
    if (threadIdx.x == 0 && row_end > end) report_cache_range(a.status);
    const uint32_t* row = table_row(a.v, slot, layer);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t entries = (token - first + 1) * a.group;
    const bool vector = a.v.log2_page < 32 && a.v.log2_page >= 2 && reinterpret_cast<uintptr_t>(a.page_weights) % 16 == 0;

    // the accumulators of positions p .. p + 3, from `sum`; `first_turn`: on top of what counts already
    auto whole = [&](uint32_t p) { return vector && p >= begin && p + 4 <= end; };
    auto slot_of = [&](uint32_t p, uint32_t page) {
        return reinterpret_cast<float4*>(a.page_weights + weight_index(a.v, page, kv_head, page_place(a.v, p)));
    };
    auto add = [&](uint32_t p, const float (&sum)[4], uint32_t page, float4 old, bool first_turn) {
        if (whole(p)) {
            if (page == kNoPage) {
                report_cache_range(a.status);
                return;
            }
            auto base = [&](float x, uint32_t at) { return !first_turn ? x : at < held ? a.decay * x : 0.0f; };
            *slot_of(p, page) = make_float4(base(old.x, p) + sum[0], base(old.y, p + 1) + sum[1],
                                            base(old.z, p + 2) + sum[2], base(old.w, p + 3) + sum[3]);
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (p + i < begin || p + i >= end) continue;
            const uint32_t id = page_of(a.v, row, p + i, a.v.num_weight_pages);
            if (id == kNoPage) {
                report_cache_range(a.status);
                continue;
            }
            float* acc = a.page_weights + weight_index(a.v, id, kv_head, page_place(a.v, p + i));
            *acc = (!first_turn ? *acc : p + i < held ? a.decay * *acc : 0.0f) + sum[i];
        }
    };
    const uint32_t start = (begin & ~3u) + threadIdx.x * 4;

    if (entries <= kFewEntries && token == first) {
        // one token: its position is the row's last at most, so every key of the row is visible
        const float* token_logits = a.logits + logit_index(a.logits_stride, a.group, (uint64_t)token * a.v.hkv + kv_head, 0, 0);
        float4 l[kFewEntries];
        uint32_t page = kNoPage;
        float4 old = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto fetch = [&](uint32_t p) {
#pragma unroll
            for (uint32_t e = 0; e < kFewEntries; ++e)
                if (e < entries) l[e] = *reinterpret_cast<const float4*>(token_logits + logit_index(0, a.group, 0, p, e));
            page = page_of(a.v, row, p, a.v.num_weight_pages);
            if (whole(p) && page != kNoPage) old = *slot_of(p, page);
        };
        if (start < end) fetch(start);
        if (wave < entries) {
            const float2 x = norm_of(a, p0, p1, kv_head * a.group + wave, lane);
            if (lane == 0) norm[wave] = x;
        }
        __syncthreads();
        for (uint32_t p = start; p < end; p += kFinishThreads * 4) {
            if (p != start) fetch(p);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t e = 0; e < kFewEntries; ++e) {
                if (e >= entries) continue;
                const float x[4] = {l[e].x, l[e].y, l[e].z, l[e].w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sum[i] += p + i <= own ? __builtin_amdgcn_exp2f(x[i] - norm[e].x) * norm[e].y : 0.0f;
            }
            add(p, sum, page, old, true);
        }
        return;
    }
    for (uint32_t base = 0; base < entries; base += kNormEntries) {
        const uint32_t count = min(kNormEntries, entries - base);
        if (base > 0) __syncthreads();
        for (uint32_t e = wave; e < count; e += kFinishWaves) {
            const uint32_t t = first + (base + e) / a.group;
            const float2 x = norm_of(a, a.cu_kv_splits[t], a.cu_kv_splits[t + 1], kv_head * a.group + (base + e) % a.group, lane);
            if (lane == 0) norm[e] = x;
        }
        __syncthreads();
        for (uint32_t p = start; p < end; p += kFinishThreads * 4) {
            const uint32_t page = page_of(a.v, row, p, a.v.num_weight_pages);
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            uint32_t t = base / a.group, g = base % a.group;
            for (uint32_t e = 0; e < count; ++e) {
                const uint32_t last = a.flat_token_indices[first + t];
                const float4 l = *reinterpret_cast<const float4*>(
                    a.logits + logit_index(a.logits_stride, a.group, (uint64_t)(first + t) * a.v.hkv + kv_head, p, g));
                const float x[4] = {l.x, l.y, l.z, l.w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sum[i] += p + i <= last ? __builtin_amdgcn_exp2f(x[i] - norm[e].x) * norm[e].y : 0.0f;
                if (++g == a.group) {
                    g = 0;
                    ++t;
                }
            }
            const float4 old = whole(p) && page != kNoPage ? *slot_of(p, page) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            add(p, sum, page, old, base == 0);
        }
    }
}

// The combine and the accumulators in one launch: the first workgroups take a (kv_split row, KV head) each, the others
// the output rows, a wave each or (kWide) a workgroup each, as the combine's own launch does.
template <typename Tag, int D>
__global__ __launch_bounds__(kFinishThreads) void finish_kernel(WeightsArgs w, ReduceArgs r, uint32_t weight_groups,
                                                                uint32_t wide) {
    __shared__ union {
        float2 norm[kNormEntries];
        WideReduceLds<D> wide;
    } lds;
    static_assert(kWideWaves == kFinishWaves, "a wide row takes the whole workgroup");
    if (blockIdx.x < weight_groups) {
        accumulate_row(w, blockIdx.x / w.v.hkv, blockIdx.x % w.v.hkv, lds.norm);
        return;
    }
    resolve_active(r);
    const uint64_t group = blockIdx.x - weight_groups;
    if (wide) {
        if (r.row_index != nullptr) reduce_row_wide<Tag, D, true>(r, group, lds.wide);
        else reduce_row_wide<Tag, D, false>(r, group, lds.wide);
        return;
    }
    const uint64_t row_out = group * kFinishWaves + (threadIdx.x >> 6);
    if (row_out >= (uint64_t)r.num_active_tokens * r.hq) return;
    if (r.row_index != nullptr) reduce_row<Tag, D, true>(r, row_out);
    else reduce_row<Tag, D, false>(r, row_out);
}

// The accumulators alone, next to the shape-generic combine.
__global__ __launch_bounds__(kFinishThreads) void accumulate_kernel(WeightsArgs w) {
    __shared__ float2 norm[kNormEntries];
    accumulate_row(w, blockIdx.x / w.v.hkv, blockIdx.x % w.v.hkv, norm);
}

static uint64_t logits_stride(uint32_t max_context_tokens) { return ((uint64_t)max_context_tokens + 63) / 64 * 64; }

int check_kv_weights(const psi_hip_gqa_config* cfg, const psi_hip_page_table_layout* layout, const uint32_t* page_ids,
                     uint32_t gqa_layer_index, uint64_t kv_pages_bytes, const psi_hip_kv_weights* weights,
                     uint32_t num_total_tokens, CacheView* view) {
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(weights->page_weights && weights->logits, "weight accumulation buffers must not be null");
    PSI_REQUIRE(weights->decay >= 0.0f && weights->decay <= 1.0f, "the decay must lie in [0, 1]");
    PSI_REQUIRE(num_total_tokens > 0 && weights->max_context_tokens > 0, "logits need tokens and a context");
    PSI_REQUIRE(reinterpret_cast<uintptr_t>(weights->logits) % 16 == 0, "the logits must be 16-byte aligned");
    uint64_t needed = 0;
    rc = psi_hip_split_kv_single_q_logits_bytes(cfg, num_total_tokens, weights->max_context_tokens, &needed);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(weights->logits_bytes >= needed, "logits buffer too small: %llu < %llu",
                (unsigned long long)weights->logits_bytes, (unsigned long long)needed);
    return make_cache_view(g, layout, page_ids, gqa_layer_index, kv_pages_bytes, weights->page_weights_bytes, view);
}

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
    PSI_REQUIRE(flat_token_indices && cu_kv_splits && output, "weight accumulation buffers must not be null");
    WeightsArgs a;
    ReduceArgs r;
    rc = check_kv_weights(cfg, layout, page_ids, gqa_layer_index, kv_pages_bytes, weights, num_total_tokens, &a.v);
    if (rc != PSI_HIP_OK) return rc;
    rc = single_q_reduce_args(ctx, cfg, scratch, scratch_bytes, cu_kv_splits, output, num_total_tokens,
                              num_total_kv_splits, num_active_tokens, partial_row_index, gate, &g, &r);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE((uint64_t)num_total_kv_splits * g.hkv <= 0x7fffffffull, "too many KV splits");
    a.v.num_weight_pages = std::min(a.v.num_weight_pages, a.v.num_pages);  // no page beyond the arena either

    DeviceGuard guard(ctx->device);
    float* logits = static_cast<float*>(weights->logits);
    const uint64_t stride = logits_stride(weights->max_context_tokens);
    rc = single_q_map_impl(ctx, cfg, layout, q, kv_pages, kv_pages_bytes, req_slots, page_ids, kv_splits, worker_cu,
                           num_workers, scratch, scratch_bytes, gqa_layer_index, num_total_tokens, num_total_kv_splits,
                           num_active_tokens, num_active_kv_splits, flat_k, flat_v, flat_token_indices, logits, stride);
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
    const uint64_t weight_groups = (uint64_t)num_active_kv_splits * g.hkv;
    const bool wide = reduce_is_wide(r);
    const uint64_t rows = (uint64_t)num_active_tokens * g.hq, row_groups = wide ? rows : (rows + kFinishWaves - 1) / kFinishWaves;
    if (ctx->force_generic || (g.d != 128 && g.d != 256) || weight_groups + row_groups > 0x7fffffffull) {
        rc = launch_single_q_reduce(ctx, g, r);
        if (rc != PSI_HIP_OK) return rc;
        LaunchScope scope(ctx, "kv_weights");
        hipLaunchKernelGGL(accumulate_kernel, dim3((uint32_t)weight_groups), dim3(kFinishThreads), 0, ctx->stream, a);
        PSI_HIP_CHECK(hipGetLastError());
        return PSI_HIP_OK;
    }
    LaunchScope scope(ctx, "kv_weights");
    const dim3 grid((uint32_t)(weight_groups + row_groups)), threads(kFinishThreads);
#define PSI_FINISH(TAG)                                                                                                \
    do {                                                                                                               \
        if (g.d == 256)                                                                                                \
            hipLaunchKernelGGL((finish_kernel<TAG, 256>), grid, threads, 0, ctx->stream, a, r, (uint32_t)weight_groups, \
                               wide ? 1u : 0u);                                                                        \
        else                                                                                                           \
            hipLaunchKernelGGL((finish_kernel<TAG, 128>), grid, threads, 0, ctx->stream, a, r, (uint32_t)weight_groups, \
                               wide ? 1u : 0u);                                                                        \
    } while (0)
    if (r.out_dtype == PSI_HIP_F32) PSI_FINISH(F32Tag);
    else if (r.out_dtype == PSI_HIP_BF16) PSI_FINISH(BF16Tag);
    else PSI_FINISH(F16Tag);
#undef PSI_FINISH
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
