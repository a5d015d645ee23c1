// Which cached tokens a (request, KV head) keeps: the first num_first, the last num_recent, and of the others those with
// the largest accumulated weight until `budget` are chosen; equal weights go to the lower position.  The chosen
// positions come out in ascending order.  A NaN weight counts as -inf, -0 as 0.
//
// The budget-th largest weight is found by radix selection on order-preserving integer keys (eight bits a pass, the
// histogram in LDS), the positions by ballots and prefix counts: no sort, and the same answer on every run.
#include "kv_eviction.h"

namespace psi {

struct SelectArgs {
    CacheView v;
    const float* page_weights;
    const uint32_t* requests;
    uint32_t* kept;
    uint32_t* status;
    uint32_t max_cached, budget, num_first, num_recent;
};

// Larger weight, larger key.
__device__ __forceinline__ uint32_t weight_key(float w) {
    uint32_t u = __float_as_uint(w);
    if ((u & 0x7fffffffu) > 0x7f800000u) u = 0xff800000u;  // NaN -> -inf
    if (u == 0x80000000u) u = 0;                           // -0 -> 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kKeepKey = 0xffffffffu;  // above every weight's key: tokens that are kept whatever their weight

constexpr uint32_t kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

// One workgroup per (request, KV head).
__global__ __launch_bounds__(kSelectThreads) void select_kept_kernel(SelectArgs a) {
    const uint32_t req = blockIdx.x / a.v.hkv, kv_head = blockIdx.x % a.v.hkv;
    const uint32_t slot = a.requests[req * kRequestWords], n = min(min(a.requests[req * kRequestWords + 1], a.max_cached), a.v.positions);
    uint32_t* kept = a.kept + (uint64_t)blockIdx.x * a.budget;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (uint32_t i = min(n, a.budget) + tid; i < a.budget; i += kSelectThreads) kept[i] = PSI_HIP_SENTINEL;
    if (slot >= a.v.num_slots) {
        for (uint32_t i = tid; i < min(n, a.budget); i += kSelectThreads) kept[i] = PSI_HIP_SENTINEL;
        report_cache_range(a.status);
        return;
    }
    if (n <= a.budget) {
        for (uint32_t i = tid; i < n; i += kSelectThreads) kept[i] = i;
        return;
    }
    const uint32_t* row = table_row(a.v, slot, a.v.layer);
    const uint32_t recent_from = n - min(a.num_recent, n);
    auto key_of = [&](uint32_t p) -> uint32_t {
        if (p < a.num_first || p >= recent_from) return kKeepKey;
        const uint32_t page = page_of(a.v, row, p, a.v.num_weight_pages);
        if (page == kNoPage) {
            report_cache_range(a.status);
            return weight_key(-INFINITY);
        }
        return weight_key(a.page_weights[weight_index(a.v, page, kv_head, page_place(a.v, p))]);
    };

    __shared__ uint32_t hist[256];
    __shared__ uint32_t above[256];
    __shared__ uint32_t chosen[2];
    __shared__ uint32_t wave_gt[kSelectWaves], wave_eq[kSelectWaves];
    uint32_t prefix = 0, remaining = a.budget;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (uint32_t p = tid; p < n; p += kSelectThreads) {
            const uint32_t key = key_of(p);
            if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid < 256) above[tid] = hist[tid];
        __syncthreads();
        // above[b] = keys in bins b and higher
        for (uint32_t step = 1; step < 256; step <<= 1) {
            uint32_t add = 0;
            if (tid < 256 && tid + step < 256) add = above[tid + step];
            __syncthreads();
            if (tid < 256) above[tid] += add;
            __syncthreads();
        }
        if (tid < 256) {
            const uint32_t higher = tid < 255 ? above[tid + 1] : 0;
            if (above[tid] >= remaining && higher < remaining) {
                chosen[0] = tid;
                chosen[1] = remaining - higher;
            }
        }
        __syncthreads();
        prefix = prefix << 8 | chosen[0];
        remaining = chosen[1];
        __syncthreads();
    }
    // `remaining` of the keys equal to the threshold belong to the kept ones: those at the lowest positions
    const uint32_t threshold = prefix;
    const uint32_t share = (n + kSelectThreads - 1) / kSelectThreads * 64;
    const uint32_t begin = min(wave * share, n), end = min(begin + share, n);
    uint32_t gt = 0, eq = 0;
    for (uint32_t base = begin; base < end; base += 64) {
        const uint32_t p = base + lane;
        const uint32_t key = p < end ? key_of(p) : 0;
        gt += __popcll(__ballot(p < end && key > threshold));
        eq += __popcll(__ballot(p < end && key == threshold));
    }
    if (lane == 0) {
        wave_gt[wave] = gt;
        wave_eq[wave] = eq;
    }
    __syncthreads();
    uint32_t gt_before = 0, eq_before = 0;
    for (uint32_t w = 0; w < wave; ++w) {
        gt_before += wave_gt[w];
        eq_before += wave_eq[w];
    }
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
    for (uint32_t base = begin; base < end; base += 64) {
        const uint32_t p = base + lane;
        const uint32_t key = p < end ? key_of(p) : 0;
        const uint64_t gt_mask = __ballot(p < end && key > threshold), eq_mask = __ballot(p < end && key == threshold);
        const uint32_t eq_rank = eq_before + __popcll(eq_mask & lower);
        const uint32_t at = gt_before + __popcll(gt_mask & lower) + min(eq_rank, remaining);
        if (p < end && (key > threshold || (key == threshold && eq_rank < remaining)) && at < a.budget) kept[at] = p;
        gt_before += __popcll(gt_mask);
        eq_before += __popcll(eq_mask);
    }
}

}  // namespace psi

using namespace psi;

extern "C" int psi_hip_kv_select_kept(psi_hip_ctx* ctx, const psi_hip_gqa_config* cfg,
                                      const psi_hip_page_table_layout* layout, const float* page_weights,
                                      uint64_t page_weights_bytes, const uint32_t* page_ids, const uint32_t* requests,
                                      uint32_t num_reqs, uint32_t max_cached_tokens, uint32_t budget, uint32_t num_first,
                                      uint32_t num_recent, uint32_t* kept, uint32_t gqa_layer_index) {
    PSI_REQUIRE(ctx != nullptr, "ctx must not be null");
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    rc = check_no_replay_counts(ctx);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(page_weights && requests && kept, "selection buffers must not be null");
    PSI_REQUIRE(num_reqs > 0, "a selection needs requests");
    PSI_REQUIRE(budget > 0, "the budget must be positive");
    PSI_REQUIRE((uint64_t)num_first + num_recent <= budget, "the tokens that are always kept exceed the budget: %u + %u > %u",
                num_first, num_recent, budget);
    SelectArgs a;
    rc = make_cache_view(g, layout, page_ids, gqa_layer_index, 0, page_weights_bytes, &a.v);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE((uint64_t)num_reqs * g.hkv <= 0x7fffffffull, "too many requests in one selection");
    a.page_weights = page_weights;
    a.requests = requests;
    a.kept = kept;
    a.status = ctx->status_device;
    a.max_cached = max_cached_tokens;
    a.budget = budget;
    a.num_first = num_first;
    a.num_recent = num_recent;
    DeviceGuard guard(ctx->device);
    LaunchScope scope(ctx, "kv_select");
    hipLaunchKernelGGL(select_kept_kernel, dim3(num_reqs * g.hkv), dim3(kSelectThreads), 0, ctx->stream, a);
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
