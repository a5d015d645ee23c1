// Moves the kept tokens of every (request, KV head) to the front of the request's pages, in order and in place: entry i
// gets the K and V line and the accumulator of position kept[i].
//
// kept ascends, so kept[i] >= i: a line moves towards the front only.  The lines are taken in runs of ascending i; a run
// is read whole before any of it is written.  What run j writes lies below the run's end, and every entry beyond that
// end reads a position at or beyond it, so later runs still find their lines.  Runs of one line slice must follow one
// another, but slices of a line (a few 16-byte chunks of K or of V) and heads are independent: a workgroup owns one.
#include "kv_eviction.h"

namespace psi {

struct CompactArgs {
    CacheView v;
    void* pages;
    float* page_weights;  // null: no accumulators beside this cache
    const uint32_t* requests;
    const uint32_t* kept;
    uint32_t* status;
    uint32_t max_cached, budget;
    uint32_t line_units, slice_units, num_slices;  // units of a line, of a slice; slices of a line
};

constexpr uint32_t kCompactThreads = 1024;
constexpr int kCompactUnroll = 4;

// One workgroup per (request, KV head, slice of K | slice of V | accumulators); slice_units divides kCompactThreads.
template <typename Unit>
__global__ __launch_bounds__(kCompactThreads) void compact_kernel(CompactArgs a) {
    const uint32_t parts = 2 * a.num_slices + (a.page_weights != nullptr ? 1u : 0u);
    const uint32_t part = blockIdx.x % parts, kv_head = blockIdx.x / parts % a.v.hkv, req = blockIdx.x / parts / a.v.hkv;
    const uint32_t slot = a.requests[req * kRequestWords], n = min(min(a.requests[req * kRequestWords + 1], a.max_cached), a.v.positions);
    if (n <= a.budget) return;  // everything is kept where it is
    if (slot >= a.v.num_slots) {
        report_cache_range(a.status);
        return;
    }
    const uint32_t* kept = a.kept + ((uint64_t)req * a.v.hkv + kv_head) * a.budget;
    const uint32_t* row = table_row(a.v, slot, a.v.layer);
    const bool is_weights = part == 2 * a.num_slices;
    const uint32_t kind = part / a.num_slices, unit0 = part % a.num_slices * a.slice_units;
    const uint32_t width = is_weights ? 1 : a.slice_units, per_round = kCompactThreads / width;
    const uint32_t my_line = threadIdx.x / width, my_unit = unit0 + threadIdx.x % width;
    const bool in_line = is_weights || my_unit < a.line_units;
    const uint32_t limit = is_weights ? a.v.num_weight_pages : a.v.num_pages;
    Unit* lines = static_cast<Unit*>(a.pages);
    auto unit_index = [&](uint32_t page, uint32_t place) -> uint64_t {
        const uint64_t line = ((uint64_t)page * 2 + kind) * a.v.hkv * a.v.tokens_per_page +
                              (uint64_t)kv_head * a.v.tokens_per_page + place;
        return line * a.line_units + my_unit;
    };
    for (uint32_t base = 0; base < a.budget; base += per_round * kCompactUnroll) {
        Unit held[kCompactUnroll] = {};
        float weight[kCompactUnroll] = {};
        uint32_t to_page[kCompactUnroll];
        uint32_t i[kCompactUnroll];
#pragma unroll
        for (int u = 0; u < kCompactUnroll; ++u) {
            i[u] = base + u * per_round + my_line;
            to_page[u] = kNoPage;
            if (!in_line || i[u] >= a.budget) continue;
            const uint32_t src = kept[i[u]];
            if (src == i[u]) continue;
            if (src < i[u] || src >= n) {  // no ascending choice among the cached tokens: nothing is moved for it
                report_cache_range(a.status);
                continue;
            }
            const uint32_t from_page = page_of(a.v, row, src, limit);
            to_page[u] = page_of(a.v, row, i[u], limit);
            if (from_page == kNoPage || to_page[u] == kNoPage) {
                report_cache_range(a.status);
                to_page[u] = kNoPage;
                continue;
            }
            if (is_weights) weight[u] = a.page_weights[weight_index(a.v, from_page, kv_head, page_place(a.v, src))];
            else held[u] = lines[unit_index(from_page, page_place(a.v, src))];
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the run has been read ...
        __syncthreads();                                  // ... by every wave before any of it is written
#pragma unroll
        for (int u = 0; u < kCompactUnroll; ++u) {
            if (to_page[u] == kNoPage) continue;
            if (is_weights) a.page_weights[weight_index(a.v, to_page[u], kv_head, page_place(a.v, i[u]))] = weight[u];
            else lines[unit_index(to_page[u], page_place(a.v, i[u]))] = held[u];
        }
    }
}

}  // namespace psi

using namespace psi;

extern "C" int psi_hip_kv_compact(psi_hip_ctx* ctx, const psi_hip_gqa_config* cfg,
                                  const psi_hip_page_table_layout* layout, void* kv_pages, uint64_t kv_pages_bytes,
                                  float* page_weights, uint64_t page_weights_bytes, const uint32_t* page_ids,
                                  const uint32_t* requests, uint32_t num_reqs, uint32_t max_cached_tokens,
                                  uint32_t budget, const uint32_t* kept, uint32_t gqa_layer_index) {
    PSI_REQUIRE(ctx != nullptr, "ctx must not be null");
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    rc = check_no_replay_counts(ctx);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(kv_pages && requests && kept, "compaction buffers must not be null");
    PSI_REQUIRE(num_reqs > 0, "a compaction needs requests");
    PSI_REQUIRE(budget > 0, "the budget must be positive");
    PSI_REQUIRE((page_weights == nullptr) == (page_weights_bytes == 0), "accumulators need their size and vice versa");
    CompactArgs a;
    // without accumulators their bound does not matter
    rc = make_cache_view(g, layout, page_ids, gqa_layer_index, kv_pages_bytes,
                         page_weights != nullptr ? page_weights_bytes : ~0ull, &a.v);
    if (rc != PSI_HIP_OK) return rc;
    a.pages = kv_pages;
    a.page_weights = page_weights;
    a.requests = requests;
    a.kept = kept;
    a.status = ctx->status_device;
    a.max_cached = max_cached_tokens;
    a.budget = budget;
    const uint32_t line_bytes = g.d * g.elem;
    const uint32_t unit = (line_bytes | (uint32_t)(reinterpret_cast<uintptr_t>(kv_pages) & 15)) % 16 == 0 ? 16 : g.elem;
    a.line_units = line_bytes / unit;
    // 128 bytes of a line to a workgroup
    const uint32_t most = 128 / unit;
    a.slice_units = 1;
    while (a.slice_units < most && a.slice_units < a.line_units) a.slice_units *= 2;
    a.num_slices = (a.line_units + a.slice_units - 1) / a.slice_units;
    const uint64_t grid = (uint64_t)num_reqs * g.hkv * (2 * a.num_slices + (page_weights != nullptr ? 1 : 0));
    PSI_REQUIRE(grid <= 0x7fffffffull, "too many requests in one compaction");
    DeviceGuard guard(ctx->device);
    LaunchScope scope(ctx, "kv_compact");
    const dim3 blocks((uint32_t)grid), threads(kCompactThreads);
    if (unit == 16) hipLaunchKernelGGL(compact_kernel<uint4>, blocks, threads, 0, ctx->stream, a);
    else if (unit == 4) hipLaunchKernelGGL(compact_kernel<uint32_t>, blocks, threads, 0, ctx->stream, a);
    else hipLaunchKernelGGL(compact_kernel<uint16_t>, blocks, threads, 0, ctx->stream, a);
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
