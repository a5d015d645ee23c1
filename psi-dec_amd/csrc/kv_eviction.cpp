// Host side of the operators that bound a paged cache: views, plans and their checks.
#include "kv_eviction.h"

#include <algorithm>
#include <vector>

namespace psi {

DeviceGuard::DeviceGuard(int device) {
    int current = -1;
    if (hipGetDevice(&current) == hipSuccess && current != device && hipSetDevice(device) == hipSuccess) previous_ = current;
}
DeviceGuard::~DeviceGuard() {
    if (previous_ >= 0) (void)hipSetDevice(previous_);
}

int make_cache_view(const Geometry& g, const psi_hip_page_table_layout* layout, const uint32_t* page_ids,
                    uint32_t gqa_layer_index, uint64_t kv_pages_bytes, uint64_t page_weights_bytes, CacheView* view) {
    int rc = check_layout(layout);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(page_ids != nullptr, "the page table must not be null");
    PSI_REQUIRE(gqa_layer_index < layout->num_gqa_layers, "GQA page-table index exceeds layer count");
    const uint64_t entries = (uint64_t)layout->num_blocks * layout->num_page_ids_per_block;
    PSI_REQUIRE(entries * g.tokens_per_page <= INT32_MAX, "a request's token positions must stay below 2^31");
    const uint64_t page_bytes = g.page_elems * g.elem;
    PSI_REQUIRE(kv_pages_bytes == 0 || kv_pages_bytes >= page_bytes, "GQA page arena is smaller than one page");
    const uint64_t weight_pages = page_weights_bytes / (4ull * g.hkv * g.tokens_per_page);
    PSI_REQUIRE(weight_pages > 0, "the weight accumulators are smaller than one page's");
    view->page_ids = page_ids;
    view->page_elems = g.page_elems;
    view->num_slots = layout->num_req_slots;
    view->num_layers = layout->num_gqa_layers;
    view->layer = gqa_layer_index;
    view->entries = (uint32_t)entries;
    view->positions = (uint32_t)(entries * g.tokens_per_page);
    view->hkv = g.hkv;
    view->d = g.d;
    view->tokens_per_page = g.tokens_per_page;
    const bool power = (g.tokens_per_page & (g.tokens_per_page - 1)) == 0;
    view->log2_page = power ? 31u - __builtin_clz(g.tokens_per_page) : 32u;
    view->num_pages = (uint32_t)std::min<uint64_t>(kv_pages_bytes ? kv_pages_bytes / page_bytes : kNoPage, kNoPage);
    view->num_weight_pages = (uint32_t)std::min<uint64_t>(weight_pages, kNoPage);
    return PSI_HIP_OK;
}

int check_no_replay_counts(const psi_hip_ctx* ctx) {
    if (ctx->replay_counts != nullptr)
        return fail(PSI_HIP_ERR_UNSUPPORTED,
                    "this entry point takes its counts by value: unbind the device-side counts "
                    "(psi_hip_ctx_bind_replay_counts with null)");
    return PSI_HIP_OK;
}

// Requests of one call: slots inside the table and each named once (two would write the same pages), tokens inside it.
static int check_slots(const Geometry& g, const psi_hip_page_table_layout* layout, const uint32_t* req_slots,
                       uint32_t num_reqs, uint64_t* out_capacity) {
    int rc = check_layout(layout);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(req_slots != nullptr && num_reqs > 0, "cache eviction needs requests");
    const uint64_t entries = (uint64_t)layout->num_blocks * layout->num_page_ids_per_block;
    PSI_REQUIRE(entries * g.tokens_per_page <= INT32_MAX, "a request's token positions must stay below 2^31");
    *out_capacity = entries * g.tokens_per_page;
    for (uint32_t r = 0; r < num_reqs; ++r)
        PSI_REQUIRE(req_slots[r] < layout->num_req_slots,
                    "GQA request page table req_slot out of range: req_slot=%u num_req_slots=%u", req_slots[r],
                    layout->num_req_slots);
    try {
        std::vector<uint32_t> sorted(req_slots, req_slots + num_reqs);
        std::sort(sorted.begin(), sorted.end());
        for (uint32_t r = 1; r < num_reqs; ++r)
            PSI_REQUIRE(sorted[r] != sorted[r - 1], "req_slot %u is named twice in one call", sorted[r]);
    } catch (const std::bad_alloc&) {
        return fail(PSI_HIP_ERR_RESOURCE_EXHAUSTED, "no host memory for the request check");
    }
    return PSI_HIP_OK;
}

}  // namespace psi

using namespace psi;

extern "C" int psi_hip_kv_page_weights_bytes(const psi_hip_gqa_config* cfg, uint64_t num_pages, uint64_t* out_bytes) {
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(out_bytes != nullptr, "out pointer must not be null");
    PSI_REQUIRE(num_pages > 0 && num_pages <= UINT32_MAX, "the number of pages must be positive and fit u32");
    *out_bytes = num_pages * g.hkv * g.tokens_per_page * 4;
    return PSI_HIP_OK;
}

// Workgroups that a plan aims at, over all windows and KV heads: one per compute unit, as a workgroup fills it (two
// rounds of them take a fifth longer with 8 prompts of 1k-8k and with one of 65536).
constexpr uint32_t kObserveWorkgroups = 256;
constexpr uint32_t kObserveRowTokens = 64;  // rows are cut at multiples of this (256: 18 us for 13 with one prompt of 777)

extern "C" int psi_hip_kv_observe_plan(const psi_hip_gqa_config* cfg, const psi_hip_page_table_layout* layout,
                                       const uint32_t* req_slots, const uint32_t* token_indices,
                                       const uint32_t* cu_tokens, const uint32_t* num_held, uint32_t num_reqs,
                                       uint32_t* windows, uint32_t* rows, uint32_t rows_capacity,
                                       uint32_t* out_num_rows, uint32_t* out_max_window, uint64_t* out_scratch_bytes) {
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    uint64_t capacity = 0;
    rc = check_slots(g, layout, req_slots, num_reqs, &capacity);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(token_indices && cu_tokens && out_num_rows && out_max_window && out_scratch_bytes,
                "observation plan: arrays and out pointers must not be null");
    PSI_REQUIRE((windows == nullptr) == (rows == nullptr), "observation plan: windows and rows are written together");
    PSI_REQUIRE(cu_tokens[0] == 0, "cu_tokens must start at zero");
    uint64_t total = 0;
    uint32_t max_window = 0;
    for (uint32_t r = 0; r < num_reqs; ++r) {
        PSI_REQUIRE(cu_tokens[r] < cu_tokens[r + 1], "observation plan: every request needs a query token");
        const uint32_t window = cu_tokens[r + 1] - cu_tokens[r];
        const uint64_t context = (uint64_t)token_indices[r] + window;
        PSI_REQUIRE(context <= capacity, "request %u: %llu tokens exceed the page table's %llu", r,
                    (unsigned long long)context, (unsigned long long)capacity);
        total += context;
        max_window = std::max(max_window, window);
    }
    // the shortest rows of which no more than that many workgroups come, or one row to a window
    const uint64_t aim = std::max<uint64_t>(std::max<uint64_t>(1, kObserveWorkgroups / g.hkv), num_reqs);
    uint64_t part = ((total + aim - 1) / aim + kObserveRowTokens - 1) / kObserveRowTokens * kObserveRowTokens;
    auto rows_at = [&](uint64_t tokens) {
        uint64_t rows = 0;
        for (uint32_t r = 0; r < num_reqs; ++r)
            rows += ((uint64_t)token_indices[r] + (cu_tokens[r + 1] - cu_tokens[r]) + tokens - 1) / tokens;
        return rows;
    };
    while (rows_at(part) > aim) part += std::max<uint64_t>(kObserveRowTokens, part / 16 / kObserveRowTokens * kObserveRowTokens);
    uint64_t n = 0;
    for (uint32_t r = 0; r < num_reqs; ++r) {
        const uint64_t context = (uint64_t)token_indices[r] + (cu_tokens[r + 1] - cu_tokens[r]);
        const uint64_t cuts = (context + part - 1) / part;
        if (windows != nullptr) {
            PSI_REQUIRE(n + cuts <= rows_capacity, "observation plan: %u rows are not enough", rows_capacity);
            uint32_t* w = windows + (uint64_t)r * kWindowWords;
            w[0] = req_slots[r];
            w[1] = cu_tokens[r];
            w[2] = cu_tokens[r + 1] - cu_tokens[r];
            w[3] = token_indices[r];
            w[4] = num_held != nullptr ? num_held[r] : token_indices[r];
            w[5] = (uint32_t)n;
            w[6] = (uint32_t)(n + cuts);
            w[7] = 0;
            for (uint64_t c = 0; c < cuts; ++c) {
                rows[(n + c) * 3] = r;
                rows[(n + c) * 3 + 1] = (uint32_t)(c * part);
                rows[(n + c) * 3 + 2] = (uint32_t)std::min(context, (c + 1) * part);
            }
        }
        n += cuts;
    }
    PSI_REQUIRE(n <= UINT32_MAX, "observation plan: too many rows");
    *out_num_rows = (uint32_t)n;
    *out_max_window = max_window;
    *out_scratch_bytes = (n * max_window + cu_tokens[num_reqs]) * g.hq * 8;
    return PSI_HIP_OK;
}

extern "C" int psi_hip_kv_evict_plan(const psi_hip_gqa_config* cfg, const psi_hip_page_table_layout* layout,
                                     const uint32_t* req_slots, const uint32_t* num_cached, uint32_t num_reqs,
                                     uint32_t* requests, uint32_t* out_max_cached) {
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    uint64_t capacity = 0;
    rc = check_slots(g, layout, req_slots, num_reqs, &capacity);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(num_cached && requests && out_max_cached, "eviction plan: arrays and out pointers must not be null");
    uint32_t most = 0;
    for (uint32_t r = 0; r < num_reqs; ++r) {
        PSI_REQUIRE(num_cached[r] <= capacity, "request %u: %u tokens exceed the page table's %llu", r, num_cached[r],
                    (unsigned long long)capacity);
        most = std::max(most, num_cached[r]);
    }
    for (uint32_t r = 0; r < num_reqs; ++r) {
        requests[r * kRequestWords] = req_slots[r];
        requests[r * kRequestWords + 1] = num_cached[r];
    }
    *out_max_cached = most;
    return PSI_HIP_OK;
}
