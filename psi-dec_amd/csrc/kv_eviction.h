// What the operators that bound a paged cache share (kv_weights.hip, kv_observe.hip, kv_select.hip, kv_compact.hip):
// the view of one layer's cache and of the accumulators beside it.
//
// Accumulators are f32 [page][KV head][token in page], found through the same page IDs as K and V, so that a page's
// accumulators go where the page goes and no array is cut for the longest request.
#pragma once
#include "common.h"
#include "device_types.h"

namespace psi {

struct CacheView {
    const uint32_t* page_ids;
    uint64_t page_elems;
    uint32_t num_slots, num_layers, layer, entries;  // entries: page IDs of one (slot, layer)
    uint32_t positions;                              // tokens that those pages hold
    uint32_t hkv, d, tokens_per_page, log2_page;  // log2_page: 32 when tokens_per_page is no power of two
    uint32_t num_pages, num_weight_pages;         // of the arena and of the accumulators; page IDs beyond are left out
};

constexpr uint32_t kNoPage = 0xffffffffu;
constexpr uint32_t kStatusCacheRange = 2;  // status word: bit 2 of the PSI_HIP_DEVICE_ERR_* mask

__device__ __forceinline__ uint32_t page_index(const CacheView& v, uint32_t position) {
    return v.log2_page < 32 ? position >> v.log2_page : position / v.tokens_per_page;
}
__device__ __forceinline__ uint32_t page_place(const CacheView& v, uint32_t position) {
    return v.log2_page < 32 ? position & (v.tokens_per_page - 1) : position % v.tokens_per_page;
}
// First page-table entry of (slot, layer): block and ID index of a position are the two digits of its page number, so
// the entry of a position is this plus page_index().
__device__ __forceinline__ const uint32_t* table_row(const CacheView& v, uint32_t req_slot, uint32_t layer) {
    return v.page_ids + ((uint64_t)req_slot * v.num_layers + layer) * v.entries;
}
__device__ __forceinline__ uint32_t page_of(const CacheView& v, const uint32_t* row, uint32_t position, uint32_t limit) {
    const uint32_t entry = page_index(v, position);
    if (entry >= v.entries) return kNoPage;
    const uint32_t id = row[entry];
    return id < limit ? id : kNoPage;
}
__device__ __forceinline__ uint64_t weight_index(const CacheView& v, uint32_t page_id, uint32_t kv_head, uint32_t place) {
    return ((uint64_t)page_id * v.hkv + kv_head) * v.tokens_per_page + place;
}
__device__ __forceinline__ uint64_t line_index(const CacheView& v, uint32_t page_id, uint32_t kind, uint32_t kv_head,
                                               uint32_t place) {
    return page_id * v.page_elems + (((uint64_t)kind * v.hkv + kv_head) * v.tokens_per_page + place) * v.d;
}

// The GPU's side of PSI_HIP_DEVICE_ERR_CACHE_RANGE: a word of pinned host memory, written with a plain store.
__device__ __forceinline__ void report_cache_range(uint32_t* status) { status[kStatusCacheRange] = 1; }

// One request of a selection or compaction, as psi_hip_kv_evict_plan writes it.
constexpr uint32_t kRequestWords = 2;  // {req_slot, cached tokens}
// One window of an observation, as psi_hip_kv_observe_plan writes it: {req_slot, first query row, query rows, position
// of the first, positions whose accumulators count already, first and last + 1 of its rows, 0}.
constexpr uint32_t kWindowWords = 8;

// Fills the view; refuses accumulators that hold no page.  kv_pages_bytes 0: the arena's end is not checked.
int make_cache_view(const Geometry& g, const psi_hip_page_table_layout* layout, const uint32_t* page_ids,
                    uint32_t gqa_layer_index, uint64_t kv_pages_bytes, uint64_t page_weights_bytes, CacheView* view);
// Refuses a context with device-side counts bound: these entry points take theirs by value.
int check_no_replay_counts(const psi_hip_ctx* ctx);
// What a step that accumulates asks of its weights (kv_weights.hip), so that a layer can ask it before its first launch.
int check_kv_weights(const psi_hip_gqa_config* cfg, const psi_hip_page_table_layout* layout, const uint32_t* page_ids,
                     uint32_t gqa_layer_index, uint64_t kv_pages_bytes, const psi_hip_kv_weights* weights,
                     uint32_t num_total_tokens, CacheView* view);

// Launches go to the context's GPU whatever the calling thread's current device is.
class DeviceGuard {
  public:
    explicit DeviceGuard(int device);
    ~DeviceGuard();

  private:
    int previous_ = -1;
};

}  // namespace psi
