// Moves the kept tokens of every (request, KV head) to the front of the request's pages, in order and in place: entry i
// gets the K and V line and the accumulator of position kept[i].
//
// kept ascends, so kept[i] >= i: a line moves towards the front only.  The lines are taken in runs of ascending i; a run
// is read whole before any of it is written.  What run j writes lies below the run's end, and every entry beyond that
// end reads a position at or beyond it, so later runs still find their lines.  Runs of one line slice must follow one
// another, but slices of a line (a few 16-byte chunks of K or of V) and heads are independent: a workgroup owns one.
//
// Few requests give few such workgroups, and a run waits for memory once.  Then most lines move in launches of their own
// that need no order within: call an entry of level 0 if its position lies at or beyond the budget, so that no entry
// overwrites it, and of level k + 1 if its position is that of an entry of level k, which overwrites it.  Entries of one
// level read what lies outside the level, so a level moves at once, and higher levels have to move first.  As kept
// ascends, higher levels are lower entries: the runs move what is left at the front, then the levels follow, 0 last.
#include "kv_eviction.h"

namespace psi {

typedef uint32_t unit_u32x4 __attribute__((ext_vector_type(4)));

struct CompactArgs {
    CacheView v;
    void* pages;
    float* page_weights;  // null: no accumulators beside this cache
    const uint32_t* requests;
    const uint32_t* kept;
    uint32_t* status;
    uint32_t max_cached, budget;
    uint32_t line_units, slice_units, num_slices;  // units of a line, of a slice; slices of a line
    uint32_t num_reqs, group_stride;               // group_stride: workgroups between two slices of a line
    uint32_t levels;                               // entries of lower levels move in launches of their own
};

// The request of a workgroup; false: there is nothing to move.
__device__ __forceinline__ bool load_request(const CompactArgs& a, uint32_t req, uint32_t* slot, uint32_t* n) {
    *slot = a.requests[req * kRequestWords];
    *n = min(min(a.requests[req * kRequestWords + 1], a.max_cached), a.v.positions);
    if (*n <= a.budget) return false;  // everything is kept where it is
    if (*slot >= a.v.num_slots) {
        report_cache_range(a.status);
        return false;
    }
    return true;
}

// First of `count` ascending values that is `bound` or more, by a wave: 64 probes a step.
__device__ __forceinline__ uint32_t lower_bound(const uint32_t* values, uint32_t count, uint32_t bound) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t lo = 0, hi = count;  // values below lo are less than bound, hi's (if any) is not
    while (lo < hi) {
        const uint32_t step = (hi - lo + 63) / 64, at = lo + lane * step;
        const uint64_t reached = __ballot(at >= hi || values[min(at, hi - 1)] >= bound);
        const uint32_t first = reached != 0 ? (uint32_t)__builtin_ctzll(reached) : 64;
        if (first < 64) hi = min(hi, lo + first * step);
        if (first > 0) lo = min(hi, lo + (first - 1) * step + 1);
    }
    return lo;
}

// The runs of one (request, KV head, slice): a workgroup takes `per_step` lines at a time, a unit a lane, kUnroll
// steps a run.  No run writes what a later one reads, so the lines of the next run are asked for before those of this one
// have come; what they need is asked for ahead of that, a link of the chain per run: the kept positions three runs ahead,
// the page IDs two runs ahead.  (Loads come back in the order of their issue: lines are asked for after the page IDs and
// kept positions of an iteration, which the next one waits for first.)  Entries that move nothing read the first unit of
// the array in place of a line, so that the loads of a run stand without branches between them.
template <bool kStream, int kUnroll, typename Unit, typename Index>
__device__ __forceinline__ void move_runs(const CompactArgs& a, const uint32_t* kept, const uint32_t* table, uint32_t n,
                                          uint32_t entries, uint32_t num_pages, Unit* data, uint32_t my_line,
                                          uint32_t per_step, bool in_line, Index index) {
    const uint32_t per_run = per_step * kUnroll;
    struct Places {
        uint32_t src[kUnroll], from[kUnroll], to[kUnroll];
    };
    struct Lines {
        Unit held[kUnroll];
        uint32_t to[kUnroll];  // kNoPage: nothing is moved
    };
    auto entry = [&](uint32_t base, int u) -> uint32_t { return base + u * per_step + my_line; };
    auto fetch_kept = [&](uint32_t base, uint32_t (&out)[kUnroll]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t i = entry(base, u);
            const bool there = in_line && i < entries;
            const uint32_t k = kept[there ? i : 0];
            out[u] = there ? k : i;  // an entry that stays where it is moves nothing
        }
    };
    auto fetch_pages = [&](uint32_t base, const uint32_t (&at)[kUnroll], Places& p) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t i = entry(base, u);
            const bool moves = at[u] > i && at[u] < n;  // (n's positions have entries in the table)
            p.src[u] = at[u];
            p.from[u] = table[moves ? page_index(a.v, at[u]) : 0];
            p.to[u] = table[moves ? page_index(a.v, i) : 0];
            if (!moves) p.to[u] = kNoPage;
        }
    };
    auto fetch_lines = [&](uint32_t base, const Places& p, Lines& l) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const bool found = p.from[u] < num_pages && p.to[u] < num_pages;
            // beyond the cached tokens or the arena, or not ascending: nothing is moved for this entry
            if (!found && p.src[u] != entry(base, u)) report_cache_range(a.status);
            const Unit* from = data + (found ? index(p.from[u], p.src[u]) : 0);
            l.held[u] = kStream ? __builtin_nontemporal_load(from) : *from;
            l.to[u] = found ? p.to[u] : kNoPage;
        }
    };
    auto store_lines = [&](uint32_t base, Lines& l) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) asm volatile("" : "+v"(l.held[u]));  // the run has been read ...
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();  // ... by every wave before any of it is written
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (l.to[u] != kNoPage) data[index(l.to[u], entry(base, u))] = l.held[u];
    };
    if (entries == 0) return;
    uint32_t at[kUnroll];
    Places even, odd;
    Lines first, second;
    fetch_kept(0, at);
    fetch_pages(0, at, even);
    fetch_kept(per_run, at);
    fetch_pages(per_run, at, odd);
    fetch_kept(2 * per_run, at);
    fetch_lines(0, even, first);
    for (uint32_t base = 0; base < entries; base += 2 * per_run) {
        fetch_pages(base + 2 * per_run, at, even);
        fetch_kept(base + 3 * per_run, at);
        fetch_lines(base + per_run, odd, second);
        store_lines(base, first);
        if (base + per_run >= entries) break;
        fetch_pages(base + 3 * per_run, at, odd);
        fetch_kept(base + 4 * per_run, at);
        fetch_lines(base + 2 * per_run, even, first);
        store_lines(base + per_run, second);
    }
}

// One workgroup per (slice, request, KV head, K | V), then one per (request, KV head) for the accumulators; slice_units
// divides kThreads.  The slices of a line are a multiple of eight workgroups apart, so that they go to one XCD and share
// in its L2 the lines of memory that a slice of less than 128 bytes reads a part of.
template <typename Unit, int kThreads, int kUnroll, bool kStream>
__global__ __launch_bounds__(kThreads, kThreads == 1024 ? 4 : 8) void compact_kernel(CompactArgs a) {
    const uint32_t line_groups = a.group_stride * a.num_slices;
    const bool is_weights = blockIdx.x >= line_groups;
    const uint32_t pair = is_weights ? (blockIdx.x - line_groups) * 2 : blockIdx.x % a.group_stride;
    const uint32_t kind = pair % 2, kv_head = pair / 2 % a.v.hkv, req = pair / 2 / a.v.hkv;
    if (req >= a.num_reqs) return;
    uint32_t slot, n;
    if (!load_request(a, req, &slot, &n)) return;
    const uint32_t* kept = a.kept + ((uint64_t)req * a.v.hkv + kv_head) * a.budget;
    const uint32_t* table = table_row(a.v, slot, a.v.layer);
    uint32_t entries = a.budget;
    for (uint32_t l = 0; l < a.levels; ++l) entries = lower_bound(kept, entries, entries);
    if (is_weights) {
        move_runs<kStream, kUnroll>(a, kept, table, n, entries, a.v.num_weight_pages, reinterpret_cast<uint32_t*>(a.page_weights),
                           threadIdx.x, kThreads, true, [&](uint32_t page, uint32_t position) {
                               return weight_index(a.v, page, kv_head, page_place(a.v, position));
                           });
        return;
    }
    const uint32_t my_unit = blockIdx.x / a.group_stride * a.slice_units + threadIdx.x % a.slice_units;
    move_runs<kStream, kUnroll>(a, kept, table, n, entries, a.v.num_pages, static_cast<Unit*>(a.pages), threadIdx.x / a.slice_units,
                       kThreads / a.slice_units, my_unit < a.line_units, [&](uint32_t page, uint32_t position) -> uint64_t {
                           const uint64_t line = (((uint64_t)page * 2 + kind) * a.v.hkv + kv_head) * a.v.tokens_per_page +
                                                 page_place(a.v, position);
                           return line * a.line_units + my_unit;
                       });
}

// The entries of one level: a workgroup takes kLevelEntries of a (request, KV head), whole lines of 2^log2_line units of
// 16 bytes, K and V, eight units of a thread under way (78 us with 64 entries a workgroup, 86 with 128, 90 with 256).
constexpr uint32_t kLevelEntries = 64, kLevelThreads = 256;
__global__ __launch_bounds__(kLevelThreads) void compact_level_kernel(CompactArgs a, uint32_t level, uint32_t log2_line,
                                                                      uint32_t chunks) {
    const uint32_t kv_head = blockIdx.x / chunks % a.v.hkv, req = blockIdx.x / chunks / a.v.hkv;
    const uint32_t base = blockIdx.x % chunks * kLevelEntries;
    uint32_t slot, n;
    if (!load_request(a, req, &slot, &n)) return;
    const uint32_t* kept = a.kept + ((uint64_t)req * a.v.hkv + kv_head) * a.budget;
    const uint32_t* table = table_row(a.v, slot, a.v.layer);
    __shared__ uint64_t from_line[kLevelEntries], to_line[kLevelEntries];  // of K; all ones: nothing to move
    __shared__ uint32_t moving;
    constexpr uint64_t kNoLine = ~0ull;
    const uint64_t kind_lines = (uint64_t)a.v.hkv * a.v.tokens_per_page;  // from a line of K to its line of V
    if (threadIdx.x < kLevelEntries) {
        const uint32_t i = base + threadIdx.x;
        uint32_t at = i, src = i;
        bool ours = i < a.budget;
        for (uint32_t l = 0; l <= level; ++l) {
            const uint32_t next = ours ? kept[at] : 0;
            if (l == 0) src = next;
            ours = ours && (l < level ? next > at && next < a.budget : next >= a.budget);
            at = next;
        }
        from_line[threadIdx.x] = kNoLine;
        if (ours) {
            const bool there = src < n;
            const uint32_t from = there ? table[page_index(a.v, src)] : kNoPage;
            const uint32_t to = there ? table[page_index(a.v, i)] : kNoPage;
            if (from < a.v.num_pages && to < a.v.num_pages) {
                auto line_of = [&](uint32_t page, uint32_t p) {
                    return ((uint64_t)page * 2 * a.v.hkv + kv_head) * a.v.tokens_per_page + page_place(a.v, p);
                };
                from_line[threadIdx.x] = line_of(from, src);
                to_line[threadIdx.x] = line_of(to, i);
            } else {
                report_cache_range(a.status);
            }
            if (a.page_weights != nullptr) {
                if (from < a.v.num_weight_pages && to < a.v.num_weight_pages)
                    a.page_weights[weight_index(a.v, to, kv_head, page_place(a.v, i))] =
                        a.page_weights[weight_index(a.v, from, kv_head, page_place(a.v, src))];
                else
                    report_cache_range(a.status);
            }
        }
        const uint64_t any = __ballot(ours);
        if (threadIdx.x == 0) moving = any != 0;
    }
    __syncthreads();
    if (!moving) return;
    unit_u32x4* data = static_cast<unit_u32x4*>(a.pages);
    constexpr int kUnroll = 8;
    const uint32_t units = kLevelEntries * 2 << log2_line;
    for (uint32_t u0 = threadIdx.x; u0 < units; u0 += kLevelThreads * kUnroll) {
        unit_u32x4 held[kUnroll];
        uint64_t target[kUnroll];
        bool moves[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const uint32_t at = u0 + u * kLevelThreads, line = at >> log2_line, unit = at & ((1u << log2_line) - 1);
            const uint32_t entry = min(line / 2, kLevelEntries - 1);
            moves[u] = at < units && from_line[entry] != kNoLine;
            const uint64_t kind = line % 2 ? kind_lines : 0;
            held[u] = __builtin_nontemporal_load(data + (moves[u] ? ((from_line[entry] + kind) << log2_line) + unit : 0));
            target[u] = ((to_line[entry] + kind) << log2_line) + unit;
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (moves[u]) data[target[u]] = held[u];
    }
}

// Slices of a line: down to 128 bytes until there are four workgroups to a compute unit (32 requests of 1k-8k tokens cut
// to 1024, 4 heads of 256: 86 us with whole lines, 48 us with 128 bytes, both with part of the lines in the memory-side
// cache; with none there 57 us, which is 4.6 TB/s read and written); where that leaves compute units without one, down to 32 bytes (one request of 8000 cut to 4000, 2 heads of 256: 14.4 us, 15.3 with
// 64 bytes; two of 65536 cut to 50000, 4 heads of 128: 164 and 172 us).
inline uint32_t compact_slices(uint64_t pairs, uint32_t line_bytes) {
    uint32_t slices = 1;
    auto can_halve = [&](uint32_t least) { return line_bytes / (2 * slices) >= least; };
    while ((slices * pairs < 1024 && can_halve(128)) || (slices * pairs < 256 && can_halve(32))) slices *= 2;
    return slices;
}

// Levels that get launches of their own, where the runs have a workgroup for every second compute unit at most: as long
// as a level is likely to hold kLevelLeast entries, if the share of a request that is kept is spread evenly.  Without, with
// one, with all of them: one request of 61001 cut to 30000 (4 heads of 256) 126, 78, 72 us; one of 131072 cut to 30000 (1
// head of 256) 76, 36, 31 us; two of 65536 cut to 50000 (4 heads of 128) 197, 181, 164 us (seven levels cost what they
// gain); four of 16000 cut to 8000 (8 heads of 128), 256 workgroups, 61 us either way.
constexpr uint32_t kFewGroups = 128, kLevelLeast = 2048, kMostLevels = 4;
inline uint32_t compact_levels(uint64_t groups, uint32_t budget, uint32_t max_cached) {
    if (groups > kFewGroups || max_cached <= budget) return 0;
    const double share = (double)budget / max_cached;
    uint32_t levels = 0;
    for (double left = budget; levels < kMostLevels && left * (1.0 - share) >= kLevelLeast; left *= share) ++levels;
    return levels;
}

template <typename Unit>
static void launch_compact(psi_hip_ctx* ctx, const CompactArgs& a, uint32_t grid) {
    // Many workgroups: a unit a lane, four workgroups to a compute unit, streaming loads (the 32 requests above, cached in
    // part: 48 us; 57 with two units, whose registers leave room for three; 65 with ordinary loads, 65 with the other
    // launch).  Few: long
    // runs and ordinary loads, as slices share lines of memory (one of 8000 cut to 4000: 14.4 us, 18.9 with the other
    // launch; four of 16000 cut to 8000: 61 and 76 us).
    if (grid >= 512)
        hipLaunchKernelGGL((compact_kernel<Unit, 512, 1, true>), dim3(grid), dim3(512), 0, ctx->stream, a);
    else
        hipLaunchKernelGGL((compact_kernel<Unit, 1024, 4, false>), dim3(grid), dim3(1024), 0, ctx->stream, a);
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
    PSI_REQUIRE(budget > 0 && budget <= INT32_MAX, "the budget must be positive and below 2^31");
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
    const uint64_t pairs = (uint64_t)num_reqs * g.hkv * 2, stride = (pairs + 7) / 8 * 8;
    const uint32_t slices = compact_slices(pairs, line_bytes);
    a.slice_units = 1;
    while (a.slice_units < 512 && a.slice_units * slices < a.line_units) a.slice_units *= 2;
    a.num_slices = (a.line_units + a.slice_units - 1) / a.slice_units;
    a.num_reqs = num_reqs;
    const uint64_t grid = stride * a.num_slices + (page_weights != nullptr ? pairs / 2 : 0);
    PSI_REQUIRE(grid <= 0x7fffffffull, "too many requests in one compaction");
    a.levels = 0;
    const uint64_t chunks = ((uint64_t)budget + kLevelEntries - 1) / kLevelEntries;
    const uint64_t level_grid = chunks * (pairs / 2);
    if (unit == 16 && (a.line_units & (a.line_units - 1)) == 0 && level_grid <= 0x7fffffffull)
        a.levels = compact_levels(pairs * a.num_slices, budget, max_cached_tokens);
    DeviceGuard guard(ctx->device);
    LaunchScope scope(ctx, "kv_compact");
    a.group_stride = (uint32_t)stride;
    if (unit == 16) launch_compact<unit_u32x4>(ctx, a, (uint32_t)grid);
    else if (unit == 4) launch_compact<uint32_t>(ctx, a, (uint32_t)grid);
    else launch_compact<uint16_t>(ctx, a, (uint32_t)grid);
    for (uint32_t level = a.levels; level-- > 0;)
        hipLaunchKernelGGL(compact_level_kernel, dim3((uint32_t)level_grid), dim3(kLevelThreads), 0, ctx->stream, a, level,
                           (uint32_t)__builtin_ctz(a.line_units), (uint32_t)chunks);
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
