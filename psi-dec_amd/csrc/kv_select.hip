// Which cached tokens a (request, KV head) keeps: the first num_first, the last num_recent, and of the others those with
// the largest accumulated weight until `budget` are chosen; equal weights go to the lower position.  The chosen
// positions come out in ascending order.  A NaN weight counts as -inf, -0 as 0.
//
// The budget-th largest weight is found by radix selection on order-preserving integer keys (three digits, counted in
// LDS), the positions by ballots and prefix counts: no sort, and the same answer on every run.
#include "kv_eviction.h"

#include <algorithm>

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
// Digits of a key, from the top: 11, 11 and 10 bits.  The first one holds the sign, the exponent and two bits of the
// mantissa, so that accumulated weights, which span few exponents, still spread over some tens of counters.
constexpr uint32_t kBins = 2048;
constexpr int kDigits = 3;
__device__ __forceinline__ uint32_t digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t digit_of(uint32_t key, int d) { return d == 2 ? key & 1023 : key >> digit_shift(d) & 2047; }

struct SelectRow {
    const uint32_t* table;
    uint32_t kv_head, n, recent_from;
    bool vector;  // four adjacent positions share a page and a 16-byte aligned address
};
__device__ __forceinline__ SelectRow make_row(const SelectArgs& a, uint32_t slot, uint32_t kv_head, uint32_t n) {
    SelectRow r;
    r.table = table_row(a.v, slot, a.v.layer);
    r.kv_head = kv_head;
    r.n = n;
    r.recent_from = n - min(a.num_recent, n);
    r.vector = a.v.log2_page < 32 && a.v.log2_page >= 2 && reinterpret_cast<uintptr_t>(a.page_weights) % 16 == 0;
    return r;
}

// Keys of positions p .. p + 3 (p a multiple of four); of positions from n on: 0, which no weight has (-inf's is higher).
__device__ __forceinline__ void load_keys(const SelectArgs& a, const SelectRow& r, uint32_t p, uint32_t (&key)[4]) {
    float w[4];
    uint32_t missing = 0;
    if (r.vector) {
        const uint32_t page = p < r.n ? page_of(a.v, r.table, p, a.v.num_weight_pages) : kNoPage;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (page != kNoPage)
            x = *reinterpret_cast<const float4*>(a.page_weights + weight_index(a.v, page, r.kv_head, page_place(a.v, p)));
        else missing = 15;
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
        w[3] = x.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t page = p + i < r.n ? page_of(a.v, r.table, p + i, a.v.num_weight_pages) : kNoPage;
            w[i] = 0.0f;
            if (page != kNoPage) w[i] = a.page_weights[weight_index(a.v, page, r.kv_head, page_place(a.v, p + i))];
            else missing |= 1u << i;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool always = p + i < a.num_first || p + i >= r.recent_from;
        if ((missing >> i & 1) && !always && p + i < r.n) {  // counts as the lightest
            w[i] = -INFINITY;
            report_cache_range(a.status);
        }
        key[i] = p + i >= r.n ? 0u : always ? kKeepKey : weight_key(w[i]);
    }
}

// What the selection of one row has settled after some digits: the keys to keep are those whose leading bits exceed
// `prefix`, and `remaining` of those whose leading bits equal it.
struct SelectState {
    uint32_t prefix, remaining;
};
__device__ __forceinline__ bool matches(uint32_t key, int digit, uint32_t prefix) {
    return digit == 0 || key >> digit_shift(digit - 1) == prefix;
}

struct BinSearch {
    uint32_t totals[kSelectWaves];
    uint32_t chosen[2];
};
// The counter that the `remaining`-th largest key falls into, and how many of that counter's keys are still to be kept.
// Thread t brings the counts of counters kBins - 1 - 2t (`high`) and the one below (`low`).
__device__ __forceinline__ void find_bin(BinSearch& lds, uint32_t tid, uint32_t high, uint32_t low, SelectState& st, int digit) {
    const uint32_t lane = tid & 63, wave = tid >> 6;
    uint32_t sum = high + low;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t other = __shfl_up(sum, off, 64);
        if ((int)lane >= off) sum += other;
    }
    if (lane == 63) lds.totals[wave] = sum;
    __syncthreads();
    uint32_t above = sum - high - low;
    for (uint32_t w = 0; w < wave; ++w) above += lds.totals[w];
    if (above < st.remaining && st.remaining <= above + high + low) {
        const bool first = st.remaining <= above + high;
        lds.chosen[0] = kBins - 1 - 2 * tid - (first ? 0 : 1);
        lds.chosen[1] = st.remaining - above - (first ? 0 : high);
    }
    __syncthreads();
    st.prefix = digit == 2 ? st.prefix << 10 | lds.chosen[0] : st.prefix << 11 | lds.chosen[0];
    st.remaining = lds.chosen[1];
}

// What every selection starts with: the row's request, the padding behind what it keeps, and the rows that keep all.
// False: nothing is left to do.
__device__ __forceinline__ bool begin_row(const SelectArgs& a, uint32_t row, bool writes, SelectRow* r, uint32_t** kept) {
    const uint32_t req = row / a.v.hkv, slot = a.requests[req * kRequestWords];
    const uint32_t n = min(min(a.requests[req * kRequestWords + 1], a.max_cached), a.v.positions);
    *kept = a.kept + (uint64_t)row * a.budget;
    const bool valid = slot < a.v.num_slots;
    if (writes) {
        const uint32_t filled = valid ? min(n, a.budget) : 0;
        for (uint32_t i = filled + threadIdx.x; i < a.budget; i += kSelectThreads) (*kept)[i] = PSI_HIP_SENTINEL;
        if (valid && n <= a.budget)
            for (uint32_t i = threadIdx.x; i < n; i += kSelectThreads) (*kept)[i] = i;
        if (!valid) report_cache_range(a.status);
    }
    if (!valid || n <= a.budget) return false;
    *r = make_row(a, slot, row % a.v.hkv, n);
    return true;
}

// Writes the kept positions among the four keys a thread holds in each of kQuads turns (turn q, thread t: positions
// first + 4 (q * 1024 + t) ..).  gt_before, eq_before: keys above and equal to the threshold ahead of `first`; of the equal
// ones the first `take` are kept.
struct EmitLds {
    uint32_t gt[16 * kSelectWaves], eq[16 * kSelectWaves];
};
template <int kQuads>
__device__ __forceinline__ void emit(const SelectArgs& a, EmitLds& lds, const uint32_t (&key)[kQuads][4], uint32_t first,
                                     uint32_t threshold, uint32_t take, uint32_t gt_before, uint32_t eq_before,
                                     uint32_t* kept) {
    static_assert(kQuads <= 16, "turns of a thread");
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint64_t lower = ((uint64_t)1 << lane) - 1;
    auto lanes_below = [&](uint32_t count, uint32_t* total) {  // sum over the lower lanes and over the wave; count <= 4
        const uint64_t b0 = __ballot(count & 1), b1 = __ballot(count & 2), b2 = __ballot(count & 4);
        *total = __popcll(b0) + 2 * __popcll(b1) + 4 * __popcll(b2);
        return (uint32_t)(__popcll(b0 & lower) + 2 * __popcll(b1 & lower) + 4 * __popcll(b2 & lower));
    };
    uint32_t gt_at[kQuads], eq_at[kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        uint32_t gt = 0, eq = 0, total;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            gt += key[q][i] > threshold;
            eq += key[q][i] == threshold;
        }
        gt_at[q] = lanes_below(gt, &total);
        if (lane == 0) lds.gt[q * kSelectWaves + wave] = total;
        eq_at[q] = lanes_below(eq, &total);
        if (lane == 0) lds.eq[q * kSelectWaves + wave] = total;
    }
    __syncthreads();
    for (uint32_t w = 0; w < wave; ++w) {
        gt_before += lds.gt[w];
        eq_before += lds.eq[w];
    }
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
        uint32_t gt = gt_before + gt_at[q], eq = eq_before + eq_at[q];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool above = key[q][i] > threshold, equal = key[q][i] == threshold;
            const uint32_t at = gt + min(eq, take);
            if ((above || (equal && eq < take)) && at < a.budget) kept[at] = first + 4 * (q * kSelectThreads + tid) + i;
            gt += above;
            eq += equal;
        }
        if (q + 1 < kQuads)
            for (uint32_t w = wave; w < wave + kSelectWaves; ++w) {  // the waves from this one on, then the next turn's first
                gt_before += lds.gt[q * kSelectWaves + w];
                eq_before += lds.eq[q * kSelectWaves + w];
            }
    }
}

// Counters in LDS, four copies that the lanes share out, so that the lanes of a wave that meet in a counter are fewer.
constexpr uint32_t kCopies = 4;
__device__ __forceinline__ void clear_bins(uint32_t* hist, uint32_t tid) {
    uint4* h = reinterpret_cast<uint4*>(hist);
    for (uint32_t i = tid; i < kCopies * kBins / 4; i += kSelectThreads) h[i] = make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ uint32_t bin_count(const uint32_t* hist, uint32_t bin) {
    uint32_t sum = 0;
#pragma unroll
    for (uint32_t c = 0; c < kCopies; ++c) sum += hist[c * kBins + bin];
    return sum;
}
template <int kQuads>
__device__ __forceinline__ void count_digits(uint32_t* hist, const uint32_t (&key)[kQuads][4], int digit, uint32_t prefix) {
    uint32_t* mine = hist + (threadIdx.x % kCopies) * kBins;
#pragma unroll
    for (int q = 0; q < kQuads; ++q)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (key[q][i] != 0 && matches(key[q][i], digit, prefix)) atomicAdd(&mine[digit_of(key[q][i], digit)], 1u);
}

// One workgroup per (request, KV head), its keys in registers: rows of up to 4096 * kQuads positions.
template <int kQuads>
__global__ __launch_bounds__(kSelectThreads) void select_row_kernel(SelectArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t hist[kCopies * kBins];
    __shared__ BinSearch search;
    __shared__ EmitLds emit_lds;
    SelectRow r;
    uint32_t* kept;
    if (!begin_row(a, blockIdx.x, true, &r, &kept)) return;
    const uint32_t tid = threadIdx.x;
    uint32_t key[kQuads][4];
#pragma unroll
    for (int q = 0; q < kQuads; ++q) load_keys(a, r, 4 * (q * kSelectThreads + tid), key[q]);
    SelectState st = {0, a.budget};
    for (int digit = 0; digit < kDigits; ++digit) {
        clear_bins(hist, tid);
        __syncthreads();
        count_digits<kQuads>(hist, key, digit, st.prefix);
        __syncthreads();
        find_bin(search, tid, bin_count(hist, kBins - 1 - 2 * tid), bin_count(hist, kBins - 2 - 2 * tid), st, digit);
    }
    emit<kQuads>(a, emit_lds, key, 0, st.prefix, st.remaining, 0, 0, kept);
}

// Longer rows: a workgroup per (row, chunk of 4096 or 8192 positions) and a launch per digit.  Each launch adds up the counters
// that the one before left for every chunk of the row, which gives the digit's value and, from the chunks ahead, the
// number of kept positions before this chunk's first; so nothing is cleared or added atomically in memory.
constexpr uint32_t chunk_keys(int quads) { return 4 * quads * kSelectThreads; }
struct ChunkState {
    uint32_t prefix, remaining, gt_before, unused;
};
inline uint64_t select_chunks(uint32_t max_cached, int quads) {
    return ((uint64_t)max_cached + chunk_keys(quads) - 1) / chunk_keys(quads);
}
// Chunks of 4096 while those of 8192 would leave half of the compute units without one (4 requests of 131072 on 2 heads: 28
// us for 30; 6 of up to 38290 on 4 heads: 25 for 29), which costs a chunk twice the counters to add up (40 requests of
// 30000 on 8 heads: 128 us for 100).
constexpr uint64_t kFewChunks = 128;
inline int chunk_quads(uint64_t rows, uint32_t max_cached) { return rows * select_chunks(max_cached, 2) <= kFewChunks ? 1 : 2; }
// Chunks that the scratch of a capacity holds: those of every selection of fewer rows or shorter requests too, though a
// launch of small chunks can have more of them than a larger one of large chunks.
inline uint64_t scratch_chunks(uint64_t rows, uint32_t max_cached) {
    static_assert(chunk_keys(2) == 2 * chunk_keys(1), "a large chunk makes at most two small ones");
    return std::max(rows * select_chunks(max_cached, 2), std::min(rows * select_chunks(max_cached, 1), 2 * kFewChunks));
}

// kPass 0 .. 2: counts digit kPass; kPass 3: writes the positions.
template <int kPass, int kChunkQuads>
__global__ __launch_bounds__(kSelectThreads) void select_chunk_kernel(SelectArgs a, uint32_t num_chunks, uint16_t* hists,
                                                                      ChunkState* states) {
    constexpr uint32_t kChunkKeys = chunk_keys(kChunkQuads);
    __shared__ __attribute__((aligned(16))) uint32_t hist[kCopies * kBins];
    __shared__ BinSearch search;
    __shared__ EmitLds emit_lds;
    __shared__ uint32_t wave_sum[kSelectWaves], equal_before;
    const uint32_t row = blockIdx.x / num_chunks, chunk = blockIdx.x % num_chunks, tid = threadIdx.x;
    SelectRow r;
    uint32_t* kept;
    if (!begin_row(a, row, kPass == 0 && chunk == 0, &r, &kept)) return;
    const uint32_t first = chunk * kChunkKeys, row_chunks = (r.n + kChunkKeys - 1) / kChunkKeys;
    if (chunk >= row_chunks) return;
    const uint64_t rows = gridDim.x / num_chunks;
    auto bins_of = [&](int digit, uint32_t c) { return hists + ((digit * rows + row) * num_chunks + c) * kBins; };
    uint32_t key[kChunkQuads][4];
#pragma unroll
    for (int q = 0; q < kChunkQuads; ++q) load_keys(a, r, first + 4 * (q * kSelectThreads + tid), key[q]);

    SelectState st = {0, a.budget};
    uint32_t gt_before = 0;
    if constexpr (kPass > 0) {
        ChunkState* mine = states + row * (uint64_t)num_chunks + chunk;
        if (kPass > 1) {
            const ChunkState s = *mine;
            st = {s.prefix, s.remaining};
            gt_before = s.gt_before;
        }
        // counters kBins - 1 - 2t and the one below: over the row, and over the chunks ahead
        uint32_t high = 0, low = 0, high_ahead = 0, low_ahead = 0;
        const uint32_t at = kBins - 2 - 2 * tid;
        constexpr uint32_t kAhead = 16;  // chunks asked for at a time
        for (uint32_t c0 = 0; c0 < row_chunks; c0 += kAhead) {
            uint32_t v[kAhead];
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u)
                v[u] = c0 + u < row_chunks ? *reinterpret_cast<const uint32_t*>(bins_of(kPass - 1, c0 + u) + at) : 0;
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) {
                low += v[u] & 0xffff;
                high += v[u] >> 16;
                if (c0 + u < chunk) {
                    low_ahead += v[u] & 0xffff;
                    high_ahead += v[u] >> 16;
                }
            }
        }
        find_bin(search, tid, high, low, st, kPass - 1);
        // keys ahead whose digit exceeds the chosen one, and (last digit) those that equal the threshold
        const uint32_t bin = search.chosen[0];
        uint32_t ahead = (at + 1 > bin ? high_ahead : 0) + (at > bin ? low_ahead : 0);
        if (at == bin) equal_before = low_ahead;
        if (at + 1 == bin) equal_before = high_ahead;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) ahead += __shfl_xor(ahead, off, 64);
        if ((tid & 63) == 0) wave_sum[tid >> 6] = ahead;
        __syncthreads();
        for (uint32_t w = 0; w < kSelectWaves; ++w) gt_before += wave_sum[w];
        if (kPass < 3 && tid == 0) *mine = {st.prefix, st.remaining, gt_before, 0};
    }
    if constexpr (kPass < 3) {
        clear_bins(hist, tid);
        __syncthreads();
        count_digits<kChunkQuads>(hist, key, kPass, st.prefix);
        __syncthreads();
        static_assert(kBins == 2 * kSelectThreads && kChunkKeys < 65536, "two counters of 16 bits a thread");
        reinterpret_cast<uint32_t*>(bins_of(kPass, chunk))[tid] = bin_count(hist, 2 * tid) | bin_count(hist, 2 * tid + 1) << 16;
    } else {
        emit<kChunkQuads>(a, emit_lds, key, first, st.prefix, st.remaining, gt_before, equal_before, kept);
    }
}

// Rows of up to this many positions go to one workgroup each: what its registers hold.  One launch of it takes 17 us at
// 16384 positions and 11 at 8192, the four launches over chunks 23 and 22 (32 sequences: 19 and 12 against 31 and 25).
constexpr uint32_t kRowPositions = 16384;

}  // namespace psi

using namespace psi;

extern "C" int psi_hip_kv_select_scratch_bytes(const psi_hip_gqa_config* cfg, uint32_t num_reqs,
                                               uint32_t max_cached_tokens, uint64_t* out_bytes) {
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(out_bytes != nullptr, "out pointer must not be null");
    PSI_REQUIRE(num_reqs > 0, "a selection needs requests");
    const uint64_t rows = (uint64_t)num_reqs * g.hkv;
    *out_bytes = max_cached_tokens <= kRowPositions
                     ? 0
                     : scratch_chunks(rows, max_cached_tokens) * (kDigits * kBins * 2 + sizeof(ChunkState));
    return PSI_HIP_OK;
}

extern "C" int psi_hip_kv_select_kept(psi_hip_ctx* ctx, const psi_hip_gqa_config* cfg,
                                      const psi_hip_page_table_layout* layout, const float* page_weights,
                                      uint64_t page_weights_bytes, const uint32_t* page_ids, const uint32_t* requests,
                                      uint32_t num_reqs, uint32_t max_cached_tokens, uint32_t budget, uint32_t num_first,
                                      uint32_t num_recent, uint32_t* kept, void* scratch, uint64_t scratch_bytes,
                                      uint32_t gqa_layer_index) {
    PSI_REQUIRE(ctx != nullptr, "ctx must not be null");
    Geometry g;
    int rc = make_geometry(cfg, &g);
    if (rc != PSI_HIP_OK) return rc;
    rc = check_no_replay_counts(ctx);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(page_weights && requests && kept, "selection buffers must not be null");
    PSI_REQUIRE(num_reqs > 0, "a selection needs requests");
    PSI_REQUIRE(budget > 0 && budget <= INT32_MAX, "the budget must be positive and below 2^31");
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
    uint64_t needed = 0;
    rc = psi_hip_kv_select_scratch_bytes(cfg, num_reqs, max_cached_tokens, &needed);
    if (rc != PSI_HIP_OK) return rc;
    PSI_REQUIRE(scratch_bytes >= needed && (needed == 0 || scratch != nullptr), "selection scratch too small: %llu < %llu",
                (unsigned long long)scratch_bytes, (unsigned long long)needed);
    PSI_REQUIRE(reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "the selection scratch must be 16-byte aligned");
    const uint32_t rows = num_reqs * g.hkv;
    DeviceGuard guard(ctx->device);
    LaunchScope scope(ctx, "kv_select");
    const dim3 threads(kSelectThreads);
    if (max_cached_tokens <= 4096) {
        hipLaunchKernelGGL(select_row_kernel<1>, dim3(rows), threads, 0, ctx->stream, a);
    } else if (max_cached_tokens <= 8192) {
        hipLaunchKernelGGL(select_row_kernel<2>, dim3(rows), threads, 0, ctx->stream, a);
    } else if (max_cached_tokens <= kRowPositions) {
        hipLaunchKernelGGL(select_row_kernel<4>, dim3(rows), threads, 0, ctx->stream, a);
    } else {
        const int quads = chunk_quads(rows, max_cached_tokens);
        const uint64_t chunks = select_chunks(max_cached_tokens, quads), grid = rows * chunks;
        PSI_REQUIRE(grid <= 0x7fffffffull, "too many requests of this length in one selection");
        uint16_t* hists = static_cast<uint16_t*>(scratch);
        ChunkState* states = reinterpret_cast<ChunkState*>(hists + grid * kDigits * kBins);
        const dim3 blocks((uint32_t)grid);
        auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, blocks, threads, 0, ctx->stream, a, (uint32_t)chunks, hists, states);
        };
        launch(quads == 1 ? select_chunk_kernel<0, 1> : select_chunk_kernel<0, 2>);
        launch(quads == 1 ? select_chunk_kernel<1, 1> : select_chunk_kernel<1, 2>);
        launch(quads == 1 ? select_chunk_kernel<2, 1> : select_chunk_kernel<2, 2>);
        launch(quads == 1 ? select_chunk_kernel<3, 1> : select_chunk_kernel<3, 2>);
    }
    PSI_HIP_CHECK(hipGetLastError());
    return PSI_HIP_OK;
}
