// gfx950 observation kernels for 2-byte K and head_dim 128 or 256, any page size.
//
// One workgroup = one (row of keys, KV head).  The window's columns are staged in LDS in the operand order of the matrix
// product; a wave takes 16 * kTiles keys at a time straight from their pages into registers, in the operand order too (as
// in split_kv_decode_kernel.h: lane = token lane%16, 8-dim chunk lane/16, a 128-bit load per 32 dims), and multiplies
// them with one block of 16 columns after the other.  The keys stay in registers for all columns, so that a column
// operand read from LDS (8 cycles of the compute unit's LDS) feeds kTiles products (16 cycles of a SIMD each), and waves
// share nothing but the columns: there is no barrier in the loops over keys and columns.
//
// A result lane holds 4 * kTiles keys of one column: the maximum and sum of a column (first pass) are reduced over the
// lane and then over the four lanes of the column, the weights of a key (second pass) over the columns of a lane first
// and over the lanes once per turn.  Where waves share the columns of a key, their sums meet in LDS.
//
// Measured: 8 prompts of 1k-8k (bf16, D 256, 32 tokens, 24 heads over 4) 56-61 us for two walks of 75 MB and 2 * 14
// GFLOP; one prompt of 65536 (D 128, 64 tokens, 40 heads over 8) 122-126 us for 2 * 134 MB and 2 * 43 GFLOP, 690 TFLOP/s.
// More columns than the LDS holds at a time (256 with D 256, 384 with D 128) take another walk over the keys for each
// such part in both passes: a whole prompt of 2048 tokens 0.58 ms (40 heads over 8 of 128).  The first of these is bound by the lines: a workgroup has two turns, each a burst of reads and then a wait (27 of 33 us of its first pass
// remained with a sixth of the products).  The second is bound by products and exponentials, which share a SIMD's issue.
#pragma once
#include "kv_observe.h"
#include "split_kv_decode_kernel.h"

namespace psi {

// Normalisers are joined inside the second pass as long as (rows of the longest window) * (columns) stays within this,
// which saves a launch (at 104: 13.2 for 15.7 us in all, at 2496: 55.7 for 58.5, at 6656: 10.9 for 13.3); at 8064 and 9024
// the two come out even (24.8 for 23.9, 59.2 for 58.8), and beyond, repeating the join in every workgroup of a long window
// costs more than a launch, however short the other windows are (one prompt of 60000 beside three of 500, 22656: 44 for 39
// us; one of 100000 beside 31 of 64, 57344: 53 for 44; one of 200000 beside 63 of 64, 94208: 139 for 117).
constexpr uint64_t kFusedJoins = 8192;

// Blocks of columns from which the waves of a short row share them: 64 tokens, 40 heads over 8, of one prompt of 1500
// take 25 us for 34, 70 tokens, 12 heads over 2, of four of 413-826 35 us for 45; with 12 or 13 blocks sharing changes
// little (14 prompts of 100: 28 us for 29, two of 550: 26 for 25).
constexpr uint32_t kShareBlocks = 16;

template <int kCtrl>
__device__ __forceinline__ float dpp_of(float x) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), kCtrl, 0xf, 0xf, false));
}
// One step of the sum over the 16 lanes of a DPP row that leaves value i to lane i: the lane keeps the half of its values
// that `high` names and adds the other half of the lane that kCtrl pairs it with.
template <int kCtrl, int kHalf>
__device__ __forceinline__ void halve_sums(float (&v)[16], bool high) {
#pragma unroll
    for (int i = 0; i < kHalf; ++i) {
        const float keep = high ? v[i + kHalf] : v[i], give = high ? v[i] : v[i + kHalf];
        v[i] = keep + dpp_of<kCtrl>(give);
    }
}
// Sum over the 16 lanes of a row of each of 16 values; lane i % 16 gets value i's.  Row mirror, half-row mirror and the
// two quad permutations pair the lanes by 15, 7, 2 and 1 in exclusive or, which together reach every lane of the row.
__device__ __forceinline__ float row_sums(float (&v)[16], uint32_t lane) {
    halve_sums<0x140, 8>(v, lane & 8);
    halve_sums<0x141, 4>(v, lane & 4);
    halve_sums<0x4e, 2>(v, lane & 2);
    halve_sums<0xb1, 1>(v, lane & 1);
    return v[0];
}

// Barrier that orders LDS only: K lines that a wave has asked for stay on their way.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// kSum false: the maxima and sums of the row's columns.  kSum true: the weights.
template <typename Tag, int D, int kTiles, int kBlocks, int kMaxBlocks, int kWaves, bool kSum>
__global__ __launch_bounds__(64 * kWaves, kWaves / 4) void observe_kernel(ObserveArgs a) {
    static_assert(kMaxBlocks % kBlocks == 0, "whole steps of columns");
    constexpr int kSteps = D / 32;
    constexpr uint32_t kThreads = 64 * kWaves, kColumns = 16 * kMaxBlocks, kChunks = D / 8;
    constexpr int kWords = (kTiles + 3) / 4;
    constexpr uint32_t kKeys = 16 * kTiles, kTurn = kWaves * kKeys;  // keys of a wave's turn, of all waves'
    __shared__ __attribute__((aligned(16))) uint4 q_lds[kMaxBlocks * kSteps * 64];
    __shared__ int last_lds[kColumns];                                  // last key of the row that a column sees
    __shared__ float2 norm_lds[kSum ? kColumns : 1];
    __shared__ float part_lds[kSum && kMaxBlocks >= kShareBlocks ? kWaves * kKeys : 1];  // sums over a part of the columns
    __shared__ float2 state_lds[kSum ? 1 : kWaves][kSum ? 1 : kColumns];  // maximum and sum so far

    const uint32_t row = blockIdx.x / a.v.hkv, kv_head = blockIdx.x % a.v.hkv;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lane_row = lane & 15, lane_quarter = lane >> 4;
    const ObserveRow r = load_row(a, row);
    if (!r.live) return;
    const uint32_t* table = table_row(a.v, r.slot, a.v.layer);
    const uint16_t* q = static_cast<const uint16_t*>(a.q);
    const uint16_t* pages = static_cast<const uint16_t*>(a.pages);
    const uint32_t columns = r.num_q * a.group;

    for (uint32_t c0 = 0; c0 < columns; c0 += kColumns) {
        const uint32_t count = min(columns - c0, kColumns), blocks = (count + 16 * kBlocks - 1) / (16 * kBlocks) * kBlocks;
        const uint32_t key_end = min(r.end, r.position + (c0 + count - 1) / a.group + 1);  // what the last column sees
        // Short rows of many columns: the waves that have no keys of their own share the columns of the others' keys.
        const uint32_t length = key_end > r.begin ? key_end - r.begin : 0, key_groups = max((length + kKeys - 1) / kKeys, 1u);
        const bool share = kMaxBlocks >= kShareBlocks && blocks >= kShareBlocks && key_groups * 2 <= kWaves;
        const uint32_t parts = share ? min(kWaves / key_groups, blocks / kBlocks) : 1;
        const uint32_t part = share ? wave / key_groups : 0, key_group = share ? wave % key_groups : wave;
        const uint32_t part_blocks = (blocks / kBlocks + parts - 1) / parts * kBlocks;
        const uint32_t block_begin = part * part_blocks, block_end = min(blocks, block_begin + part_blocks);
        // The page IDs of a wave's turn are asked for a turn ahead.  Its lines are not: a second buffer of them costs the
        // registers of a wave in three, and the other waves of the SIMD fill the wait better (one prompt of 65536, 64
        // tokens: 78 and 60 us a pass with two buffers, 68 and 57 with one).
        uint32_t next_ids[kTiles];
        auto fetch_ids = [&](uint32_t base) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
                next_ids[t] = page_of(a.v, table, min(base + t * 16 + lane_row, key_end - 1), a.v.num_pages);
        };
        struct Keys {
            uint4 line[kTiles][kSteps];
            uint64_t missing[kWords];  // keys on pages beyond the arena: bit t % 4 * 16 + row of word t / 4
        };
        auto fetch_lines = [&](uint32_t base, Keys& k) __attribute__((always_inline)) {
            bool bad = false;
#pragma unroll
            for (int t = 0; t < kTiles; ++t) {
                const uint32_t p = min(base + t * 16 + lane_row, key_end - 1);
                const bool missing = next_ids[t] == kNoPage;
                bad |= missing;
                const uint16_t* line = pages + line_index(a.v, missing ? 0 : next_ids[t], 0, kv_head, page_place(a.v, p)) +
                                       lane_quarter * 8;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) k.line[t][i] = *reinterpret_cast<const uint4*>(line + i * 32);
            }
#pragma unroll
            for (int w = 0; w < kWords; ++w) k.missing[w] = 0;
            if (__any(bad)) {
                report_cache_range(a.status);
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                    k.missing[t / 4] |= (__ballot(next_ids[t] == kNoPage) & 0xffffull) << (16 * (t % 4));
            }
        };
        Keys k;
        // The second pass walks the turns backwards: what the first pass read last may still be in the cache of the XCD
        // (27.3 for 28.8 us at 8 prompts of 1k-8k, the same at 65536).  Loads are ordinary ones for that reason: streaming
        // ones take 33 + 31 us for 30 + 27, and 67 + 58 for 62 + 52 at 65536.
        const uint32_t first = r.begin + key_group * kKeys;
        uint32_t turns = first < key_end && block_begin < block_end ? (key_end - first + kTurn - 1) / kTurn : 0;
        const uint32_t step = kSum ? 0 - kTurn : kTurn;
        uint32_t base = kSum ? first + (turns - 1) * kTurn : first;
        if (turns > 0) {
            fetch_ids(base);
            fetch_lines(base, k);  // on their way while the columns are staged
            if (turns > 1) fetch_ids(base + step);
        }

        if (c0 > 0) __syncthreads();
        constexpr int kStage = 4;  // units of a thread under way
        const uint32_t units = blocks * 16 * kChunks;
        for (uint32_t i0 = tid; i0 < units; i0 += kThreads * kStage) {
            uint4 value[kStage];
#pragma unroll
            for (int u = 0; u < kStage; ++u) {
                // (columns that fill up the last block repeat the last one: what is finite there stays finite)
                const uint32_t i = i0 + u * kThreads, c = min(c0 + i / kChunks, columns - 1);
                const uint64_t q_row = (uint64_t)(r.q_begin + c / a.group) * a.hq + kv_head * a.group + c % a.group;
                value[u] = *reinterpret_cast<const uint4*>(q + q_row * D + i % kChunks * 8);
            }
#pragma unroll
            for (int u = 0; u < kStage; ++u) {
                const uint32_t i = i0 + u * kThreads, column = i / kChunks, chunk = i % kChunks;
                if (i < units)
                    q_lds[((column / 16) * kSteps + chunk / 4) * 64 + (chunk % 4) * 16 + column % 16] = value[u];
            }
        }
        for (uint32_t i = tid; i < blocks * 16; i += kThreads) {
            const uint32_t c = c0 + i;
            last_lds[i] = c < columns ? (int)min(r.position + c / a.group, key_end - 1) : -1;
            if (kSum && (a.norm != nullptr || c >= columns))
                norm_lds[i] = c >= columns
                                  ? make_float2(INFINITY, 0.0f)
                                  : a.norm[(uint64_t)(r.q_begin + c / a.group) * a.hq + kv_head * a.group + c % a.group];
        }
        if (kSum && a.norm == nullptr) {
            // a column's rows are shared out among the lanes that its neighbours leave (8 tokens of 13234, 208 rows: 10.9
            // us for 19.8 with a lane a column)
            const uint32_t rows = r.row_end - min(r.row_begin, r.row_end);
            uint32_t parts = 1;
            while (parts < 64 && 2 * parts * count <= kThreads && 8 * parts < rows) parts *= 2;
            for (uint32_t i = tid; i < count * parts; i += kThreads) {
                const float2 norm = join_column(a, r, kv_head, c0 + i / parts, i % parts, parts);
                if (i % parts == 0) norm_lds[i / parts] = norm;
            }
        }
        if constexpr (!kSum)
            for (uint32_t i = lane; i < blocks * 16; i += 64) state_lds[wave][i] = make_float2(kEmptyMax, 0.0f);
        lds_barrier();

        for (; turns > 0; --turns, base += step) {
            bool masked = base + kKeys > min(r.position + 1, key_end);
#pragma unroll
            for (int w = 0; w < kWords; ++w) masked |= k.missing[w] != 0;
            float sums[kWords][16];
            if constexpr (kSum) {
#pragma unroll
                for (int w = 0; w < kWords; ++w)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sums[w][i] = 0.0f;
            }
            for (uint32_t b0 = block_begin; b0 < block_end; b0 += kBlocks) {
                // kBlocks blocks at a time: independent products and exponentials to fill each other's latencies
                f32x4_t acc[kBlocks][kTiles];
#pragma unroll
                for (int h = 0; h < kBlocks; ++h) {
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) acc[h][t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        const uint4 qv = q_lds[((b0 + h) * kSteps + i) * 64 + lane];
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) acc[h][t] = mfma_16x16x32<Tag>(k.line[t][i], qv, acc[h][t]);
                    }
                }
                if (masked) {
#pragma unroll
                    for (int h = 0; h < kBlocks; ++h) {
                        const int last = last_lds[(b0 + h) * 16 + lane_row];
#pragma unroll
                        for (int t = 0; t < kTiles; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t at = lane_quarter * 4 + e;
                                if ((int)(base + t * 16 + at) > last || (k.missing[t / 4] >> (t % 4 * 16 + at) & 1))
                                    acc[h][t][e] = -INFINITY;
                            }
                    }
                }
#pragma unroll
                for (int h = 0; h < kBlocks; ++h) {
                    const uint32_t column = (b0 + h) * 16 + lane_row;
                    if constexpr (!kSum) {
                        const float2 old = state_lds[wave][column];
                        float top = acc[h][0][0];
#pragma unroll
                        for (int t = 0; t < kTiles; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[h][t][e]);
                        const float next = fmaxf(old.x, quarter_wave_max(top) * a.scale_log2);
                        float sum = 0.0f;
#pragma unroll
                        for (int t = 0; t < kTiles; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                sum += __builtin_amdgcn_exp2f(fmaf(acc[h][t][e], a.scale_log2, -next));
                        sum = fmaf(old.y, __builtin_amdgcn_exp2f(old.x - next), quarter_wave_sum(sum));
                        if (lane < 16) state_lds[wave][column] = make_float2(next, sum);
                    } else {
                        const float2 norm = norm_lds[column];
#pragma unroll
                        for (int t = 0; t < kTiles; ++t)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float& sum = sums[t / 4][t % 4 * 4 + e];
                                sum = fmaf(__builtin_amdgcn_exp2f(fmaf(acc[h][t][e], a.scale_log2, -norm.x)), norm.y, sum);
                            }
                    }
                }
            }
            if constexpr (kSum) {
                // lane_row's value of a word: of tile lane_row / 4, key lane_quarter * 4 + lane_row % 4 of it
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    const float sum = row_sums(sums[w], lane);
                    const uint32_t tile = lane_row / 4, at = tile * 16 + lane_quarter * 4 + lane_row % 4, p = base + w * 64 + at;
                    if (share) {
                        if (w * 4 + tile < kTiles) part_lds[wave * kKeys + w * 64 + at] = sum;
                    } else if (w * 4 + tile < kTiles && p < key_end && !(k.missing[w] >> at & 1)) {
                        add_weight(a, r, table, kv_head, p, sum, c0 == 0);
                    }
                }
            }
            if (turns > 1) {
                fetch_lines(base + step, k);
                if (turns > 2) fetch_ids(base + 2 * step);
            }
        }
        if constexpr (!kSum) {
            lds_barrier();
            for (uint32_t i = tid; i < count; i += kThreads) {
                float m = kEmptyMax, s = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) m = fmaxf(m, state_lds[w][i].x);
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const float2 part = state_lds[w][i];
                    s = fmaf(part.y, __builtin_amdgcn_exp2f(part.x - m), s);
                }
                a.stats[stat_index(a, row, kv_head, c0 + i)] = make_float2(m, s);
            }
        } else {
            if (share) {
                // wave part * key_groups + g has its columns' sums for the keys of group g
                lds_barrier();
                const uint32_t summed = (blocks + part_blocks - 1) / part_blocks;
                for (uint32_t i = tid; i < length; i += kThreads) {
                    float sum = 0.0f;
                    for (uint32_t q = 0; q < summed; ++q) sum += part_lds[q * key_groups * kKeys + i];
                    if (page_of(a.v, table, r.begin + i, a.v.num_pages) != kNoPage)
                        add_weight(a, r, table, kv_head, r.begin + i, sum, c0 == 0);
                }
            }
            // positions of the row that no column of the first columns sees still get their turn's base
            if (c0 == 0)
                for (uint32_t p = max(key_end, r.begin) + tid; p < r.end; p += kThreads)
                    if (page_of(a.v, table, p, a.v.num_pages) != kNoPage) add_weight(a, r, table, kv_head, p, 0.0f, true);
        }
    }
}

// kTiles, kBlocks, kWaves of either pass.  Three waves a SIMD of 160 registers each: with two (and half again the
// keys a turn) the batch of eight prompts, 32 tokens each, takes 36 + 31 us for 30 + 27, with four the lines spill.
template <int kTiles_, int kBlocks_, int kWaves_>
struct ObservePass {
    static constexpr int kTiles = kTiles_, kBlocks = kBlocks_, kWaves = kWaves_;
};
template <typename Tag, int D, int kMaxBlocks, typename Stats, typename Sum>
inline void launch_observe_blocks(psi_hip_ctx* ctx, const ObserveArgs& a, uint32_t window_rows) {
    const dim3 grid(a.num_rows * a.v.hkv);
    ObserveArgs fused = a;
    const uint64_t joins = (uint64_t)window_rows * a.max_window * a.group;
    if (joins <= kFusedJoins) fused.norm = nullptr;
    hipLaunchKernelGGL((observe_kernel<Tag, D, Stats::kTiles, Stats::kBlocks, kMaxBlocks, Stats::kWaves, false>), grid,
                       dim3(64 * Stats::kWaves), 0, ctx->stream, a);
    if (fused.norm != nullptr) launch_observe_join(ctx, a);
    hipLaunchKernelGGL((observe_kernel<Tag, D, Sum::kTiles, Sum::kBlocks, kMaxBlocks, Sum::kWaves, true>), grid,
                       dim3(64 * Sum::kWaves), 0, ctx->stream, fused);
}
template <typename Tag>
inline void launch_observe(psi_hip_ctx* ctx, const ObserveArgs& a, uint32_t window_rows) {
    // few columns: a fraction of the LDS, which launches faster (8 tokens over a prompt of 777: 13.3 for 14.2 us)
    const bool narrow = (uint64_t)a.max_window * a.group <= 64;
    if (a.v.d == 256) {
        using Pass = ObservePass<2, 2, 12>;
        if (narrow) launch_observe_blocks<Tag, 256, 4, Pass, Pass>(ctx, a, window_rows);
        else launch_observe_blocks<Tag, 256, 16, Pass, Pass>(ctx, a, window_rows);
    } else {
        // 64 keys a turn for the maxima (with streaming loads 68 us; 78 with 32), 32 for the weights, whose sums need
        // registers too (57; 58 with 48)
        using Stats = ObservePass<4, 1, 12>;
        using Sum = ObservePass<2, 2, 12>;
        if (narrow) launch_observe_blocks<Tag, 128, 4, Sum, Sum>(ctx, a, window_rows);
        else launch_observe_blocks<Tag, 128, 24, Stats, Sum>(ctx, a, window_rows);
    }
}

}  // namespace psi
