// gfx950 observation kernels for 2-byte K and head_dim 128 or 256, any page size.
//
// One workgroup (8 waves) = one (row of keys, KV head).  The window's columns are staged in LDS in the operand order of
// the matrix product, up to 256 at a time; a wave takes 64 keys at a time straight from their pages into registers, in
// the operand order too (as in split_kv_decode_kernel.h: lane = token lane%16, 8-dim chunk lane/16, a 128-bit load per
// 32 dims), and multiplies them with one block of 16 columns after the other.  Waves share nothing but the columns, so
// there is no barrier in the loop over keys.  64 keys to a wave: a column operand read from LDS (8 cycles of the
// compute unit's LDS) then feeds four products (64 cycles of a SIMD), which the four SIMDs' reads just fill half of.
//
// A result lane holds 16 keys of one column, so the maximum and sum of a column (first pass) stay in the lane until the
// row's end, and the weights of a key (second pass) are summed over the columns of a lane first and over the lanes once
// per 64 keys.
#pragma once
#include "kv_observe.h"
#include "split_kv_decode_kernel.h"

namespace psi {

constexpr int kObserveWaves = 8, kObserveThreads = 64 * kObserveWaves;
constexpr int kObserveTiles = 4;                      // 16-key tiles of a wave's turn
constexpr uint32_t kObserveKeys = 16 * kObserveTiles;

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

// kSum false: the maxima and sums of the row's columns.  kSum true: the weights.
template <typename Tag, int D, int kMaxBlocks, bool kSum>
__global__ __launch_bounds__(kObserveThreads, 2) void observe_kernel(ObserveArgs a) {
    constexpr int kSteps = D / 32;
    constexpr uint32_t kColumns = 16 * kMaxBlocks, kChunks = D / 8;
    __shared__ __attribute__((aligned(16))) uint4 q_lds[kMaxBlocks * kSteps * 64];
    __shared__ int last_lds[kColumns];                        // last key that a column sees
    __shared__ float lse_lds[kSum ? kColumns : 1];
    __shared__ float2 merge_lds[kSum ? 1 : kObserveWaves][kSum ? 1 : kColumns];

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
        const uint32_t count = min(columns - c0, kColumns), blocks = (count + 15) / 16;
        const uint32_t key_end = min(r.end, r.position + (c0 + count - 1) / a.group + 1);  // what the last column sees
        if (c0 > 0) __syncthreads();
        for (uint32_t i = tid; i < blocks * 16 * kChunks; i += kObserveThreads) {
            const uint32_t column = i / kChunks, chunk = i % kChunks, c = c0 + column;
            uint4 value = make_uint4(0, 0, 0, 0);
            if (c < columns)
                value = *reinterpret_cast<const uint4*>(
                    q + ((uint64_t)(r.q_begin + c / a.group) * a.hq + kv_head * a.group + c % a.group) * D + chunk * 8);
            q_lds[((column / 16) * kSteps + chunk / 4) * 64 + (chunk % 4) * 16 + column % 16] = value;
        }
        for (uint32_t i = tid; i < blocks * 16; i += kObserveThreads) {
            const uint32_t c = c0 + i;
            last_lds[i] = c < columns ? (int)(r.position + c / a.group) : -1;
            if constexpr (kSum) lse_lds[i] = c < columns ? join_column(a, r, kv_head, c) : INFINITY;
        }
        __syncthreads();

        float col_max[kSum ? 1 : kMaxBlocks], col_sum[kSum ? 1 : kMaxBlocks];
        if constexpr (!kSum) {
#pragma unroll
            for (int b = 0; b < kMaxBlocks; ++b) {
                col_max[b] = kEmptyMax;
                col_sum[b] = 0.0f;
            }
        }
        // page IDs of the wave's next 64 keys, a turn ahead of their lines
        uint32_t page_id[kObserveTiles];
        auto fetch_ids = [&](uint32_t base) {
#pragma unroll
            for (int t = 0; t < kObserveTiles; ++t) {
                const uint32_t p = min(base + t * 16 + lane_row, key_end - 1);
                page_id[t] = page_of(a.v, table, p, a.v.num_pages);
            }
        };
        uint32_t base = r.begin + wave * kObserveKeys;
        if (base < key_end) fetch_ids(base);
        for (; base < key_end; base += kObserveWaves * kObserveKeys) {
            uint4 k[kObserveTiles][kSteps];
            bool bad = false;
#pragma unroll
            for (int t = 0; t < kObserveTiles; ++t) {
                const uint32_t p = min(base + t * 16 + lane_row, key_end - 1);
                const bool missing = page_id[t] == kNoPage;
                bad |= missing;
                const uint16_t* line = pages + line_index(a.v, missing ? 0 : page_id[t], 0, kv_head, page_place(a.v, p)) +
                                       lane_quarter * 8;
#pragma unroll
                for (int i = 0; i < kSteps; ++i) k[t][i] = stream_load_b128(line + i * 32);
            }
            // keys on pages beyond the arena: bit t * 16 + row, the same for the four quarters
            uint64_t missing_keys = 0;
            if (__any(bad)) {
                report_cache_range(a.status);
#pragma unroll
                for (int t = 0; t < kObserveTiles; ++t)
                    missing_keys |= (__ballot(page_id[t] == kNoPage) & 0xffffull) << (16 * t);
            }
            if (base + kObserveWaves * kObserveKeys < key_end) fetch_ids(base + kObserveWaves * kObserveKeys);
            const bool masked = base + kObserveKeys > r.position + 1 || missing_keys != 0;

            auto logits_of = [&](uint32_t block, f32x4_t (&acc)[kObserveTiles]) __attribute__((always_inline)) {
#pragma unroll
                for (int t = 0; t < kObserveTiles; ++t) acc[t] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < kSteps; ++i) {
                    const uint4 qv = q_lds[(block * kSteps + i) * 64 + lane];
#pragma unroll
                    for (int t = 0; t < kObserveTiles; ++t) acc[t] = mfma_16x16x32<Tag>(k[t][i], qv, acc[t]);
                }
                if (masked) {
                    const int last = last_lds[block * 16 + lane_row];
#pragma unroll
                    for (int t = 0; t < kObserveTiles; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t at = t * 16 + lane_quarter * 4 + e;
                            if ((int)(base + at) > last || (missing_keys >> at & 1)) acc[t][e] = -INFINITY;
                        }
                }
            };
            if constexpr (!kSum) {
#pragma unroll
                for (int b = 0; b < kMaxBlocks; ++b) {
                    if (b >= (int)blocks) continue;
                    f32x4_t acc[kObserveTiles];
                    logits_of(b, acc);
                    float top = acc[0][0];
#pragma unroll
                    for (int t = 0; t < kObserveTiles; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[t][e]);
                    const float next = fmaxf(col_max[b], top * a.scale_log2);
                    float sum = 0.0f;
#pragma unroll
                    for (int t = 0; t < kObserveTiles; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sum += __builtin_amdgcn_exp2f(fmaf(acc[t][e], a.scale_log2, -next));
                    col_sum[b] = fmaf(col_sum[b], __builtin_amdgcn_exp2f(col_max[b] - next), sum);
                    col_max[b] = next;
                }
            } else {
                float sums[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) sums[i] = 0.0f;
                for (uint32_t b = 0; b < blocks; ++b) {
                    f32x4_t acc[kObserveTiles];
                    logits_of(b, acc);
                    const float lse = lse_lds[b * 16 + lane_row];
#pragma unroll
                    for (int t = 0; t < kObserveTiles; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            sums[t * 4 + e] += __builtin_amdgcn_exp2f(fmaf(acc[t][e], a.scale_log2, -lse));
                }
                const float sum = row_sums(sums, lane);  // of tile lane_row / 4, token lane_quarter * 4 + lane_row % 4
                const uint32_t at = lane_row / 4 * 16 + lane_quarter * 4 + lane_row % 4, p = base + at;
                if (p < key_end && !(missing_keys >> at & 1)) add_weight(a, r, table, kv_head, p, sum, c0 == 0);
            }
        }
        if constexpr (!kSum) {
#pragma unroll
            for (int b = 0; b < kMaxBlocks; ++b) {
                if (b >= (int)blocks) continue;
                const float m = quarter_wave_max(col_max[b]);
                const float s = quarter_wave_sum(col_sum[b] * __builtin_amdgcn_exp2f(col_max[b] - m));
                if (lane < 16) merge_lds[wave][b * 16 + lane] = make_float2(m, s);
            }
            __syncthreads();
            for (uint32_t i = tid; i < count; i += kObserveThreads) {
                float m = kEmptyMax, s = 0.0f;
#pragma unroll
                for (int w = 0; w < kObserveWaves; ++w) m = fmaxf(m, merge_lds[w][i].x);
#pragma unroll
                for (int w = 0; w < kObserveWaves; ++w)
                    s = fmaf(merge_lds[w][i].y, __builtin_amdgcn_exp2f(merge_lds[w][i].x - m), s);
                a.stats[stat_index(a, row, kv_head, c0 + i)] = make_float2(m, s);
            }
        } else {
            // positions of the row that no column of the first columns sees still get their turn's base
            if (c0 == 0)
                for (uint32_t p = max(key_end, r.begin) + tid; p < r.end; p += kObserveThreads)
                    if (page_of(a.v, table, p, a.v.num_pages) != kNoPage) add_weight(a, r, table, kv_head, p, 0.0f, true);
        }
    }
}

template <typename Tag, int D, int kMaxBlocks>
inline void launch_observe_blocks(psi_hip_ctx* ctx, const ObserveArgs& a) {
    const dim3 grid(a.num_rows * a.v.hkv), threads(kObserveThreads);
    hipLaunchKernelGGL((observe_kernel<Tag, D, kMaxBlocks, false>), grid, threads, 0, ctx->stream, a);
    hipLaunchKernelGGL((observe_kernel<Tag, D, kMaxBlocks, true>), grid, threads, 0, ctx->stream, a);
}
template <typename Tag>
inline void launch_observe(psi_hip_ctx* ctx, const ObserveArgs& a) {
    const bool narrow = (uint64_t)a.max_window * a.group <= 64;
    if (a.v.d == 256) {
        if (narrow) launch_observe_blocks<Tag, 256, 4>(ctx, a);
        else launch_observe_blocks<Tag, 256, 16>(ctx, a);
    } else {
        if (narrow) launch_observe_blocks<Tag, 128, 4>(ctx, a);
        else launch_observe_blocks<Tag, 128, 16>(ctx, a);
    }
}

}  // namespace psi
