// The log-sum-exp combine of decode rows, as device functions: the combine kernels (split_kv_decode_fast.hip) and the
// launch that accumulates weights next to it (kv_weights.hip) run the same code.
#pragma once
#include "split_kv.h"

namespace psi {

// Log-sum-exp combine: one wave per (token, q_head), lanes over head_dim.  The accumulator rows are
// read four at a time so that a wave keeps several 1 KiB reads in flight instead of one; the overall
// maximum comes from the first four rows' own values and a lane-parallel pass over the rest.
template <typename Tag, int D, bool kIndexed>
__device__ __forceinline__ void reduce_row(const ReduceArgs& a, uint64_t row_out) {
    constexpr int kPerLane = D / 64;  // 4 or 2
    constexpr int kUnroll = 4;
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t token = (uint32_t)(row_out / a.hq), q_head = (uint32_t)(row_out % a.hq);
    const uint32_t begin = a.cu_kv_splits[token], end = a.cu_kv_splits[token + 1];
    const uint32_t* row_index = a.row_index;
    auto row_of = [&](uint32_t p) -> uint64_t { return (uint64_t)(kIndexed ? row_index[p] : p) * a.hq + q_head; };
    // The first four rows are asked for before anything waits: their maxima (the same in every lane) enter the
    // overall maximum from registers, and the lane-parallel pass over the maxima covers the rows behind them only,
    // so that a short list - the usual case - costs one round trip to memory instead of two.
    float m[kUnroll], sums[kUnroll], part[kUnroll][kPerLane];
    auto fetch = [&](uint32_t p0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const bool live = p0 + u < end;
            const uint64_t row = row_of(live ? p0 + u : begin);
            m[u] = a.part_max[row];
            if (!live) m[u] = -INFINITY;
            sums[u] = a.part_sum[row];
            const float* src = a.part_acc + row * D + lane * kPerLane;
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) part[u][e] = src[e];
        }
    };
    if (begin < end) fetch(begin);
    float global_max = -INFINITY;
    for (uint32_t p = begin + kUnroll + lane; p < end; p += 64) global_max = fmaxf(global_max, a.part_max[row_of(p)]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) global_max = fmaxf(global_max, __shfl_xor(global_max, off, 64));
    if (begin < end) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) global_max = fmaxf(global_max, m[u]);
    }
    float weight_sum = 0.0f, value[kPerLane];
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) value[e] = 0.0f;
    for (uint32_t p0 = begin; p0 < end; p0 += kUnroll) {
        if (p0 != begin) fetch(p0);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const float w = m[u] > -INFINITY ? exp2f(m[u] - global_max) : 0.0f;
            weight_sum = fmaf(w, sums[u], weight_sum);
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) value[e] = fmaf(w, part[u][e], value[e]);
        }
    }
    const float inv = weight_sum > 0.0f ? 1.0f / weight_sum : 0.0f;
    const uint64_t out_index = row_out * D + lane * kPerLane;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e)
        store_from_f32<Tag>(a.output, out_index + e, finish_output<Tag>(a, value[e] * inv, token, q_head, lane * kPerLane + e));
}

// The combine for long split lists (long contexts, few tokens): one workgroup of eight waves per
// (token, q_head); wave w takes the rows begin + w, begin + w + 8, ... four at a time, and the wave
// results, all relative to the same maximum, are added through LDS.
constexpr int kWideWaves = 8;
template <int D>
struct WideReduceLds {
    float max[kWideWaves];
    float sum[kWideWaves];
    float val[kWideWaves][D];
};
template <typename Tag, int D, bool kIndexed>
__device__ __forceinline__ void reduce_row_wide(const ReduceArgs& a, uint64_t row_out, WideReduceLds<D>& lds) {
    constexpr int kPerLane = D / 64;
    constexpr int kUnroll = 4;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t token = (uint32_t)(row_out / a.hq), q_head = (uint32_t)(row_out % a.hq);
    // The grid is cut for the by-value count; with device-side counts bound that is the bucket's capacity, and a
    // workgroup beyond the active tokens must touch nothing (its cu_kv_splits entries are stale).  Uniform over
    // the workgroup and ahead of the first barrier.
    if (token >= a.num_active_tokens) return;
    const uint32_t begin = a.cu_kv_splits[token], end = a.cu_kv_splits[token + 1];
    const uint32_t* row_index = a.row_index;
    float global_max = -INFINITY;
    for (uint32_t p = begin + threadIdx.x; p < end; p += 64 * kWideWaves)
        global_max = fmaxf(global_max, a.part_max[(uint64_t)(kIndexed ? row_index[p] : p) * a.hq + q_head]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) global_max = fmaxf(global_max, __shfl_xor(global_max, off, 64));
    if (lane == 0) lds.max[wave] = global_max;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWideWaves; ++w) global_max = fmaxf(global_max, lds.max[w]);
    float weight_sum = 0.0f, value[kPerLane];
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) value[e] = 0.0f;
    for (uint32_t p0 = begin + wave; p0 < end; p0 += kWideWaves * kUnroll) {
        float w[kUnroll], sums[kUnroll], part[kUnroll][kPerLane];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const bool live = p0 + u * kWideWaves < end;
            const uint32_t p = live ? p0 + u * kWideWaves : begin;
            const uint64_t row = (uint64_t)(kIndexed ? row_index[p] : p) * a.hq + q_head;
            const float m = a.part_max[row];
            sums[u] = a.part_sum[row];
            w[u] = live && m > -INFINITY ? exp2f(m - global_max) : 0.0f;
            const float* src = a.part_acc + row * D + lane * kPerLane;
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) part[u][e] = src[e];
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            weight_sum = fmaf(w[u], sums[u], weight_sum);
#pragma unroll
            for (int e = 0; e < kPerLane; ++e) value[e] = fmaf(w[u], part[u][e], value[e]);
        }
    }
    if (lane == 0) lds.sum[wave] = weight_sum;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) lds.val[wave][lane * kPerLane + e] = value[e];
    __syncthreads();
    if (wave != 0) return;
    weight_sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) value[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWideWaves; ++w) {
        weight_sum += lds.sum[w];
#pragma unroll
        for (int e = 0; e < kPerLane; ++e) value[e] += lds.val[w][lane * kPerLane + e];
    }
    const float inv = weight_sum > 0.0f ? 1.0f / weight_sum : 0.0f;
    const uint64_t out_index = row_out * D + lane * kPerLane;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e)
        store_from_f32<Tag>(a.output, out_index + e, finish_output<Tag>(a, value[e] * inv, token, q_head, lane * kPerLane + e));
}

}  // namespace psi
