// Dispatch of the gfx950 split-KV decode map (instantiated per element type and head_dim in the
// split_kv_decode_*.hip files) and the gfx950 log-sum-exp combine kernel.
#include "split_kv_reduce_kernel.h"

namespace psi {

int launch_decode_map_bf16_d256(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);
int launch_decode_map_bf16_d128(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);
int launch_decode_map_f16_d256(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);
int launch_decode_map_f16_d128(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);
// the variants that store the logits as well (MapArgs::logits)
int launch_decode_logits_bf16_d256(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);
int launch_decode_logits_bf16_d128(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);
int launch_decode_logits_f16_d256(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);
int launch_decode_logits_f16_d128(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a);

// One wave per (token, q_head), four to a workgroup.
template <typename Tag, int D, bool kIndexed>
__global__ __launch_bounds__(256) void split_kv_reduce_fast(ReduceArgs a) {
    resolve_active(a);
    const uint64_t row_out = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row_out >= (uint64_t)a.num_active_tokens * a.hq) return;
    reduce_row<Tag, D, kIndexed>(a, row_out);
}

// One workgroup per (token, q_head).
template <typename Tag, int D, bool kIndexed>
__global__ __launch_bounds__(64 * kWideWaves) void split_kv_reduce_wide(ReduceArgs a) {
    resolve_active(a);
    __shared__ WideReduceLds<D> lds;
    reduce_row_wide<Tag, D, kIndexed>(a, blockIdx.x, lds);
}

// The same combine for Q-token tiles: one wave per (tile, token in tile, q_head); the tile's partial
// rows are cu_kv_splits[tile] .. cu_kv_splits[tile + 1].
template <typename Tag, int D, bool kIndexed>
__global__ __launch_bounds__(256) void split_kv_reduce_tiled_fast(ReduceArgs a) {
    resolve_active(a);
    constexpr int kPerLane = D / 64;
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t id = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t rows = a.rows_per_split_head;
    const uint32_t q_head = (uint32_t)(id % a.hq);
    const uint32_t tile_row = (uint32_t)((id / a.hq) % rows);
    const uint64_t tile = id / ((uint64_t)a.hq * rows);
    if (tile >= a.num_active_q_token_tiles) return;
    const uint32_t flat_begin = a.q_token_tiles[tile * 2], flat_end = a.q_token_tiles[tile * 2 + 1];
    const uint32_t token = flat_begin + tile_row;
    if (token >= flat_end) return;
    const uint32_t begin = a.cu_kv_splits[tile], end = a.cu_kv_splits[tile + 1];
    constexpr int kUnroll = 4;
    const uint32_t* row_index = a.row_index;
    auto row_of = [&](uint32_t p) -> uint64_t {
        return ((uint64_t)(kIndexed ? row_index[p] : p) * a.hq + q_head) * rows + tile_row;
    };
    // (the first four rows ahead of the pass over the maxima, as in split_kv_reduce_fast)
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
    const uint64_t out_index = ((uint64_t)token * a.hq + q_head) * D + lane * kPerLane;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e)
        store_from_f32<Tag>(a.output, out_index + e, finish_output<Tag>(a, value[e] * inv, token, q_head, lane * kPerLane + e));
}

// Shapes and pointers for which the MFMA decode map runs, i.e. for which the append can be folded into it.
bool decode_map_takes_append(const psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a) {
    if (ctx->force_generic) return false;
    const bool two_byte = g.dtype == PSI_HIP_BF16 || g.dtype == PSI_HIP_F16;
    const uint32_t p = g.tokens_per_page;
    const bool page_ok = p >= 8 && (p & (p - 1)) == 0;
    auto aligned = [](const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 16 == 0; };
    return two_byte && page_ok && g.group <= 8 && (g.d == 256 || g.d == 128) && aligned(a.q) && aligned(a.kv_pages) &&
           aligned(a.flat_k) && aligned(a.flat_v) && (uint64_t)a.num_total_kv_splits * g.hkv <= 0x7fffffffull;
}

int launch_decode_map_fast(psi_hip_ctx* ctx, const Geometry& g, const MapArgs& a) {
    if (ctx->force_generic) return PSI_HIP_ERR_UNSUPPORTED;
    const bool two_byte = g.dtype == PSI_HIP_BF16 || g.dtype == PSI_HIP_F16;
    const uint32_t p = g.tokens_per_page;
    const bool page_ok = p >= 8 && (p & (p - 1)) == 0;
    const bool aligned = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && reinterpret_cast<uintptr_t>(a.kv_pages) % 16 == 0;
    if (!two_byte || !page_ok || !aligned || g.group > 8 || (g.d != 256 && g.d != 128)) return PSI_HIP_ERR_UNSUPPORTED;
    if ((uint64_t)a.num_total_kv_splits * g.hkv > 0x7fffffffull) return PSI_HIP_ERR_UNSUPPORTED;
    if (a.logits != nullptr) {
        if (g.dtype == PSI_HIP_BF16)
            return g.d == 256 ? launch_decode_logits_bf16_d256(ctx, g, a) : launch_decode_logits_bf16_d128(ctx, g, a);
        return g.d == 256 ? launch_decode_logits_f16_d256(ctx, g, a) : launch_decode_logits_f16_d128(ctx, g, a);
    }
    if (g.dtype == PSI_HIP_BF16)
        return g.d == 256 ? launch_decode_map_bf16_d256(ctx, g, a) : launch_decode_map_bf16_d128(ctx, g, a);
    return g.d == 256 ? launch_decode_map_f16_d256(ctx, g, a) : launch_decode_map_f16_d128(ctx, g, a);
}

int launch_reduce_fast(psi_hip_ctx* ctx, const Geometry& g, const ReduceArgs& a) {
    if (ctx->force_generic) return PSI_HIP_ERR_UNSUPPORTED;
    if (g.d != 256 && g.d != 128) return PSI_HIP_ERR_UNSUPPORTED;
    const bool tiled = a.q_token_tiles != nullptr;
    const uint64_t rows = tiled ? (uint64_t)a.num_active_q_token_tiles * a.rows_per_split_head * g.hq
                                : (uint64_t)a.num_active_tokens * g.hq;
    if ((rows + 3) / 4 > 0x7fffffffull) return PSI_HIP_ERR_UNSUPPORTED;
    const dim3 grid((uint32_t)((rows + 3) / 4)), block(256);
    const bool wide = !tiled && reduce_is_wide(a);
#define PSI_REDUCE_D(TAG, DIM, INDEXED)                                                                          \
    do {                                                                                                         \
        if (tiled) hipLaunchKernelGGL((split_kv_reduce_tiled_fast<TAG, DIM, INDEXED>), grid, block, 0, ctx->stream, a); \
        else if (wide) hipLaunchKernelGGL((split_kv_reduce_wide<TAG, DIM, INDEXED>), dim3((uint32_t)rows), dim3(64 * kWideWaves), 0, ctx->stream, a); \
        else hipLaunchKernelGGL((split_kv_reduce_fast<TAG, DIM, INDEXED>), grid, block, 0, ctx->stream, a);     \
    } while (0)
#define PSI_REDUCE(TAG)                                                   \
    do {                                                                  \
        if (g.d == 256) {                                                 \
            if (a.row_index) PSI_REDUCE_D(TAG, 256, true);                \
            else PSI_REDUCE_D(TAG, 256, false);                           \
        } else {                                                          \
            if (a.row_index) PSI_REDUCE_D(TAG, 128, true);                \
            else PSI_REDUCE_D(TAG, 128, false);                           \
        }                                                                 \
    } while (0)
    if (a.out_dtype == PSI_HIP_F32) PSI_REDUCE(F32Tag);
    else if (a.out_dtype == PSI_HIP_BF16) PSI_REDUCE(BF16Tag);
    else PSI_REDUCE(F16Tag);
#undef PSI_REDUCE_D
#undef PSI_REDUCE
    return PSI_HIP_OK;
}

}  // namespace psi
