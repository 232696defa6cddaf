// Attention over a paged cache in its simplest form: a CTA for a token row and query head, its warps taking the keys in turn.
#pragma once

#include "paged_attention.cuh"

namespace augur_sm100 {
namespace {

template <uint32_t kHeadDim, bool kE4m3>
__global__ void __launch_bounds__(128) attention_simple_kernel(const void* keys, const void* values, const int32_t* prefix_table, const __grid_constant__ AttentionParams p) {
    constexpr uint32_t kEach = kHeadDim / 32;
    __shared__ float best[4], total[4], sums[4][kHeadDim];
    const uint32_t row = blockIdx.x, head = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32, kv_head = head / (p.query_heads / p.kv_heads);
    int32_t sequence = -1;
    for (uint32_t b = 0; b < p.sequences; ++b) {
        const int32_t from = p.token_starts[b], to = p.token_starts[b + 1];
        if (from < 0 || to > static_cast<int32_t>(p.rows) || to < from || to - from > static_cast<int32_t>(p.max_new)) {
            if (threadIdx.x == 0) atomicCAS(p.status_word, 0u, kStatusRows);
        } else if (from <= static_cast<int32_t>(row) && static_cast<int32_t>(row) < to) {
            sequence = static_cast<int32_t>(b);
        }
    }
    if (sequence < 0) return;
    const uint32_t shared = prefix_table ? shared_tokens(p.prefix_tokens, p.prefix_pages, p.page_shift) : 0;
    if (prefix_table && threadIdx.x == 0 && *p.prefix_tokens > static_cast<int32_t>(p.prefix_pages << p.page_shift)) atomicCAS(p.status_word, 0u, kStatusPage);
    int32_t length = p.lengths[sequence];
    if (length > static_cast<int32_t>(p.table_pages << p.page_shift)) {
        length = static_cast<int32_t>(p.table_pages << p.page_shift);
        if (threadIdx.x == 0) atomicCAS(p.status_word, 0u, kStatusPage);
    }
    const int32_t limit = length - p.token_starts[sequence + 1] + static_cast<int32_t>(row) + 1;
    float q[kEach], o[kEach] = {}, m = -INFINITY, l = 0.0f;
    for (uint32_t i = 0; i < kEach; ++i) q[i] = __bfloat162float(p.query[(static_cast<uint64_t>(row) * p.query_heads + head) * kHeadDim + i * 32 + lane]);
    for (int32_t key = static_cast<int32_t>(warp); key < limit; key += 4) {
        const uint32_t index = static_cast<uint32_t>(key) >> p.page_shift;
        const int32_t page = key < static_cast<int32_t>(shared) ? prefix_table[index] : p.page_table[static_cast<uint64_t>(sequence) * p.table_pages + index];
        if (page < 0 || static_cast<uint32_t>(page) >= p.pages) {
            if (lane == 0) atomicCAS(p.status_word, 0u, kStatusPage);
            continue;
        }
        const uint64_t slot = ((static_cast<uint64_t>(page) * p.kv_heads + kv_head) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
        float scale_k = 1.0f, scale_v = 1.0f;
        if (kE4m3) {
            auto scale = [&](uint32_t byte) { return byte == 255 ? NAN : __uint_as_float((byte < kE4m3LeastScale ? kE4m3LeastScale : byte > kE4m3LargestScale ? kE4m3LargestScale : byte) << 23); };
            scale_k = scale(p.scales[2 * slot]), scale_v = scale(p.scales[2 * slot + 1]);
        }
        auto element = [&](const void* from, uint32_t i) -> float {
            const uint64_t at = slot * kHeadDim + i * 32 + lane;
            if (!kE4m3) return __bfloat162float(static_cast<const __nv_bfloat16*>(from)[at]);
            uint32_t halves;
            asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(static_cast<uint16_t>(static_cast<const uint8_t*>(from)[at])));
            float x;
            asm("{.reg .b16 low, high; mov.b32 {low, high}, %1; cvt.f32.f16 %0, low;}" : "=f"(x) : "r"(halves));
            return x;
        };
        float s = 0.0f;
        for (uint32_t i = 0; i < kEach; ++i) s = fmaf(q[i], element(keys, i), s);
        for (uint32_t step = 16; step; step /= 2) s += __shfl_xor_sync(0xffffffffu, s, step);
        s *= scale_k * p.scale_log2;
        const float now = fmaxf(m, s), factor = m == -INFINITY ? 0.0f : exp2f(m - now), w = exp2f(s - (now == -INFINITY ? 0.0f : now));
        l = l * factor + w, m = now;
        for (uint32_t i = 0; i < kEach; ++i) o[i] = o[i] * factor + w * (element(values, i) * scale_v);
    }
    if (lane == 0) best[warp] = m, total[warp] = l;
    for (uint32_t i = 0; i < kEach; ++i) sums[warp][i * 32 + lane] = o[i];
    __syncthreads();
    const float top = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
    for (uint32_t d = threadIdx.x; d < kHeadDim; d += 128) {
        float sum = 0.0f, all = 0.0f;
        for (uint32_t w = 0; w < 4; ++w) {
            if (best[w] == -INFINITY && total[w] == 0.0f) continue;
            const float f = exp2f(best[w] - top);
            sum += f * sums[w][d], all += f * total[w];
        }
        p.output[(static_cast<uint64_t>(row) * p.query_heads + head) * kHeadDim + d] = __float2bfloat16_rn(all == 0.0f ? 0.0f : sum / all);
    }
}

}  // namespace
}  // namespace augur_sm100
