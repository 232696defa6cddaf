// The paged key-value cache as its entries see it: checks of the descriptors and the lookup of a step's sequences.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "nvfp4_internal.h"

namespace augur_sm100 {

constexpr uint32_t kKvMinPageTokens = 16, kKvMaxPageTokens = 1024;

// Elements of a strided [rows][heads][head_dim] view from its first to its last; 0 where that does not fit 2^62.
inline uint64_t strided_elements(uint64_t rows, uint64_t heads, uint64_t head_dim, uint64_t row_stride, uint64_t head_stride) {
    if (row_stride >= (UINT64_C(1) << 40) || head_stride >= (UINT64_C(1) << 40) || rows > (1u << 20) || heads > (1u << 16)) return 0;
    return (rows - 1) * row_stride + (heads - 1) * head_stride + head_dim;
}

inline bool kv_layer_ok(const augur_cuda_nvfp4_sm100_kv_layer_v1& l) {
    if (!l.pages || !l.kv_heads || l.kv_heads > 1024 || (l.head_dim != 128 && l.head_dim != 256)) return false;
    if (l.page_tokens < kKvMinPageTokens || l.page_tokens > kKvMaxPageTokens || (l.page_tokens & (l.page_tokens - 1)) != 0) return false;
    const uint64_t rows = static_cast<uint64_t>(l.pages) * l.kv_heads * l.page_tokens;   // below 2^52
    return rows < (UINT64_C(1) << 31) && l.len_bytes == rows * l.head_dim * 2;
}

inline bool kv_layer_ok(const augur_cuda_nvfp4_sm100_kv_e4m3_layer_v1& l) {
    const uint64_t rows = static_cast<uint64_t>(l.pages) * l.kv_heads * l.page_tokens;
    return kv_layer_ok(augur_cuda_nvfp4_sm100_kv_layer_v1{l.keys, l.values, 2 * l.len_bytes, l.pages, l.kv_heads, l.page_tokens, l.head_dim}) &&
           l.len_bytes <= UINT64_MAX / 2 && l.scales_len_bytes == rows * 2;
}

// The tensors of a layer, for the checks of ranges: at most kKvRanges.
constexpr size_t kKvRanges = 3;
inline size_t kv_ranges(const augur_cuda_nvfp4_sm100_kv_layer_v1& l, Range* to) {
    to[0] = {l.keys, l.len_bytes, 16}, to[1] = {l.values, l.len_bytes, 16};
    return 2;
}
inline size_t kv_ranges(const augur_cuda_nvfp4_sm100_kv_e4m3_layer_v1& l, Range* to) {
    to[0] = {l.keys, l.len_bytes, 16}, to[1] = {l.values, l.len_bytes, 16}, to[2] = {l.scales, l.scales_len_bytes, 16};
    return 3;
}

// Scale bytes of the E4M3 cache: 2^(byte - 127).
constexpr uint32_t kE4m3LeastScale = 127 - 60, kE4m3LargestScale = 127 + 60;

inline bool kv_batch_ok(const augur_cuda_nvfp4_sm100_kv_batch_v1& b) {
    return b.sequences >= 1 && b.sequences <= AUGUR_NVFP4_SM100_MAX_SEQUENCES && b.table_pages >= 1 && b.table_pages <= (1u << 24) && b.rows >= 1 &&
           b.rows <= (1u << 20) && b.reserved == 0 && b.page_table_len_bytes == static_cast<uint64_t>(b.sequences) * b.table_pages * 4 &&
           b.lengths_len_bytes == static_cast<uint64_t>(b.sequences) * 4 && b.token_starts_len_bytes == static_cast<uint64_t>(b.sequences + 1) * 4;
}

}  // namespace augur_sm100
