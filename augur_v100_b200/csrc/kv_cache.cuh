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

inline bool kv_batch_ok(const augur_cuda_nvfp4_sm100_kv_batch_v1& b) {
    return b.sequences >= 1 && b.sequences <= AUGUR_NVFP4_SM100_MAX_SEQUENCES && b.table_pages >= 1 && b.table_pages <= (1u << 24) && b.rows >= 1 &&
           b.rows <= (1u << 20) && b.reserved == 0 && b.page_table_len_bytes == static_cast<uint64_t>(b.sequences) * b.table_pages * 4 &&
           b.lengths_len_bytes == static_cast<uint64_t>(b.sequences) * 4 && b.token_starts_len_bytes == static_cast<uint64_t>(b.sequences + 1) * 4;
}

}  // namespace augur_sm100
