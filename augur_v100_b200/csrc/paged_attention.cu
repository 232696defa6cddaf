// Attention of a step's new tokens over a paged key-value cache on sm_100a.
#include "kv_cache.cuh"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_paged_attention_args_v1) == 160, "attention ABI");

constexpr uint32_t kMaxQueries = 64;   // new tokens x query heads of a key-value head
constexpr uint32_t kStatusPage = 0x401, kStatusRows = 0x402;

struct AttentionParams {
    const __nv_bfloat16 *query, *keys, *values;
    __nv_bfloat16* output;
    const int32_t *page_table, *lengths, *token_starts;
    uint32_t* status_word;
    uint32_t rows, sequences, table_pages, pages, query_heads, kv_heads, page_shift, max_new;
    float scale_log2;   // scale * log2(e)
};

// One CTA per token row and query head, a warp per key, online softmax in registers.
template <uint32_t kHeadDim>
__global__ void __launch_bounds__(256) attention_simple_kernel(const AttentionParams p) {
    constexpr uint32_t kPer = kHeadDim / 32, kWarps = 8;
    __shared__ float part[kWarps][kHeadDim], tops[kWarps], sums[kWarps];
    __shared__ int32_t sequence_at;
    const uint32_t row = blockIdx.x / p.query_heads, head = blockIdx.x % p.query_heads, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) sequence_at = -1;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < p.sequences; b += 256) {
        const int32_t from = p.token_starts[b], to = p.token_starts[b + 1];
        if (from < 0 || to > static_cast<int32_t>(p.rows) || to - from > static_cast<int32_t>(p.max_new)) atomicCAS(p.status_word, 0u, kStatusRows);
        else if (static_cast<int32_t>(row) >= from && static_cast<int32_t>(row) < to) sequence_at = static_cast<int32_t>(b);
    }
    __syncthreads();
    if (sequence_at < 0) return;
    const uint32_t b = static_cast<uint32_t>(sequence_at), kv_head = head / (p.query_heads / p.kv_heads);
    const int64_t length = p.lengths[b], room = static_cast<int64_t>(p.table_pages) << p.page_shift;
    if (length > room) atomicCAS(p.status_word, 0u, kStatusPage);
    int64_t keys = length - p.token_starts[b + 1] + row + 1;
    if (keys > room) keys = room;
    float q[kPer], sum[kPer], top = -INFINITY, total = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) {
        q[i] = __bfloat162float(p.query[(static_cast<uint64_t>(row) * p.query_heads + head) * kHeadDim + i * 32 + lane]);
        sum[i] = 0.0f;
    }
    for (int64_t j = warp; j < keys; j += kWarps) {
        const int32_t page = p.page_table[static_cast<uint64_t>(b) * p.table_pages + (j >> p.page_shift)];
        if (page < 0 || static_cast<uint32_t>(page) >= p.pages) {
            if (lane == 0) atomicCAS(p.status_word, 0u, kStatusPage);
            continue;
        }
        const uint64_t at = (((static_cast<uint64_t>(page) * p.kv_heads + kv_head) << p.page_shift) + (j & ((1 << p.page_shift) - 1))) * kHeadDim + lane;
        float dot = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) dot = fmaf(q[i], __bfloat162float(p.keys[at + i * 32]), dot);
#pragma unroll
        for (uint32_t step = 16; step; step /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, step);
        const float score = dot * p.scale_log2, above = fmaxf(top, score);
        if (above == -INFINITY) continue;
        const float keep = exp2f(top - above), weight = exp2f(score - above);
        top = above;
        total = total * keep + weight;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) sum[i] = sum[i] * keep + weight * __bfloat162float(p.values[at + i * 32]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kPer; ++i) part[warp][i * 32 + lane] = sum[i];
    if (lane == 0) tops[warp] = top, sums[warp] = total;
    __syncthreads();
    float above = -INFINITY, all = 0.0f;
    for (uint32_t w = 0; w < kWarps; ++w) above = fmaxf(above, tops[w]);
    for (uint32_t w = 0; w < kWarps; ++w) all += tops[w] == -INFINITY ? 0.0f : sums[w] * exp2f(tops[w] - above);
    for (uint32_t d = threadIdx.x; d < kHeadDim; d += 256) {
        float value = 0.0f;
        for (uint32_t w = 0; w < kWarps; ++w) value += tops[w] == -INFINITY ? 0.0f : part[w][d] * exp2f(tops[w] - above);
        p.output[(static_cast<uint64_t>(row) * p.query_heads + head) * kHeadDim + d] = __float2bfloat16_rn(above == -INFINITY ? 0.0f : value / all);
    }
}

bool shape_ok(uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_new) {
    return kv_heads && kv_heads <= 1024 && query_heads && query_heads <= 1024 && query_heads % kv_heads == 0 && (head_dim == 128 || head_dim == 256) &&
           max_new >= 1 && max_new <= AUGUR_NVFP4_SM100_MAX_SMALL_TOKENS && query_heads / kv_heads * max_new <= kMaxQueries;
}

bool check_attention(int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_paged_attention_args_v1* a,
                     bool full, augur_cuda_result_v1* failure) {
    *failure = invalid();
    if (!header_ok(d, s, a)) {
        if (a && s && d >= 0 && s->ordinal == d && a->abi_version != AUGUR_CUDA_ABI_VERSION_V1) *failure = make_result(AUGUR_CUDA_STATUS_ABI_VERSION_MISMATCH);
        return false;
    }
    if (!plan_ok(plan, d, s) || !kv_layer_ok(a->layer) || !kv_batch_ok(a->batch) || a->reserved != 0) return false;
    if (!shape_ok(a->query_heads, a->layer.kv_heads, a->layer.head_dim, a->max_new_tokens) || !std::isfinite(a->scale)) return false;
    const uint64_t bytes = static_cast<uint64_t>(a->batch.rows) * a->query_heads * a->layer.head_dim * 2;
    if (a->query_len_bytes != bytes || a->output_len_bytes != bytes) return false;
    uint64_t need = 0;
    if (augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(a->query_heads, a->layer.kv_heads, a->layer.head_dim, a->max_new_tokens, plan->sm_count,
                                                                      &need).status != AUGUR_CUDA_STATUS_OK || plan->scratch_bytes < need) return false;
    const Range r[8] = {{a->query, a->query_len_bytes, 16}, {a->output, a->output_len_bytes, 16}, {a->layer.keys, a->layer.len_bytes, 16},
                        {a->layer.values, a->layer.len_bytes, 16}, {a->batch.page_table, a->batch.page_table_len_bytes, 4},
                        {a->batch.lengths, a->batch.lengths_len_bytes, 4}, {a->batch.token_starts, a->batch.token_starts_len_bytes, 4}, plan_scratch_range(plan)};
    if (!all_disjoint(r, 8)) return false;
    return !full || inspect_device_ranges(d, r, 7, failure);
}

}  // namespace
}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(
    uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_new_tokens, uint32_t sm_count, uint64_t* out_bytes) {
    if (!out_bytes || !shape_ok(query_heads, kv_heads, head_dim, max_new_tokens) || !sm_count || sm_count > 4096) return invalid();
    *out_bytes = kCounterBytes;
    return ok();
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_paged_attention_preflight_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_paged_attention_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_attention(d, s, plan, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_paged_attention_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_paged_attention_args_v1* a) {
    augur_cuda_result_v1 failure;
    if (!check_attention(d, s, plan, a, false, &failure)) return failure;
    if (consume_injected_fault()) return make_result(AUGUR_CUDA_STATUS_DIAGNOSTIC_FAULT_INJECTED);
    const cudaError_t e = cudaSetDevice(d);
    if (e != cudaSuccess) return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE, e);
    AttentionParams p{};
    p.query = reinterpret_cast<const __nv_bfloat16*>(a->query);
    p.keys = reinterpret_cast<const __nv_bfloat16*>(a->layer.keys);
    p.values = reinterpret_cast<const __nv_bfloat16*>(a->layer.values);
    p.output = reinterpret_cast<__nv_bfloat16*>(a->output);
    p.page_table = reinterpret_cast<const int32_t*>(a->batch.page_table);
    p.lengths = reinterpret_cast<const int32_t*>(a->batch.lengths);
    p.token_starts = reinterpret_cast<const int32_t*>(a->batch.token_starts);
    p.status_word = plan->status_word;
    p.rows = a->batch.rows, p.sequences = a->batch.sequences, p.table_pages = a->batch.table_pages, p.pages = a->layer.pages;
    p.query_heads = a->query_heads, p.kv_heads = a->layer.kv_heads, p.page_shift = static_cast<uint32_t>(__builtin_ctz(a->layer.page_tokens));
    p.max_new = a->max_new_tokens;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    if (a->layer.head_dim == 256) {
        launch_dependent(s->stream, attention_simple_kernel<256>, p.rows * p.query_heads, 256, 0, p);
    } else {
        launch_dependent(s->stream, attention_simple_kernel<128>, p.rows * p.query_heads, 256, 0, p);
    }
    count_launch();
    return submitted();
}
