// Attention of a step's new tokens over a paged cache whose sequences share a prefix, on sm_100a.
#include "attention_simple.cuh"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_shared_prefix_attention_args_v1) == 192, "attention ABI");

bool check_shared(int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_shared_prefix_attention_args_v1* a,
                  bool full, augur_cuda_result_v1* failure) {
    Range ranges[kAttentionRanges + 2];
    size_t count;
    if (!attention_args_ok(d, s, plan, a, ranges, &count, failure)) return false;
    const uint64_t pages = a->prefix_pages_len_bytes / 4;
    if (!pages || a->prefix_pages_len_bytes % 4 != 0 || pages * a->layer.page_tokens > (1u << kMaxTokensLog2) || pages > (1u << kMaxTokensLog2) || a->prefix_tokens_len_bytes != 4) return false;
    ranges[count] = ranges[count - 1];   // the scratch stays the last
    ranges[count - 1] = {a->prefix_pages, a->prefix_pages_len_bytes, 4};
    ranges[count + 1] = ranges[count], ranges[count] = {a->prefix_tokens, 4, 4};
    count += 2;
    if (!all_disjoint(ranges, count)) return false;
    uint64_t need = 0;
    if (augur_cuda_nvfp4_sm100_shared_prefix_attention_scratch_extent_host_v1(a->query_heads, a->layer.kv_heads, a->layer.head_dim, a->batch.rows, a->max_new_tokens,
                                                                              plan->sm_count, &need).status != AUGUR_CUDA_STATUS_OK || plan->scratch_bytes < need) return false;
    return !full || inspect_device_ranges(d, ranges, count - 1, failure);
}

}  // namespace
}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_shared_prefix_attention_scratch_extent_host_v1(
    uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t rows, uint32_t max_new_tokens, uint32_t sm_count, uint64_t* out_bytes) {
    if (!out_bytes || !shape_ok(query_heads, kv_heads, head_dim, max_new_tokens) || !sm_count || sm_count > 4096 || !rows || rows > (1u << 20)) return invalid();
    return augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(query_heads, kv_heads, head_dim, max_new_tokens, sm_count, out_bytes);
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_shared_prefix_attention_preflight_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_shared_prefix_attention_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_shared(d, s, plan, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_shared_prefix_attention_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_shared_prefix_attention_args_v1* a) {
    augur_cuda_result_v1 failure;
    if (!check_shared(d, s, plan, a, false, &failure)) return failure;
    if (consume_injected_fault()) return make_result(AUGUR_CUDA_STATUS_DIAGNOSTIC_FAULT_INJECTED);
    const cudaError_t e = cudaSetDevice(d);
    if (e != cudaSuccess) return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE, e);
    AttentionParams p = attention_params(plan, a);
    p.prefix_tokens = reinterpret_cast<const int32_t*>(a->prefix_tokens);
    p.prefix_pages = static_cast<uint32_t>(a->prefix_pages_len_bytes / 4);
    auto kernel = a->layer.head_dim == 256 ? attention_simple_kernel<256, false> : attention_simple_kernel<128, false>;
    kernel<<<dim3(p.rows, p.query_heads), 128, 0, s->stream>>>(reinterpret_cast<const void*>(a->layer.keys), reinterpret_cast<const void*>(a->layer.values),
                                                             reinterpret_cast<const int32_t*>(a->prefix_pages), p);
    count_launch();
    return submitted();
}
