// Attention of a step's 1..8 new tokens per sequence over a paged cache of E4M3 codes on sm_100a.
#include "attention_simple.cuh"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_paged_attention_e4m3_args_v1) == 176, "attention ABI");

}  // namespace
}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_paged_attention_e4m3_preflight_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_paged_attention_e4m3_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_attention(d, s, plan, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_paged_attention_e4m3_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_paged_attention_e4m3_args_v1* a) {
    augur_cuda_result_v1 failure;
    if (!check_attention(d, s, plan, a, false, &failure)) return failure;
    if (consume_injected_fault()) return make_result(AUGUR_CUDA_STATUS_DIAGNOSTIC_FAULT_INJECTED);
    const cudaError_t e = cudaSetDevice(d);
    if (e != cudaSuccess) return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE, e);
    AttentionParams p = attention_params(plan, a);
    p.scales = reinterpret_cast<const uint8_t*>(a->layer.scales);
    auto kernel = a->layer.head_dim == 256 ? attention_simple_kernel<256, true> : attention_simple_kernel<128, true>;
    kernel<<<dim3(p.rows, p.query_heads), 128, 0, s->stream>>>(reinterpret_cast<const void*>(a->layer.keys), reinterpret_cast<const void*>(a->layer.values), nullptr, p);
    count_launch();
    return submitted();
}
