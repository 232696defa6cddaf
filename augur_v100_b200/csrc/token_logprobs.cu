// Log probabilities of given tokens, entropy and the best alternatives of rows of logits on sm_100a.
#include <cuda_bf16.h>

#include "nvfp4_internal.h"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_token_logprobs_args_v1) == 128, "log probabilities ABI");

struct LogprobsParams {
    const void* logits;
    const int32_t* targets;
    float *logprobs, *entropy, *alternative_logprobs;
    int32_t* ids;
    uint64_t row_stride;
    uint32_t rows, vocabulary, alternatives;
};

// A logit as an unsigned number of the same order: +0 and -0 alike, every NaN above all numbers.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t bits = __float_as_uint(x + 0.0f);   // -0 becomes +0
    if (x != x) return 0xffffffffu;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t key) {
    return __uint_as_float(key == 0xffffffffu ? 0x7fffffffu : key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ float value(const float* x) { return *x; }
__device__ __forceinline__ float value(const __nv_bfloat16* x) { return __bfloat162float(*x); }

constexpr uint32_t kThreads = 512;
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_simple_kernel(const LogprobsParams p) {
    __shared__ float shared[kThreads];
    __shared__ unsigned long long best;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    float top = -INFINITY;
    for (uint32_t i = threadIdx.x; i < p.vocabulary; i += kThreads) top = max_nan(top, value(x + i));
    shared[threadIdx.x] = top;
    for (uint32_t step = kThreads / 2; step; step /= 2) {
        __syncthreads();
        if (threadIdx.x < step) shared[threadIdx.x] = max_nan(shared[threadIdx.x], shared[threadIdx.x + step]);
    }
    __syncthreads();
    top = shared[0];
    const float base = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, moment = 0.0f;
    for (uint32_t i = threadIdx.x; i < p.vocabulary; i += kThreads) {
        const float below = max_nan(value(x + i) - base, -200.0f), weight = expf(below);
        total += weight, moment = fmaf(weight, below, moment);
    }
    for (uint32_t pass = 0; pass < 2; ++pass) {
        __syncthreads();
        shared[threadIdx.x] = pass ? moment : total;
        for (uint32_t step = kThreads / 2; step; step /= 2) {
            __syncthreads();
            if (threadIdx.x < step) shared[threadIdx.x] += shared[threadIdx.x + step];
        }
        __syncthreads();
        (pass ? moment : total) = shared[0];
    }
    const bool empty = top == -INFINITY;
    const float log_total = logf(total);
    if (threadIdx.x == 0) {
        const int32_t target = p.targets[row];
        const bool inside = target >= 0 && static_cast<uint32_t>(target) < p.vocabulary;
        p.logprobs[row] = !inside ? __uint_as_float(0x7fc00000u) : empty ? -INFINITY : value(x + target) - base - log_total;
        p.entropy[row] = empty ? 0.0f : log_total - moment / total;
    }
    unsigned long long last = ~0ull;
    for (uint32_t k = 0; k < p.alternatives; ++k) {
        __syncthreads();
        if (threadIdx.x == 0) best = 0;
        __syncthreads();
        unsigned long long mine = 0;
        for (uint32_t i = threadIdx.x; i < p.vocabulary; i += kThreads) {
            const unsigned long long key = static_cast<unsigned long long>(ordered(value(x + i))) << 32 | (0xffffffffu - i);
            if ((key < last || k == 0) && key > mine) mine = key;
        }
        atomicMax(&best, mine);
        __syncthreads();
        last = best;
        if (threadIdx.x == 0) {
            p.ids[static_cast<uint64_t>(row) * p.alternatives + k] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(last));
            p.alternative_logprobs[static_cast<uint64_t>(row) * p.alternatives + k] = empty ? -INFINITY : from_ordered(static_cast<uint32_t>(last >> 32)) - base - log_total;
        }
    }
}

bool check_logprobs(int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_token_logprobs_args_v1* a,
                    bool full, augur_cuda_result_v1* failure) {
    *failure = invalid();
    if (!header_ok(d, s, a)) {
        if (a && s && d >= 0 && s->ordinal == d && a->abi_version != AUGUR_CUDA_ABI_VERSION_V1) *failure = make_result(AUGUR_CUDA_STATUS_ABI_VERSION_MISMATCH);
        return false;
    }
    if (!plan_ok(plan, d, s) || !a->rows || a->rows > (1u << 20) || !a->vocabulary || a->vocabulary > (1u << 24)) return false;
    if (a->alternatives > AUGUR_NVFP4_SM100_MAX_ALTERNATIVES || a->alternatives > a->vocabulary || a->logits_type > AUGUR_NVFP4_SM100_LOGITS_BF16) return false;
    if (a->row_stride < a->vocabulary || a->row_stride > (UINT64_C(1) << 32)) return false;
    const uint64_t size = a->logits_type == AUGUR_NVFP4_SM100_LOGITS_F32 ? 4 : 2, rows = a->rows;
    if (a->logits_len_bytes != ((rows - 1) * a->row_stride + a->vocabulary) * size) return false;
    if (a->targets_len_bytes != rows * 4 || a->logprobs_len_bytes != rows * 4 || a->entropy_len_bytes != rows * 4) return false;
    if (a->ids_len_bytes != rows * a->alternatives * 4 || a->alternative_logprobs_len_bytes != rows * a->alternatives * 4) return false;
    uint64_t need = 0;
    if (augur_cuda_nvfp4_sm100_token_logprobs_scratch_extent_host_v1(a->rows, a->alternatives, plan->sm_count, &need).status != AUGUR_CUDA_STATUS_OK ||
        plan->scratch_bytes < need) return false;
    Range r[7] = {{a->logits, a->logits_len_bytes, size}, {a->targets, a->targets_len_bytes, 4}, {a->logprobs, a->logprobs_len_bytes, 4},
                  {a->entropy, a->entropy_len_bytes, 4}, plan_scratch_range(plan), {a->ids, a->ids_len_bytes, 4},
                  {a->alternative_logprobs, a->alternative_logprobs_len_bytes, 4}};
    const size_t count = a->alternatives ? 7 : 5;
    if (!a->alternatives && (a->ids || a->alternative_logprobs)) return false;
    if (!all_disjoint(r, count)) return false;
    return !full || (inspect_device_ranges(d, r, 4, failure) && inspect_device_ranges(d, r + 5, count - 5, failure));
}

}  // namespace
}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_token_logprobs_scratch_extent_host_v1(uint32_t rows, uint32_t alternatives,
                                                                                                           uint32_t sm_count, uint64_t* out_bytes) {
    if (!out_bytes || !rows || rows > (1u << 20) || alternatives > AUGUR_NVFP4_SM100_MAX_ALTERNATIVES || !sm_count || sm_count > 4096) return invalid();
    *out_bytes = kCounterBytes;
    return ok();
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_token_logprobs_preflight_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_token_logprobs_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_logprobs(d, s, plan, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_token_logprobs_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_token_logprobs_args_v1* a) {
    augur_cuda_result_v1 failure;
    if (!check_logprobs(d, s, plan, a, false, &failure)) return failure;
    if (consume_injected_fault()) return make_result(AUGUR_CUDA_STATUS_DIAGNOSTIC_FAULT_INJECTED);
    const cudaError_t e = cudaSetDevice(d);
    if (e != cudaSuccess) return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE, e);
    LogprobsParams p{};
    p.logits = reinterpret_cast<const void*>(a->logits);
    p.targets = reinterpret_cast<const int32_t*>(a->targets);
    p.logprobs = reinterpret_cast<float*>(a->logprobs);
    p.entropy = reinterpret_cast<float*>(a->entropy);
    p.ids = reinterpret_cast<int32_t*>(a->ids);
    p.alternative_logprobs = reinterpret_cast<float*>(a->alternative_logprobs);
    p.row_stride = a->row_stride, p.rows = a->rows, p.vocabulary = a->vocabulary, p.alternatives = a->alternatives;
    if (a->logits_type == AUGUR_NVFP4_SM100_LOGITS_F32) {
        launch_dependent(s->stream, logprobs_simple_kernel<float>, p.rows, kThreads, 0, p);
    } else {
        launch_dependent(s->stream, logprobs_simple_kernel<__nv_bfloat16>, p.rows, kThreads, 0, p);
    }
    count_launch();
    return submitted();
}
