// Log probabilities of given tokens, entropy and the best alternatives of rows of logits on sm_100a.
//
//   logprob(t) = x_t - m - ln L,  entropy = ln L - W / L,  L = sum e^(x - m),  W = sum e^(x - m) (x - m)
//
// One pass over the logits, which is the bound (4 or 2 bytes an element against about eight instructions): every thread keeps a running maximum m,
// L and W of its own elements; they are brought to one m where threads, CTAs and rows meet, always in the same order.
//
// The alternatives ride along. An element becomes the whole number (order of its value, ~index): all are distinct, and the lowest index wins
// among equal values. The k-th largest of 128 maxima over disjoint groups of elements is a floor under the k-th largest of all, and
// only k groups hold anything above it, so what has to be collected is bounded whatever the row looks like. Once a floor is
// there, an element costs one comparison: what lies above it is collected, and when more than kFew have come, the best k of those
// move the floor up. Ranks of the few that are left are found by counting.
//
// Work: rows in units of 4096 elements, dealt out evenly as one span of units per CTA (three CTAs an SM), so a row may begin
// in one CTA and end in another. Such a row's parts (statistics and k candidates) meet in the plan's scratch; the CTA that comes last
// joins them in the order of the spans. (A unit per CTA and one for the join took two launches for a single row.)
#include <cuda_bf16.h>

#include "nvfp4_internal.h"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_token_logprobs_args_v1) == 128, "log probabilities ABI");

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kPer = 16;                       // elements of a thread and unit
constexpr uint32_t kUnit = kThreads * kPer;
constexpr uint32_t kMaxSpans = 2 * kThreads;        // of a launch, so that a join has at most two parts a thread
constexpr uint32_t kMaxAlternatives = AUGUR_NVFP4_SM100_MAX_ALTERNATIVES;
constexpr uint32_t kFew = 128;
constexpr uint32_t kGroups = kThreads / 2;          // maxima that a floor is found from
// Collected at most: kFew and a whole unit; at a join, k groups of two threads with two parts of k each.
constexpr uint32_t kBuffer = kFew + kUnit;
static_assert(kMaxAlternatives * 2 * (kMaxSpans / kThreads) * kMaxAlternatives <= kBuffer && kMaxAlternatives <= kGroups, "room for what is collected");
constexpr float kLowest = -200.0f;                  // e^-200 is 0 in F32: differences below it need not be told apart, infinities among them

using Key = unsigned long long;

struct Part {
    float most, sum, moment, reserved;
    Key best[kMaxAlternatives];
};
static_assert(sizeof(Part) % 16 == 0, "parts are read 16 bytes at a time");

struct LogprobsParams {
    const void* logits;
    const int32_t* targets;
    float *logprobs, *entropy, *alternative_logprobs;
    int32_t* ids;
    uint32_t* arrivals;      // [spans], zero between launches
    Part* parts;             // [spans][2]
    uint64_t row_stride;
    uint32_t rows, vocabulary, alternatives, units, spans;   // units of a row
    uint32_t aligned;        // rows start on 16 bytes
};

// A logit as a number of the same order: +0 and -0 alike, every NaN above all numbers. 0 is none.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t bits = __float_as_uint(x + 0.0f);   // -0 becomes +0
    if (x != x) return 0xffffffffu;
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t key) {
    return __uint_as_float(key == 0xffffffffu ? 0x7fffffffu : key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ Key make_key(float x, uint32_t index) { return static_cast<Key>(ordered(x)) << 32 | (0xffffffffu - index); }
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ float exp_fast(float x) {   // good to 2^-22 + |x| 2^-24
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

struct Statistics {
    float most, sum, moment;
    __device__ __forceinline__ void clear() { most = -INFINITY, sum = moment = 0.0f; }
    // Over a larger maximum: sum e^(x - m') (x - m') with x - m' = (x - m) + (m - m').
    __device__ __forceinline__ void move_to(float to) {
        if (most == to) return;          // (two -infinities are equal; a NaN goes on below and makes the sums NaN)
        const float step = max_nan(most - to, kLowest), factor = exp_fast(step);
        moment = factor * fmaf(step, sum, moment);
        sum *= factor;
        most = to;
    }
};

template <class T>
struct Load;
template <>
struct Load<float> {
    static constexpr uint32_t kVector = 4;
    static __device__ __forceinline__ float one(const float* x) { return __ldg(x); }
    static __device__ __forceinline__ void vector(const float* x, float* v) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(x));
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    }
};
template <>
struct Load<__nv_bfloat16> {
    static constexpr uint32_t kVector = 8;
    static __device__ __forceinline__ float one(const __nv_bfloat16* x) { return __bfloat162float(__ldg(x)); }
    static __device__ __forceinline__ void vector(const __nv_bfloat16* x, float* v) {
        const uint4 f = __ldg(reinterpret_cast<const uint4*>(x));
        const uint32_t word[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(word[i] << 16), v[2 * i + 1] = __uint_as_float(word[i] & 0xffff0000u);
    }
};

struct Shared {
    Key buffer[kBuffer];
    Key few[kMaxAlternatives * 2 * (kBuffer / kThreads + 1)];   // above a floor found from strided maxima of the buffer
    Key maxima[kGroups];
    Key best[kMaxAlternatives];
    Key floor;
    uint32_t count, few_count, last;
    float most[kWarps], sum[kWarps], moment[kWarps];
};

// The k-th largest of the maxima of 128 pairs of threads, or 0 where fewer than k have one. Every thread gets it.
__device__ Key floor_of(Shared& sh, Key mine, uint32_t k) {
    const Key other = __shfl_xor_sync(0xffffffffu, mine, 1);
    if (other > mine) mine = other;
    if (threadIdx.x == 0) sh.floor = 0;
    if ((threadIdx.x & 1) == 0) sh.maxima[threadIdx.x >> 1] = mine;
    __syncthreads();
    if (threadIdx.x < kGroups) {
        const Key value = sh.maxima[threadIdx.x];
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t i = 0; i < kGroups; i += 2) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&sh.maxima[i]);
            rank += (two.x > value ? 1u : 0u) + (two.y > value ? 1u : 0u);
        }
        if (value && rank == k - 1) sh.floor = value;
    }
    __syncthreads();
    return sh.floor;
}

// The k largest of list[0, count), in order, in sh.best (0 where there are fewer). All keys are distinct.
__device__ void rank_into_best(Shared& sh, const Key* list, uint32_t count, uint32_t k) {
    if (threadIdx.x < k) sh.best[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t at = threadIdx.x; at < count; at += kThreads) {
        const Key value = list[at];
        uint32_t rank = 0;
        for (uint32_t i = 0; i < count; ++i) rank += list[i] > value ? 1u : 0u;
        if (rank < k) sh.best[rank] = value;
    }
    __syncthreads();
}

// The k largest of the buffer in sh.best and at its front; what else it holds is dropped.
__device__ void prune(Shared& sh, uint32_t k) {
    __syncthreads();
    const uint32_t count = sh.count;
    if (count <= kThreads) {
        rank_into_best(sh, sh.buffer, count, k);
    } else {
        Key mine = 0;
        for (uint32_t i = threadIdx.x; i < count; i += kThreads) mine = sh.buffer[i] > mine ? sh.buffer[i] : mine;
        if (threadIdx.x == 0) sh.few_count = 0;
        const Key floor = floor_of(sh, mine, k);
        for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
            if (sh.buffer[i] >= floor) sh.few[atomicAdd(&sh.few_count, 1u)] = sh.buffer[i];
        }
        __syncthreads();
        rank_into_best(sh, sh.few, sh.few_count, k);
    }
    if (threadIdx.x < k) sh.buffer[threadIdx.x] = sh.best[threadIdx.x];
    if (threadIdx.x == 0) sh.count = count < k ? count : k;
    __syncthreads();
}

// The statistics of all threads together, for every thread.
__device__ Statistics together(Shared& sh, Statistics s) {
    float most = s.most;
#pragma unroll
    for (uint32_t step = 16; step; step /= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, step));
    s.move_to(most);
#pragma unroll
    for (uint32_t step = 16; step; step /= 2) {
        s.sum += __shfl_xor_sync(0xffffffffu, s.sum, step);
        s.moment += __shfl_xor_sync(0xffffffffu, s.moment, step);
    }
    const uint32_t warp = threadIdx.x / 32;
    if (threadIdx.x % 32 == 0) sh.most[warp] = s.most, sh.sum[warp] = s.sum, sh.moment[warp] = s.moment;
    __syncthreads();
    most = sh.most[0];
#pragma unroll
    for (uint32_t w = 1; w < kWarps; ++w) most = max_nan(most, sh.most[w]);
    Statistics all{most, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
        Statistics one{sh.most[w], sh.sum[w], sh.moment[w]};
        one.move_to(most);
        all.sum += one.sum, all.moment += one.moment;
    }
    return all;
}

template <class T>
__global__ void __launch_bounds__(kThreads, 3) token_logprobs_kernel(const __grid_constant__ LogprobsParams p) {
    __shared__ Shared sh;
    const uint32_t k = p.alternatives;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint64_t total = static_cast<uint64_t>(p.rows) * p.units;
    uint64_t unit = total * blockIdx.x / p.spans;
    const uint64_t end = total * (blockIdx.x + 1) / p.spans;
    while (unit < end) {
        const uint32_t row = static_cast<uint32_t>(unit / p.units), first = static_cast<uint32_t>(unit - static_cast<uint64_t>(row) * p.units);
        const uint32_t stop = static_cast<uint32_t>(end - unit < p.units - first ? first + (end - unit) : p.units);   // units [first, stop) of the row
        unit += stop - first;
        const T* const x = static_cast<const T*>(p.logits) + row * p.row_stride;
        // A thread's elements of a unit: vectors of 16 bytes, kThreads vectors apart; single elements where rows are not aligned.
        constexpr uint32_t kVector = Load<T>::kVector;
        auto index_of = [&](uint32_t u, uint32_t j) {
            return u * kUnit + (p.aligned ? (j / kVector * kThreads + threadIdx.x) * kVector + j % kVector : j * kThreads + threadIdx.x);
        };
        auto load = [&](uint32_t u, float (&v)[kPer]) {
            if (p.aligned && (u + 1) * kUnit <= p.vocabulary) {
#pragma unroll
                for (uint32_t j = 0; j < kPer; j += kVector) Load<T>::vector(x + index_of(u, j), v + j);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < kPer; ++j) {
                    const uint32_t i = index_of(u, j);
                    v[j] = i < p.vocabulary ? Load<T>::one(x + i) : -INFINITY;
                }
            }
        };
        Statistics s;
        s.clear();
        float floor = -INFINITY;   // logits above it are collected
        if (threadIdx.x == 0) sh.count = 0;
        float v[kPer], next[kPer];
        load(first, v);
        for (uint32_t u = first; u < stop; ++u) {
            if (u + 1 < stop) load(u + 1, next);
            float most = v[0];
#pragma unroll
            for (uint32_t j = 1; j < kPer; ++j) most = max_nan(most, v[j]);
            if (!(most <= s.most)) s.move_to(most);
            const float base = s.most == -INFINITY ? 0.0f : s.most;
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) {
                const float below = max_nan(v[j] - base, kLowest), weight = exp_fast(below);
                s.sum += weight;
                s.moment = fmaf(weight, below, s.moment);
            }
            if (k) {
                if (u == first) {
                    Key mine = 0;
#pragma unroll
                    for (uint32_t j = 0; j < kPer; ++j) {
                        const uint32_t i = index_of(u, j);
                        const Key key = i < p.vocabulary ? make_key(v[j], i) : 0;
                        mine = key > mine ? key : mine;
                    }
                    const Key least = floor_of(sh, mine, k);
                    if (mine && mine >= least) {
#pragma unroll
                        for (uint32_t j = 0; j < kPer; ++j) {
                            const uint32_t i = index_of(u, j);
                            const Key key = i < p.vocabulary ? make_key(v[j], i) : 0;
                            if (key && key >= least) sh.buffer[atomicAdd(&sh.count, 1u)] = key;
                        }
                    }
                    // Behind this unit, equal values have higher indices and lose. (No floor: fewer than k values so far.)
                    if (least) floor = from_ordered(static_cast<uint32_t>(least >> 32));
                } else if (!(most <= floor) || floor != floor) {
                    // floor is NaN where k NaNs were there before: nothing more counts
#pragma unroll
                    for (uint32_t j = 0; j < kPer; ++j) {
                        const uint32_t i = index_of(u, j);
                        if (!(v[j] <= floor) && floor == floor && i < p.vocabulary) sh.buffer[atomicAdd(&sh.count, 1u)] = make_key(v[j], i);
                    }
                }
                __syncthreads();
                if (u + 1 < stop && sh.count > kFew) {
                    prune(sh, k);
                    floor = from_ordered(static_cast<uint32_t>(sh.best[k - 1] >> 32));
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < kPer; ++j) v[j] = next[j];
        }
        if (k) prune(sh, k);
        s = together(sh, s);
        const bool alone = first == 0 && stop == p.units;
        if (!alone) {
            // ---- the row's part; the CTA that comes last goes on with all of them ----
            const uint64_t row_unit = static_cast<uint64_t>(row) * p.units;
            const uint32_t from = static_cast<uint32_t>(((row_unit + 1) * p.spans - 1) / total);              // spans that share the row
            const uint32_t to = static_cast<uint32_t>(((row_unit + p.units) * p.spans - 1) / total);
            Part* const part = p.parts + 2 * blockIdx.x + (first == 0 ? 1 : 0);
            if (threadIdx.x < k) part->best[threadIdx.x] = sh.best[threadIdx.x];
            if (threadIdx.x == 0) part->most = s.most, part->sum = s.sum, part->moment = s.moment;
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                sh.last = atomicAdd(p.arrivals + from, 1u) == to - from;
                sh.count = 0;
            }
            __syncthreads();
            if (!sh.last) continue;
            __threadfence();
            if (threadIdx.x == 0) p.arrivals[from] = 0;   // as the next launch expects it
            auto part_of = [&](uint32_t c) { return p.parts + 2 * c + (c == from ? 1 : 0); };
            s.clear();
            Key mine = 0;
            for (uint32_t c = from + threadIdx.x; c <= to; c += kThreads) {
                const float4 f = __ldcg(reinterpret_cast<const float4*>(part_of(c)));
                Statistics one{f.x, f.y, f.z};
                const float most = max_nan(s.most, one.most);
                s.move_to(most), one.move_to(most);
                s.sum += one.sum, s.moment += one.moment;
                if (k) {
                    const Key key = __ldcg(&part_of(c)->best[0]);
                    mine = key > mine ? key : mine;
                }
            }
            if (k) {
                const Key least = floor_of(sh, mine, k);
                if (mine && mine >= least) {
                    for (uint32_t c = from + threadIdx.x; c <= to; c += kThreads) {
                        for (uint32_t i = 0; i < k; ++i) {
                            const Key key = __ldcg(&part_of(c)->best[i]);
                            if (!key || key < least) break;
                            sh.buffer[atomicAdd(&sh.count, 1u)] = key;
                        }
                    }
                }
                prune(sh, k);
            }
            s = together(sh, s);
        }
        // ---- results of the row ----
        const bool nothing = s.most == -INFINITY;
        const float base = nothing ? 0.0f : s.most, log_sum = logf(s.sum);
        if (threadIdx.x == kThreads - 1) {
            const int32_t target = p.targets[row];
            const bool inside = target >= 0 && static_cast<uint32_t>(target) < p.vocabulary;
            p.logprobs[row] = !inside ? __uint_as_float(0x7fc00000u) : nothing ? -INFINITY : (Load<T>::one(x + target) - base) - log_sum;
            p.entropy[row] = nothing ? 0.0f : log_sum - s.moment / s.sum;
        }
        if (threadIdx.x < k) {
            const Key key = sh.best[threadIdx.x];
            p.ids[static_cast<uint64_t>(row) * k + threadIdx.x] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
            p.alternative_logprobs[static_cast<uint64_t>(row) * k + threadIdx.x] = nothing ? -INFINITY : (from_ordered(static_cast<uint32_t>(key >> 32)) - base) - log_sum;
        }
        __syncthreads();   // before the next row's candidates
    }
}

uint32_t most_spans(uint32_t sm_count) { return 3 * sm_count < kMaxSpans ? 3 * sm_count : kMaxSpans; }

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
    // behind the counter regions, whose words are the arrivals: two parts for every span
    *out_bytes = kCounterBytes + 2 * UINT64_C(1) * most_spans(sm_count) * sizeof(Part);
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
    p.arrivals = reinterpret_cast<uint32_t*>(plan->scratch);
    p.parts = reinterpret_cast<Part*>(plan->scratch + kCounterBytes);
    p.units = (a->vocabulary + kUnit - 1) / kUnit;
    const uint64_t total = static_cast<uint64_t>(a->rows) * p.units;
    p.spans = total < most_spans(plan->sm_count) ? static_cast<uint32_t>(total) : most_spans(plan->sm_count);
    const bool f32 = a->logits_type == AUGUR_NVFP4_SM100_LOGITS_F32;
    p.aligned = a->logits % 16 == 0 && (a->rows == 1 || a->row_stride * (f32 ? 4 : 2) % 16 == 0);
    if (f32) {
        launch_dependent(s->stream, token_logprobs_kernel<float>, p.spans, kThreads, 0, p);
    } else {
        launch_dependent(s->stream, token_logprobs_kernel<__nv_bfloat16>, p.spans, kThreads, 0, p);
    }
    count_launch();
    return submitted();
}
