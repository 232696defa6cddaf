// Log probabilities of given tokens, entropy and the best alternatives of rows of logits on sm_100a.
//
//   logprob(t) = x_t - m - ln L,  entropy = ln L - W / L,  L = sum e^(x - m),  W = sum e^(x - m) (x - m)
//
// One pass over the logits, which is the bound (4 or 2 bytes an element against about eight instructions): every thread keeps a running maximum m,
// L and W of its own elements; they are brought to one m where threads, CTAs and rows meet, always in the same order.
//
// The alternatives ride along. An element becomes the whole number (order of its value, ~index): all are distinct, and the lowest index wins
// among equal values. A floor that k elements reach comes from the first unit: the smallest, over the eight warps, of the
// k / 8-th largest of a warp's 32 maxima. From then on an element costs one comparison: what lies above the floor is
// collected, and when more than kFew have come, the best k of those move the floor up (every kBlock units at most, so that the threads
// need not meet in each). Ranks of the few that are left are found by counting. Rows whose order defeats that floor (all
// values equal, or rising) take the slow way: the k-th largest of 128 maxima of distinct numbers is a floor that only k groups of elements
// reach, so what is collected is bounded whatever the row looks like.
//
// Work: rows in units of 16 KB, dealt out evenly as one span of units per CTA (three CTAs an SM), so a row may begin
// in one CTA and end in another. Such a row's parts (statistics and k candidates) meet in the plan's scratch; the CTA that comes last
// joins them in the order of the spans.
//
// A thread copies the elements that it is going to need into slots of its own in shared memory, 48 KB ahead per CTA (cp.async: no
// registers, and nobody to wait for but itself). With the next unit in registers instead, 48 KB an SM for F32 and 24 KB for
// BF16, a pass over 509 x 248320 F32 logits took 128 us and one over 301 x 151936 BF16 logits 41.6. Rows that do not start on 16
// bytes are read from the 16 bytes before on, less what is not theirs.
#include <cuda_bf16.h>

#include <type_traits>

#include "nvfp4_internal.h"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_token_logprobs_args_v1) == 128, "log probabilities ABI");

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kVectors = 4;                    // of 16 bytes that a thread has in a unit: 4096 F32 elements, 8192 BF16
constexpr uint32_t kUnitBytes = kThreads * kVectors * 16, kMostPer = kVectors * 8;
constexpr uint32_t kMaxSpans = 1024;                // of a launch
constexpr uint32_t kRingBytes = 48 * 1024;          // what a CTA has copied ahead
constexpr uint32_t kMaxAlternatives = AUGUR_NVFP4_SM100_MAX_ALTERNATIVES;
constexpr uint32_t kFew = 64;                       // collected before the floor moves up
constexpr uint32_t kBlock = 8;                      // units between two meetings of the threads
constexpr uint32_t kGroups = kThreads / 2;          // maxima that a floor is found from
// Collected at most, above an exact floor of a unit: the elements of k groups, on top of the few that are there. (A join wants less, and a key for each part.)
constexpr uint32_t kRoom = kMaxAlternatives * 2 * kMaxAlternatives;
constexpr uint32_t kBuffer = kFew + kRoom;
static_assert(kMaxAlternatives * 2 * kMostPer <= kRoom && kMaxAlternatives <= kFew && kMaxAlternatives <= kGroups, "room for what is collected");
constexpr uint32_t kSome = kMaxAlternatives * 2 * (kBuffer / kThreads + 1);   // of the buffer, above an exact floor under its strided maxima
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
    uint32_t rows, vocabulary, alternatives, units;   // units of a row
    uint32_t spans, base, extra;                      // spans of base units, the first `extra` of one more
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
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float exp_fast(float x) { return exp2_fast(x * 1.4426950408889634f); }   // good to 2^-22 + |x| 2^-24

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

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
// 16 bytes of logits as they lie in memory: elements 2 i and 2 i + 1; the largest of four times 16 bytes; -infinity in the place of element i.
__device__ __forceinline__ uint32_t word_of(const uint4& f, uint32_t i) { return i == 0 ? f.x : i == 1 ? f.y : i == 2 ? f.z : f.w; }
__device__ __forceinline__ float2 two_of(const uint4& f, uint32_t i, float) { return make_float2(__uint_as_float(word_of(f, 2 * i)), __uint_as_float(word_of(f, 2 * i + 1))); }
__device__ __forceinline__ float2 two_of(const uint4& f, uint32_t i, __nv_bfloat16) {
    const uint32_t word = word_of(f, i);
    return make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
}
__device__ __forceinline__ float largest(const uint4 (&f)[kVectors], float) {
    float most = __uint_as_float(f[0].x);
#pragma unroll
    for (uint32_t j = 0; j < kVectors; ++j) {
        most = max_nan(most, __uint_as_float(f[j].x), __uint_as_float(f[j].y));
        most = max_nan(most, __uint_as_float(f[j].z), __uint_as_float(f[j].w));
    }
    return most;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    uint32_t c;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(c) : "r"(a), "r"(b));
    return c;
}
__device__ __forceinline__ float largest(const uint4 (&f)[kVectors], __nv_bfloat16) {
    uint32_t most = f[0].x;
#pragma unroll
    for (uint32_t j = 0; j < kVectors; ++j) most = max2_nan(max2_nan(most, max2_nan(f[j].x, f[j].y)), max2_nan(f[j].z, f[j].w));
    return max_nan(__uint_as_float(most << 16), __uint_as_float(most & 0xffff0000u));
}
__device__ __forceinline__ void set_lowest(uint4& f, uint32_t i, bool where, float) {
    uint32_t& word = i == 0 ? f.x : i == 1 ? f.y : i == 2 ? f.z : f.w;
    word = where ? 0xff800000u : word;
}
__device__ __forceinline__ void set_lowest(uint4& f, uint32_t i, bool where, __nv_bfloat16) {
    uint32_t& word = i / 2 == 0 ? f.x : i / 2 == 1 ? f.y : i / 2 == 2 ? f.z : f.w;
    word = !where ? word : i % 2 ? (word & 0xffffu) | 0xff800000u : (word & 0xffff0000u) | 0xff80u;
}

struct Meeting {
    uint32_t last;
    float most[kWarps], sum[kWarps], moment[kWarps];
};
struct Shared : Meeting {
    alignas(16) Key buffer[kBuffer + 2];
    alignas(16) Key few[kSome + 2];   // above a floor found from strided maxima of the buffer
    alignas(16) Key maxima[kGroups];
    Key best[kMaxAlternatives];
    Key floor;
    uint32_t count, few_count;
    uint32_t floors[kWarps];
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

// A value that at least k of the threads' maxima (and so k elements) reach: every warp takes its ceil(k / 8) largest away. 0: no value at all.
__device__ uint32_t quick_floor(Shared& sh, uint32_t mine, uint32_t k) {
    uint32_t most = 0;
    for (uint32_t i = 0; i < (k + kWarps - 1) / kWarps; ++i) {
        most = __reduce_max_sync(0xffffffffu, mine);
        const uint32_t holders = __ballot_sync(0xffffffffu, mine == most);
        if (threadIdx.x % 32 == __ffs(holders) - 1) mine = 0;
    }
    if (threadIdx.x % 32 == 0) sh.floors[threadIdx.x / 32] = most;
    __syncthreads();
    most = sh.floors[0];
#pragma unroll
    for (uint32_t w = 1; w < kWarps; ++w) most = min(most, sh.floors[w]);
    return most;
}

// The k largest of list[0, count), in order, in sh.best (0 where there are fewer). All keys are distinct. list has room for one more.
__device__ void rank_into_best(Shared& sh, Key* list, uint32_t count, uint32_t k) {
    if (threadIdx.x < k) sh.best[threadIdx.x] = 0;
    if (threadIdx.x == kThreads - 1) list[count] = 0;   // they are read in pairs
    __syncthreads();
    if (count <= kThreads / 4) {          // four lanes an entry
        const uint32_t at = threadIdx.x / 4;
        const Key value = at < count ? list[at] : 0;
        uint32_t rank = 0;
        for (uint32_t i = 2 * (threadIdx.x % 4); i < count; i += 8) {
            const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(list + i);
            rank += (two.x > value ? 1u : 0u) + (two.y > value ? 1u : 0u);
        }
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if (value && rank < k) sh.best[rank] = value;
    } else {
        for (uint32_t at = threadIdx.x; at < count; at += kThreads) {
            const Key value = list[at];
            uint32_t rank = 0;
#pragma unroll 8
            for (uint32_t i = 0; i < count; i += 2) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(list + i);
                rank += (two.x > value ? 1u : 0u) + (two.y > value ? 1u : 0u);
            }
            if (value && rank < k) sh.best[rank] = value;
        }
    }
    __syncthreads();
}

// Room in a list for `mine` entries of every lane of a warp, by one atomic a warp (an atomic an entry, each waited for: 4700 cycles where this takes
// a few hundred). Returns where the lane's entries go; *after: entries of the list with the warp's.
__device__ __forceinline__ uint32_t reserve(uint32_t* count, uint32_t mine, uint32_t* after) {
    const uint32_t lane = threadIdx.x % 32;
    uint32_t sum = mine;
    if (__any_sync(0xffffffffu, mine > 1)) {
#pragma unroll
        for (uint32_t step = 1; step < 32; step *= 2) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, sum, step);
            if (lane >= step) sum += other;
        }
    } else {
        sum = __popc(__ballot_sync(0xffffffffu, mine) & (0xffffffffu >> (31 - lane)));
    }
    uint32_t base = 0;
    if (lane == 31) base = atomicAdd(count, sum);
    base = __shfl_sync(0xffffffffu, base, 31);
    *after = base + __shfl_sync(0xffffffffu, sum, 31);
    return base + sum - mine;
}

// The k largest of the buffer in sh.best and at its front; what else it holds is dropped.
__device__ void prune(Shared& sh, uint32_t k) {
    __syncthreads();
    const uint32_t count = sh.count;
    if (count <= kThreads / 2) {
        rank_into_best(sh, sh.buffer, count, k);
    } else {
        // Those above a floor; a rough one first, which equal values can defeat.
        Key mine = 0;
        for (uint32_t i = threadIdx.x; i < count; i += kThreads) mine = sh.buffer[i] > mine ? sh.buffer[i] : mine;
        Key floor = static_cast<Key>(quick_floor(sh, static_cast<uint32_t>(mine >> 32), k)) << 32;
        for (uint32_t pass = 0; pass < 2; ++pass) {
            if (threadIdx.x == 0) sh.few_count = 0;
            __syncthreads();
            uint32_t passed = 0, after;
            for (uint32_t i = threadIdx.x; i < count; i += kThreads) passed += sh.buffer[i] && sh.buffer[i] >= floor ? 1 : 0;
            uint32_t at = reserve(&sh.few_count, passed, &after);
            for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
                if (sh.buffer[i] && sh.buffer[i] >= floor) {
                    if (at < kSome) sh.few[at] = sh.buffer[i];
                    ++at;
                }
            }
            __syncthreads();
            if (sh.few_count <= kSome) break;
            floor = floor_of(sh, mine, k);
        }
        rank_into_best(sh, sh.few, sh.few_count, k);
    }
    if (threadIdx.x < k) sh.buffer[threadIdx.x] = sh.best[threadIdx.x];
    if (threadIdx.x == 0) sh.count = count < k ? count : k;
    __syncthreads();
}

// The statistics of all threads together, for every thread. `uniform`: a warp's threads have one maximum.
__device__ Statistics together(Meeting& sh, Statistics s, bool uniform) {
    float most = s.most;
    if (!uniform) {
#pragma unroll
        for (uint32_t step = 16; step; step /= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, step));
        s.move_to(most);
    }
#pragma unroll
    for (uint32_t step = 16; step; step /= 2) {
        s.sum += __shfl_xor_sync(0xffffffffu, s.sum, step);
        s.moment += __shfl_xor_sync(0xffffffffu, s.moment, step);
    }
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (lane == 0) sh.most[warp] = s.most, sh.sum[warp] = s.sum, sh.moment[warp] = s.moment;
    __syncthreads();
    s.most = most = sh.most[lane % kWarps], s.sum = sh.sum[lane % kWarps], s.moment = sh.moment[lane % kWarps];
#pragma unroll
    for (uint32_t step = kWarps / 2; step; step /= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, step));
    s.move_to(most);
#pragma unroll
    for (uint32_t step = kWarps / 2; step; step /= 2) {
        s.sum += __shfl_xor_sync(0xffffffffu, s.sum, step);
        s.moment += __shfl_xor_sync(0xffffffffu, s.moment, step);
    }
    return s;
}

// The span of a unit.
__device__ __forceinline__ uint32_t span_of(const LogprobsParams& p, uint32_t unit) {
    const uint32_t longer = p.extra * (p.base + 1);
    return unit < longer ? unit / (p.base + 1) : p.extra + (unit - longer) / p.base;
}

// Without alternatives (kSelect false) a CTA needs fewer registers, and an SM holds four.
template <class T, bool kSelect>
__global__ void __launch_bounds__(kThreads, kSelect ? 3 : 4) token_logprobs_kernel(const __grid_constant__ LogprobsParams p) {
    __shared__ std::conditional_t<kSelect, Shared, Meeting> sh;
    extern __shared__ uint4 ring[];                                             // [stages][vectors of a thread][threads]
    constexpr uint32_t kVector = 16 / sizeof(T), kPer = kVectors * kVector, kUnit = kThreads * kPer, kStages = kRingBytes / kUnitBytes;
    const uint32_t k = kSelect ? p.alternatives : 0;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint32_t unit = blockIdx.x * p.base + (blockIdx.x < p.extra ? blockIdx.x : p.extra);
    const uint32_t end = unit + p.base + (blockIdx.x < p.extra ? 1 : 0);
    // A thread's elements of a unit: vectors of 16 bytes, kThreads vectors apart, counted from the 16-byte boundary at or before the row.
    uint32_t left = end - unit, ahead_row = unit / p.units, ahead_unit = unit - ahead_row * p.units, ahead_stage = 0;
    const uint32_t ring_mine = static_cast<uint32_t>(__cvta_generic_to_shared(ring + threadIdx.x));
    const T* ahead_from = nullptr;       // this thread's first vector of the next unit
    uint32_t plain_from = 0, plain_to = 0;   // units of the row that hold nothing else
    auto enter = [&]() {
        const T* const x = static_cast<const T*>(p.logits) + ahead_row * p.row_stride;
        const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uint64_t>(x) & 15) / sizeof(T);
        ahead_from = x - shift + static_cast<uint64_t>(ahead_unit) * kUnit + threadIdx.x * kVector;
        plain_from = shift ? 1 : 0, plain_to = (p.vocabulary + shift) / kUnit;
    };
    enter();
    auto fetch = [&]() {
        if (left) {
            const uint32_t slot = ring_mine + ahead_stage * (kVectors * kThreads * 16);
            if (ahead_unit >= plain_from && ahead_unit < plain_to) {
#pragma unroll
                for (uint32_t j = 0; j < kVectors; ++j) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + j * kThreads * 16), "l"(ahead_from + j * kThreads * kVector) : "memory");
                }
            } else {
                const T* const x = static_cast<const T*>(p.logits) + ahead_row * p.row_stride;
                const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uint64_t>(x) & 15) / sizeof(T);
#pragma unroll 1
                for (uint32_t j = 0; j < kVectors; ++j) {
                    const int64_t i = static_cast<int64_t>(ahead_unit) * kUnit + (j * kThreads + threadIdx.x) * kVector - static_cast<int64_t>(shift);
                    if (i < 0) {   // the row's first vector, part of which belongs to others
                        T* const to = reinterpret_cast<T*>(ring + (ahead_stage * kVectors + j) * kThreads + threadIdx.x);
                        for (uint32_t e = shift; e < kVector && e - shift < p.vocabulary; ++e) to[e] = x[e - shift];
                        continue;
                    }
                    const int64_t rest = static_cast<int64_t>(p.vocabulary) - i;
                    const uint32_t bytes = rest >= kVector ? 16 : rest > 0 ? static_cast<uint32_t>(rest) * sizeof(T) : 0;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot + j * kThreads * 16),
                                 "l"(bytes ? x + i : reinterpret_cast<const T*>(reinterpret_cast<uint64_t>(x) & ~UINT64_C(15))), "r"(bytes)
                                 : "memory");
                }
            }
            ahead_from += kUnit;
            if (++ahead_unit == p.units) {
                ahead_unit = 0, ++ahead_row;
                if (left > 1) enter();
            }
            if (++ahead_stage == kStages) ahead_stage = 0;
            --left;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");   // an empty group too: the groups are counted
    };
    uint32_t row = ahead_row, first = ahead_unit, stage = 0;
#pragma unroll 1
    for (uint32_t i = 0; i + 1 < kStages; ++i) fetch();
    while (unit < end) {
        const uint32_t stop = end - unit < p.units - first ? first + (end - unit) : p.units;   // units [first, stop) of the row
        const T* const x = static_cast<const T*>(p.logits) + row * p.row_stride;
        const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uint64_t>(x) & 15) / sizeof(T);
        // the given token's logit, on its way early
        int32_t target = -1;
        float given = 0.0f;
        if (threadIdx.x == kThreads - 1) {
            target = p.targets[row];
            if (target >= 0 && static_cast<uint32_t>(target) < p.vocabulary) given = as_float(x[target]);
            else target = -1;
        }
        Statistics s;
        s.clear();
        float floor = -INFINITY;   // logits above it are collected
        uint32_t block = first;    // first unit since the threads last met
        bool many = false;         // this thread has seen more than kFew collected
        bool ranked = false;       // the best are in order already
        if constexpr (kSelect) {
            if (threadIdx.x == 0) sh.count = 0;
        }
        // The slow way through units [block, until) of the row, again from memory: a floor of distinct numbers for each, none of which lets more than kRoom pass.
        [[maybe_unused]] auto again = [&](uint32_t until) {
          if constexpr (kSelect) {
            __syncthreads();
            const uint32_t count = sh.count < kBuffer ? sh.count : kBuffer;
            if (threadIdx.x == 0) sh.few_count = 0;
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < count; i += kThreads) {   // what came before them stays: kFew at most
                if (0xffffffffu - static_cast<uint32_t>(sh.buffer[i]) < block * kUnit - (block ? shift : 0)) sh.few[atomicAdd(&sh.few_count, 1u)] = sh.buffer[i];
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < sh.few_count; i += kThreads) sh.buffer[i] = sh.few[i];
            if (threadIdx.x == 0) sh.count = sh.few_count;
            for (uint32_t u = block; u < until; ++u) {
                Key key[kPer], mine = 0;
#pragma unroll 1
                for (uint32_t j = 0; j < kPer; ++j) {
                    const uint32_t i = u * kUnit + (j / kVector * kThreads + threadIdx.x) * kVector + j % kVector - shift;
                    key[j] = i < p.vocabulary ? make_key(as_float(x[i]), i) : 0;
                    mine = key[j] > mine ? key[j] : mine;
                }
                const Key least = floor_of(sh, mine, k);
                for (uint32_t j = 0; j < kPer; ++j) {
                    if (key[j] && key[j] >= least) sh.buffer[atomicAdd(&sh.count, 1u)] = key[j];
                }
                prune(sh, k);
            }
          }
        };
        for (uint32_t u = first; u < stop; ++u) {
            fetch();
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
            uint4 raw[kVectors];
#pragma unroll
            for (uint32_t j = 0; j < kVectors; ++j) raw[j] = ring[(stage * kVectors + j) * kThreads + threadIdx.x];
            [[maybe_unused]] const uint32_t stage_now = stage;
            if (++stage == kStages) stage = 0;
            auto index_of = [&](uint32_t j) { return u * kUnit + (j / kVector * kThreads + threadIdx.x) * kVector + j % kVector - shift; };   // below the row: huge
            const bool inside = (u || shift == 0) && (u + 1) * kUnit - shift <= p.vocabulary;
            if (!inside) {
#pragma unroll
                for (uint32_t j = 0; j < kPer; ++j) set_lowest(raw[j / kVector], j % kVector, index_of(j) >= p.vocabulary, T{});
            }
            const float most = largest(raw, T{});
            // One reference for the warp: a new maximum in one of 32 lanes is frequent, in a unit of the whole warp soon rare.
            float warp_most;
            asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(warp_most) : "f"(most));
            if (!(warp_most <= s.most)) s.move_to(max_nan(s.most, warp_most));   // (a NaN stays the maximum)
            const float base = s.most == -INFINITY ? 0.0f : s.most;
            const float2 minus_base = make_float2(-base, -base), log2e = make_float2(1.4426950408889634f, 1.4426950408889634f);
            float2 sum[2] = {make_float2(s.sum, 0.0f), make_float2(0.0f, 0.0f)}, moment[2] = {make_float2(s.moment, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
            for (uint32_t j = 0; j < kPer; j += 2) {
                float2 below = __fadd2_rn(two_of(raw[j / kVector], j % kVector / 2, T{}), minus_base);
                below.x = max_nan(below.x, kLowest), below.y = max_nan(below.y, kLowest);
                const float2 power = __fmul2_rn(below, log2e), weight = make_float2(exp2_fast(power.x), exp2_fast(power.y));
                sum[j / 2 % 2] = __fadd2_rn(sum[j / 2 % 2], weight);
                moment[j / 2 % 2] = __ffma2_rn(weight, below, moment[j / 2 % 2]);
            }
            sum[0] = __fadd2_rn(sum[0], sum[1]), moment[0] = __fadd2_rn(moment[0], moment[1]);
            s.sum = sum[0].x + sum[0].y, s.moment = moment[0].x + moment[0].y;
            if constexpr (kSelect) {
                auto collect = [&](auto passes) {
                    uint32_t mask = 0, after;
#pragma unroll
                    for (uint32_t j = 0; j < kPer; j += 2) {
                        const float2 two = two_of(raw[j / kVector], j % kVector / 2, T{});
                        mask |= (passes(two.x) ? 1u << j : 0) | (passes(two.y) ? 2u << j : 0);
                    }
                    if (!inside) {
#pragma unroll
                        for (uint32_t j = 0; j < kPer; ++j) mask &= index_of(j) < p.vocabulary ? ~0u : ~(1u << j);
                    }
                    uint32_t at = reserve(&sh.count, __popc(mask), &after);
                    for (; mask; mask &= mask - 1, ++at) {   // few: read again where they still are
                        const uint32_t j = __ffs(mask) - 1;
                        const T* const slot = reinterpret_cast<const T*>(ring + (stage_now * kVectors + j / kVector) * kThreads + threadIdx.x);
                        if (at < kBuffer) sh.buffer[at] = make_key(as_float(slot[j % kVector]), index_of(j));
                    }
                    many = many || after > kFew;
                };
                if (u == first) {
                    // (an element that is not there has the value -infinity, and makes no floor: 0 is less than the order of -infinity)
                    bool there = inside;
#pragma unroll
                    for (uint32_t j = 0; j < kPer; ++j) there = there || index_of(j) < p.vocabulary;
                    const uint32_t order = quick_floor(sh, there ? ordered(most) : 0, k);
                    if (order) floor = from_ordered(order);
                    // Here what reaches the floor counts; behind this unit, equal values have higher indices and lose.
                    if (__any_sync(0xffffffffu, !(most < floor))) collect([&](float x) { return !(x < floor); });
                } else if (!(warp_most <= floor) && floor == floor) {   // (k NaNs were there before: nothing more counts)
                    collect([&](float x) { return !(x <= floor); });
                }
                if (u == first || u - block == kBlock - 1 || u + 1 == stop) {
                    // The last to collect has seen that there are many, if anyone has. The first unit's floor is a rough one: it moves at once.
                    if (__syncthreads_or(many || (u == first && u + 1 < stop))) {
                        ranked = sh.count > kBuffer;
                        if (ranked) again(u + 1);
                        else if (u + 1 < stop) prune(sh, k);
                        if (u + 1 < stop) {
                            floor = from_ordered(static_cast<uint32_t>(sh.best[k - 1] >> 32));
                            many = ranked = false;
                            __syncthreads();
                        }
                    }
                    block = u + 1;
                }
            }
        }
        if constexpr (kSelect) {
            if (!ranked) prune(sh, k);
        }
        s = together(sh, s, true);
        const bool alone = first == 0 && stop == p.units;
        const uint32_t row_now = row, row_unit = row * p.units;
        const bool starts = first == 0;
        unit += stop - first, first = 0, ++row;
        if (!alone) {
            // ---- the row's part; the CTA that comes last goes on with all of them ----
            const uint32_t from = span_of(p, row_unit), to = span_of(p, row_unit + p.units - 1);   // spans that share the row
            Part* const part = p.parts + 2 * blockIdx.x + (starts ? 1 : 0);
            if constexpr (kSelect) {
                if (threadIdx.x < k) part->best[threadIdx.x] = sh.best[threadIdx.x];
            }
            if (threadIdx.x == 0) part->most = s.most, part->sum = s.sum, part->moment = s.moment;
            __syncthreads();
            if (threadIdx.x == 0) {   // releases what all threads wrote, and acquires what the others did
                uint32_t before;
                asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(p.arrivals + from) : "memory");
                sh.last = before == to - from;
            }
            __syncthreads();
            if (!sh.last) continue;
            if (threadIdx.x == 0) p.arrivals[from] = 0;   // as the next launch expects it
            auto part_of = [&](uint32_t c) { return p.parts + 2 * c + (c == from ? 1 : 0); };
            const bool mine = from + threadIdx.x <= to;
            float4 f = make_float4(0, 0, 0, 0);
            if (mine) f = __ldcg(reinterpret_cast<const float4*>(part_of(from + threadIdx.x)));
            if constexpr (kSelect) {
                // A floor from one candidate of each of the P parts, its depth-th: the j-th largest of those, j depth >= k, is reached by k candidates, and by at
                // most j k + (P - j) (depth - 1) < 1024. All loads are under way together. (Ranking all candidates of 61 parts took 6100 cycles;
                // following each part's list down to a floor, up to k loads one after the other, 8 rows 21.4 us.)
                const uint32_t parts = to - from + 1, depth = (k + parts - 1) / parts, wanted = (k + depth - 1) / depth;
                static_assert(kRoom / 2 + kMaxSpans <= kBuffer && kMaxAlternatives * kMaxAlternatives <= kRoom / 2, "candidates, and a key for each part behind them");
                Key* const heads = sh.buffer + kRoom / 2;
                for (uint32_t c = threadIdx.x; c < parts; c += kThreads) heads[c] = __ldcg(&part_of(from + c)->best[depth - 1]);
                constexpr uint32_t kHeld = kMaxAlternatives / 8;   // pairs of candidates that one of the four lanes of a part has
                ulonglong2 held[kHeld];
                auto load = [&](uint32_t c) {
#pragma unroll
                    for (uint32_t i = 0; i < kHeld; ++i) {
                        const uint32_t at = 2 * (threadIdx.x % 4) + 8 * i;
                        held[i] = make_ulonglong2(0, 0);
                        if (c < parts && at < k) held[i] = __ldcg(reinterpret_cast<const ulonglong2*>(&part_of(from + c)->best[at]));
                        if (at + 1 >= k) held[i].y = 0;
                    }
                };
                load(threadIdx.x / 4);
                if (threadIdx.x == 0) sh.count = 0, sh.floor = 0;
                __syncthreads();
                for (uint32_t c = threadIdx.x / 4; c < (parts + 7) / 8 * 8; c += kThreads / 4) {   // (whole warps)
                    const Key value = c < parts ? heads[c] : 0;
                    uint32_t rank = 0;
                    for (uint32_t i = threadIdx.x % 4; i < parts; i += 4) rank += heads[i] > value ? 1u : 0u;
                    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
                    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
                    if (value && rank == wanted - 1) sh.floor = value;
                }
                __syncthreads();
                const Key least = sh.floor;    // 0: fewer than k candidates in all
                for (uint32_t c = threadIdx.x / 4; c < (parts + 7) / 8 * 8; c += kThreads / 4) {
                    if (c != threadIdx.x / 4) load(c);
                    uint32_t passed = 0, after;
#pragma unroll
                    for (uint32_t i = 0; i < kHeld; ++i) {
                        passed += held[i].x && held[i].x >= least ? 1 : 0;
                        passed += held[i].y && held[i].y >= least ? 1 : 0;
                    }
                    uint32_t at = reserve(&sh.count, passed, &after);
#pragma unroll
                    for (uint32_t i = 0; i < kHeld; ++i) {
                        if (held[i].x && held[i].x >= least) sh.buffer[at++] = held[i].x;
                        if (held[i].y && held[i].y >= least) sh.buffer[at++] = held[i].y;
                    }
                }
                __syncthreads();
                rank_into_best(sh, sh.buffer, sh.count, k);
            }
            s = Statistics{mine ? f.x : -INFINITY, f.y, f.z};
            for (uint32_t c = from + threadIdx.x + kThreads; c <= to; c += kThreads) {
                f = __ldcg(reinterpret_cast<const float4*>(part_of(c)));
                Statistics one{f.x, f.y, f.z};
                const float most = max_nan(s.most, one.most);
                s.move_to(most), one.move_to(most);
                s.sum += one.sum, s.moment += one.moment;
            }
            s = together(sh, s, false);
        }
        // ---- results of the row ----
        const bool nothing = s.most == -INFINITY;
        const float base = nothing ? 0.0f : s.most, log_sum = logf(s.sum);
        if (threadIdx.x == kThreads - 1) {
            p.logprobs[row_now] = target < 0 ? __uint_as_float(0x7fc00000u) : nothing ? -INFINITY : (given - base) - log_sum;
            p.entropy[row_now] = nothing ? 0.0f : log_sum - s.moment / s.sum;
        }
        if constexpr (kSelect) {
            if (threadIdx.x < k) {
                const Key key = sh.best[threadIdx.x];
                p.ids[static_cast<uint64_t>(row_now) * k + threadIdx.x] = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(key));
                p.alternative_logprobs[static_cast<uint64_t>(row_now) * k + threadIdx.x] = nothing ? -INFINITY : (from_ordered(static_cast<uint32_t>(key >> 32)) - base) - log_sum;
            }
        }
        __syncthreads();   // before the next row's candidates
    }
}

// Rows of up to 32 kEach elements, a warp each, the row in registers. The k-th largest of the lanes' maxima is a floor that k elements reach; what
// reaches it is collected and ranked by counting. Where equal values make that too many, the alternatives are taken one after the other, by two reductions over
// the warp each. (A CTA a row: 4096 x 128 logits with 5 alternatives 57 us, now 5.4; one after the other always: 1000 x 1000 12.1, now 6.7.)
template <class T, uint32_t kEach>
__global__ void __launch_bounds__(kThreads) short_rows_kernel(const __grid_constant__ LogprobsParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t row = blockIdx.x * kWarps + threadIdx.x / 32, lane = threadIdx.x % 32, k = p.alternatives;
    if (row >= p.rows) return;
    const T* const x = static_cast<const T*>(p.logits) + row * p.row_stride;
    float v[kEach];
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) v[j] = j * 32 + lane < p.vocabulary ? as_float(x[j * 32 + lane]) : -INFINITY;
    const int32_t target = p.targets[row];
    const bool given = target >= 0 && static_cast<uint32_t>(target) < p.vocabulary;
    const float given_logit = given ? as_float(x[target]) : 0.0f;
    float most = v[0];
#pragma unroll
    for (uint32_t j = 1; j < kEach; ++j) most = max_nan(most, v[j]);
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(most) : "f"(most));
    const bool nothing = most == -INFINITY;
    const float base = nothing ? 0.0f : most;
    float sum = 0.0f, moment = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        const float below = max_nan(v[j] - base, kLowest), weight = exp_fast(below);
        sum += weight;
        moment = fmaf(weight, below, moment);
    }
#pragma unroll
    for (uint32_t step = 16; step; step /= 2) {
        sum += __shfl_xor_sync(0xffffffffu, sum, step);
        moment += __shfl_xor_sync(0xffffffffu, moment, step);
    }
    const float log_sum = logf(sum);
    if (lane == 0) {
        p.logprobs[row] = !given ? __uint_as_float(0x7fc00000u) : nothing ? -INFINITY : (given_logit - base) - log_sum;
        p.entropy[row] = nothing ? 0.0f : log_sum - moment / sum;
    }
    if (!k) return;
    uint32_t order[kEach], best = 0, id = 0;   // lane i keeps the i-th alternative
    uint32_t mine = 0, above = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) {
        order[j] = j * 32 + lane < p.vocabulary ? ordered(v[j]) : 0;   // 0: none, or taken already
        mine = max(mine, order[j]);
    }
#pragma unroll 8
    for (uint32_t i = 0; i < 32; ++i) {
        const uint32_t other = __shfl_sync(0xffffffffu, mine, i);
        above += other > mine || (other == mine && i < lane) ? 1 : 0;
    }
    // (some lane has that rank; 0 where fewer than k lanes have an element at all: everything counts)
    const uint32_t floor = __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, above == k - 1)) - 1);
    uint32_t mask = 0;
#pragma unroll
    for (uint32_t j = 0; j < kEach; ++j) mask |= order[j] && order[j] >= floor ? 1u << j : 0;
    uint32_t at = __popc(mask);
#pragma unroll
    for (uint32_t step = 1; step < 32; step *= 2) {
        const uint32_t other = __shfl_up_sync(0xffffffffu, at, step);
        if (lane >= step) at += other;
    }
    const uint32_t count = __shfl_sync(0xffffffffu, at, 31);
    constexpr uint32_t kFewest = 256;
    __shared__ __align__(16) Key lists[kWarps][kFewest + 2];
    __shared__ Key ranked[kWarps][kMaxAlternatives];
    if (count <= kFewest) {
        Key* const list = lists[threadIdx.x / 32];
        at -= __popc(mask);
#pragma unroll
        for (uint32_t j = 0; j < kEach; ++j) {
            if (mask >> j & 1) list[at++] = static_cast<Key>(order[j]) << 32 | (0xffffffffu - (j * 32 + lane));
        }
        if (lane == 0) list[count] = 0;
        __syncwarp();
        for (uint32_t i = lane; i < count; i += 32) {
            const Key value = list[i];
            uint32_t rank = 0;
#pragma unroll 4
            for (uint32_t e = 0; e < count; e += 2) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(list + e);
                rank += (two.x > value ? 1u : 0u) + (two.y > value ? 1u : 0u);
            }
            if (rank < k) ranked[threadIdx.x / 32][rank] = value;
        }
        __syncwarp();
        if (lane < k) {
            const Key key = ranked[threadIdx.x / 32][lane];
            best = static_cast<uint32_t>(key >> 32), id = 0xffffffffu - static_cast<uint32_t>(key);
        }
    }
    for (uint32_t i = 0; count > kFewest && i < k; ++i) {
        uint32_t largest = order[0], place = 0;
#pragma unroll
        for (uint32_t j = 1; j < kEach; ++j) {
            if (order[j] > largest) largest = order[j], place = j;
        }
        const uint32_t top = __reduce_max_sync(0xffffffffu, largest);
        const uint32_t where = __reduce_min_sync(0xffffffffu, largest == top ? place * 32 + lane : 0xffffffffu);
        if (where % 32 == lane) {
#pragma unroll
            for (uint32_t j = 0; j < kEach; ++j) order[j] = j == where / 32 ? 0 : order[j];
        }
        if (lane == i) best = top, id = where;
    }
    if (lane < k) {
        p.ids[static_cast<uint64_t>(row) * k + lane] = static_cast<int32_t>(id);
        p.alternative_logprobs[static_cast<uint64_t>(row) * k + lane] = nothing ? -INFINITY : (from_ordered(best) - base) - log_sum;
    }
}

constexpr uint32_t kShortRow = 1024;   // longer rows have a CTA or several
template <class T>
void launch_logprobs(cudaStream_t stream, const LogprobsParams& p) {
    const uint32_t warps = (p.rows + kWarps - 1) / kWarps;
    if (p.vocabulary <= 128) launch_dependent(stream, short_rows_kernel<T, 4>, warps, kThreads, 0, p);
    else if (p.vocabulary <= 256) launch_dependent(stream, short_rows_kernel<T, 8>, warps, kThreads, 0, p);
    else if (p.vocabulary <= kShortRow) launch_dependent(stream, short_rows_kernel<T, kShortRow / 32>, warps, kThreads, 0, p);
    else if (p.alternatives) launch_dependent(stream, token_logprobs_kernel<T, true>, p.spans, kThreads, kRingBytes, p);
    else launch_dependent(stream, token_logprobs_kernel<T, false>, p.spans, kThreads, kRingBytes, p);
}

// Units of a row: of the elements from the 16-byte boundary before it on, where rows may start between two.
uint32_t units_of(const augur_cuda_nvfp4_sm100_token_logprobs_args_v1* a) {
    const uint32_t size = a->logits_type == AUGUR_NVFP4_SM100_LOGITS_F32 ? 4 : 2;
    const bool aligned = a->logits % 16 == 0 && (a->rows == 1 || a->row_stride * size % 16 == 0);
    return (a->vocabulary + (aligned ? 0 : 16 / size - 1) + kUnitBytes / size - 1) / (kUnitBytes / size);
}
uint32_t most_spans(uint32_t sm_count, uint32_t alternatives) {
    const uint32_t ctas = (alternatives ? 3 : 4) * sm_count;
    return ctas < kMaxSpans ? ctas : kMaxSpans;
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
    if (rows * units_of(a) > INT32_MAX) return false;
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

cudaError_t logprobs_configure_device() {
    constexpr cudaFuncAttribute kSmem = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = cudaFuncSetAttribute(token_logprobs_kernel<float, true>, kSmem, kRingBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(token_logprobs_kernel<float, false>, kSmem, kRingBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(token_logprobs_kernel<__nv_bfloat16, true>, kSmem, kRingBytes);
    return e == cudaSuccess ? cudaFuncSetAttribute(token_logprobs_kernel<__nv_bfloat16, false>, kSmem, kRingBytes) : e;
}

}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_token_logprobs_scratch_extent_host_v1(uint32_t rows, uint32_t alternatives,
                                                                                                           uint32_t sm_count, uint64_t* out_bytes) {
    if (!out_bytes || !rows || rows > (1u << 20) || alternatives > AUGUR_NVFP4_SM100_MAX_ALTERNATIVES || !sm_count || sm_count > 4096) return invalid();
    // behind the counter regions, whose words are the arrivals: two parts for every span
    *out_bytes = kCounterBytes + 2 * UINT64_C(1) * most_spans(sm_count, alternatives) * sizeof(Part);
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
    p.units = units_of(a);
    const uint32_t total = a->rows * p.units;
    p.spans = total < most_spans(plan->sm_count, a->alternatives) ? total : most_spans(plan->sm_count, a->alternatives);
    p.base = total / p.spans, p.extra = total % p.spans;
    const bool f32 = a->logits_type == AUGUR_NVFP4_SM100_LOGITS_F32;
    if (f32) launch_logprobs<float>(s->stream, p);
    else launch_logprobs<__nv_bfloat16>(s->stream, p);
    count_launch();
    return submitted();
}
