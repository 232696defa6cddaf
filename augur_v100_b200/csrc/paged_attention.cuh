// What the kernels of attention over a paged cache share: the sequences of a launch and how their tokens are dealt out, instructions, and the join of parts.
#pragma once

#include <cfloat>

#include <cuda_fp16.h>

#include "kv_cache.cuh"
#include "kv_join_record.h"
#include "nvfp4_gemm.cuh"

namespace augur_sm100 {
namespace {
using namespace tc;

constexpr uint32_t kMaxQueries = 64;   // new tokens x query heads of a key-value head
constexpr uint32_t kMaxCtas = 256;     // spans that a launch deals out (the join has a thread for each)
constexpr uint32_t kUnit = 64;         // tokens of a unit of work
constexpr uint32_t kTile = 128;        // tokens of an MMA tile
constexpr uint32_t kSlotBytes = kTile * 128;   // 128 bytes of each token of a tile
constexpr uint32_t kMaxSequences = AUGUR_NVFP4_SM100_MAX_SEQUENCES;
constexpr uint32_t kMaxTokensLog2 = 24;   // of a sequence
constexpr float kSlack = 8.0f;            // how far, in powers of two, a score may pass the reference maximum
constexpr float kNoNumber = -FLT_MAX;     // a part's reference where a query sees keys but no score above -infinity (-infinity: sees none)
constexpr uint32_t kStatusPage = 0x401, kStatusRows = 0x402;
constexpr uint32_t kStatusLoad = 0x411, kStatusMma = 0x412, kStatusScores = 0x413, kStatusValues = 0x414, kStatusQuery = 0x415, kStatusGroup = 0x416, kStatusProduct = 0x417;
constexpr uint32_t kThreads = 256;        // warp 0 loads keys, 1 MMA, 2 queries, 3 values, 4..7 softmax
constexpr uint32_t kMaxWarps = 12;        // (a launch may have a second group of softmax warps)
constexpr uint32_t kSmemLimit = 227 * 1024;

}  // namespace

struct AttentionParams {
    const __nv_bfloat16* query;
    __nv_bfloat16* output;
    const int32_t *page_table, *lengths, *token_starts;
    uint32_t* status_word;
    JoinRecord* records;          // [joins]
    float* parts;                 // [spans][2][kN][head_dim], then [spans][2][kN] (reference maximum, denominator)
    uint32_t rows, sequences, table_pages, pages, query_heads, kv_heads, page_shift, max_new, spans, joins;
    float scale_log2;             // scale * log2(e)
    const uint8_t* scales;        // of an E4M3 cache
    uint32_t pair_units;          // what a pair costs beside its units, in units: its beginning and end
};

namespace {

// What a launch knows of its sequences.
struct BatchState {
    uint32_t scan[kMaxWarps];
    uint32_t units[kMaxSequences + 1]; // before sequence b, of one head
    uint32_t length[kMaxSequences];    // | new tokens << 25
    uint32_t row[kMaxSequences];       // the first token row
};

// Units of every sequence, and their running sum. All threads of the CTA; ends with everything written visible to all of them.
__device__ __forceinline__ void scan_units(BatchState* st, const AttentionParams& p, uint32_t warp, uint32_t lane) {
    auto units_of = [&](uint32_t b) {
        const int32_t from = p.token_starts[b], to = p.token_starts[b + 1];
        int32_t length = p.lengths[b];
        const int32_t room = static_cast<int32_t>(p.table_pages << p.page_shift);
        const bool rows_fit = from >= 0 && to <= static_cast<int32_t>(p.rows) && to >= from && to - from <= static_cast<int32_t>(p.max_new);
        if (!rows_fit && blockIdx.x == 0) atomicCAS(p.status_word, 0u, kStatusRows);
        if (length > room) {
            length = room;
            if (blockIdx.x == 0) atomicCAS(p.status_word, 0u, kStatusPage);
        }
        if (length < 0) length = 0;
        const uint32_t tokens = rows_fit ? static_cast<uint32_t>(to - from) : 0;
        st->row[b] = static_cast<uint32_t>(from);
        st->length[b] = static_cast<uint32_t>(length) | tokens << (kMaxTokensLog2 + 1);
        if (!tokens && p.joins < p.spans && blockIdx.x == b % p.spans) {
            for (uint32_t h = 0; h < p.kv_heads; ++h) p.records[b * p.kv_heads + h] = JoinRecord{};   // an idle slot's
        }
        return !tokens ? 0 : (length ? (static_cast<uint32_t>(length) + kUnit - 1) / kUnit : 1) + p.pair_units;   // a row that sees nothing is written too
    };
    if (p.sequences <= 32) {   // every warp for itself, all with the same result
        const uint32_t count = lane < p.sequences ? units_of(lane) : 0;
        uint32_t before = count;
#pragma unroll
        for (uint32_t step = 1; step < 32; step *= 2) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, before, step);
            if (lane >= step) before += other;
        }
        if (lane < p.sequences) st->units[lane + 1] = before;
        if (lane == 0) st->units[0] = 0;
        __syncwarp();
    } else {   // four neighbouring sequences a thread
        static_assert(kMaxSequences == 4 * kThreads, "four sequences a thread");
        uint32_t count[4], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t b = 4 * threadIdx.x + i;
            count[i] = b < p.sequences ? units_of(b) : 0;
            sum += count[i];
        }
        uint32_t before = sum;
#pragma unroll
        for (uint32_t step = 1; step < 32; step *= 2) {
            const uint32_t other = __shfl_up_sync(0xffffffffu, before, step);
            if (lane >= step) before += other;
        }
        if (lane == 31) st->scan[warp] = before;
        before -= sum;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kThreads / 32; ++w) before += w < warp ? st->scan[w] : 0;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            const uint32_t b = 4 * threadIdx.x + i;
            if (b < p.sequences) st->units[b] = before;
            before += count[i];
            if (b + 1 == p.sequences) st->units[p.sequences] = before;
        }
        __syncthreads();
    }
}

// A CTA's way through its span: one (sequence, head) after the other, in each the keys [key, key_end).
struct Walk {
    uint32_t unit, end, sequence, head, key, key_end, length, tokens;
    bool starts, ends;   // the pair's first and last key are in the span

    __device__ static uint32_t sequence_of(const BatchState* st, const AttentionParams& p, uint32_t at) {
        uint32_t low = 0, high = p.sequences;   // the last sequence whose units start at or before it
        while (high - low > 1) {
            const uint32_t middle = (low + high) / 2;
            if (st->units[middle] * p.kv_heads <= at) low = middle;
            else high = middle;
        }
        return low;
    }
    // Where a span is cut: behind the pair, if the cut falls on what it costs beside its units.
    __device__ static uint32_t cut(const BatchState* st, const AttentionParams& p, uint32_t at) {
        if (!p.pair_units || at >= st->units[p.sequences] * p.kv_heads) return at;
        const uint32_t sequence = sequence_of(st, p, at), count = st->units[sequence + 1] - st->units[sequence], within = (at - st->units[sequence] * p.kv_heads) % count;
        return within + p.pair_units >= count ? at + count - within : at;
    }
    __device__ void open(const BatchState* st, const AttentionParams& p, uint32_t from, uint32_t to) {
        unit = from, end = to, sequence = sequence_of(st, p, from);
    }
    __device__ bool next(const BatchState* st, const AttentionParams& p) {
        if (unit >= end) return false;
        while (unit >= st->units[sequence + 1] * p.kv_heads) ++sequence;
        const uint32_t count = st->units[sequence + 1] - st->units[sequence];
        const uint32_t at = unit - st->units[sequence] * p.kv_heads;
        head = at / count;
        const uint32_t first = at - head * count;
        const uint32_t take = end - unit < count - first ? end - unit : count - first;
        length = st->length[sequence] & ((1u << (kMaxTokensLog2 + 1)) - 1), tokens = st->length[sequence] >> (kMaxTokensLog2 + 1);
        const uint32_t units = count - p.pair_units;
        starts = first == 0, ends = first + take >= units;
        key = first * kUnit;
        const uint32_t stop = (first + take < units ? first + take : units) * kUnit;
        key_end = stop < length ? stop : length;
        unit += take;
        return true;
    }
};
// The same, tile by tile (pairs without keys are passed over).
struct Tiles {
    Walk walk;
    uint32_t key;
    bool valid;
    __device__ void open(const BatchState* st, const AttentionParams& p, uint32_t from, uint32_t to) {
        walk.open(st, p, from, to);
        seek(st, p);
    }
    __device__ void seek(const BatchState* st, const AttentionParams& p) {
        do {
            valid = walk.next(st, p);
        } while (valid && walk.key >= walk.key_end);
        key = walk.key;
    }
    __device__ void advance(const BatchState* st, const AttentionParams& p) {
        key += kTile;
        if (key >= walk.key_end) seek(st, p);
    }
    __device__ bool first() const { return key == walk.key; }
    __device__ bool last() const { return key + kTile >= walk.key_end; }
    __device__ uint32_t keys() const { return walk.key_end - key < kTile ? walk.key_end - key : kTile; }
};

// Operand descriptors, low and high word: address and leading offset, stride offset, version and swizzle.
// K and the narrow operands (K-major, 128-byte swizzle: 8 rows are 1024 bytes). V (MN-major): 128-byte rows of 64 dims, one per key, so the rows
// are the k dimension; 8 keys are 1024 bytes, the next 64 dims lie one ring slot further. The ones (K-major, no swizzle): 8 rows x 16 bytes are
// 128 bytes, the next 8 k 128 bytes further, the next 8 rows 256.
constexpr uint32_t kHighSwizzled = (1024 >> 4) | (1u << 14) | (2u << 29), kHighPlain = (256 >> 4) | (1u << 14);
__device__ __forceinline__ uint32_t low_word(uint32_t smem_addr, uint32_t leading) { return ((smem_addr & 0x3ffffu) >> 4) | ((leading >> 4) << 16); }
// Up to four MMAs of 16 k of a converged warp, the 128-row operand kStep (of 16 bytes) further and the narrow one 32 bytes further each time, as
// predicated instructions whose operands are uniform (behind a branch, one by one, an MMA took 65 cycles to issue; the pipe needs 32).
template <uint32_t kHigh, uint32_t kStep>
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate, uint32_t steps) {
    asm volatile(
        "{\n.reg .pred e, p, q, e1, e2, e3;\n.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n.reg .b32 l1, l2, l3, m1, m2, m3;\n"
        "elect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\nsetp.eq.u32 q, 0, 0;\n"
        "setp.gt.and.u32 e1, %5, 1, e;\nsetp.gt.and.u32 e2, %5, 2, e;\nsetp.gt.and.u32 e3, %5, 3, e;\n"
        "add.s32 l1, %1, %8;\nadd.s32 l2, l1, %8;\nadd.s32 l3, l2, %8;\nadd.s32 m1, %2, 2;\nadd.s32 m2, %2, 4;\nadd.s32 m3, %2, 6;\n"
        "mov.b64 a0, {%1, %6};\nmov.b64 a1, {l1, %6};\nmov.b64 a2, {l2, %6};\nmov.b64 a3, {l3, %6};\n"
        "mov.b64 b0, {%2, %7};\nmov.b64 b1, {m1, %7};\nmov.b64 b2, {m2, %7};\nmov.b64 b3, {m3, %7};\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a0, b0, %3, p;\n"
        "@e1 tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, q;\n"
        "@e2 tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, q;\n"
        "@e3 tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, q;\n}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(steps), "r"(kHigh), "r"(kHighSwizzled), "n"(kStep)
        : "memory");
}
// The elected lane's commit (elect.sync always names the same lane of a whole warp: the one that issued the MMAs).
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("{\n.reg .pred e;\nelect.sync _|e, 0xffffffff;\n@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(bar) : "memory");
}
template <uint32_t kCount>
__device__ __forceinline__ void load_columns(uint32_t taddr, uint32_t* v) {
    static_assert(kCount == 8 || kCount == 16, "columns at a time");
    if constexpr (kCount == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                     : "r"(taddr)
                     : "memory");
    } else {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                       "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                     : "r"(taddr)
                     : "memory");
    }
}
__device__ __forceinline__ void store_columns16(uint32_t taddr, const uint32_t* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};"
                 ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                   "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// y 2^x for x <= 0 down to 2^-226, where 2^x alone is zero below 2^-126. With values whose scales are part of the reference (an E4M3 cache's), a
// denominator under a lower one may be 2^(2 * 60 + 8) times its number of keys, and that much more counts than its factor says.
__device__ __forceinline__ float scaled_down(float y, float x) { return x < -100.0f ? y * exp2_fast(x + 100.0f) * 0x1p-100f : y * exp2_fast(x); }
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

// Joins the parts of one pair, in the order of their spans. A CTA takes queries blockIdx.y, blockIdx.y + gridDim.y, ...; four outputs a
// thread, and the threads of a query's outputs as many times over as there are, each with every so many-th part.
constexpr uint32_t kJoinThreads = 256, kJoinCtas = 1184;   // about as many as run at once
// Few CTAs have as many loads under way as the parts of one sequence want; of many (kMany) six run at once on an SM, and take their places while the attention's last CTAs
// are still at work. (148 x 6 of eight columns, two an SM: the last of them began 4.7 us behind the attention.) Either sums in the same order.
template <uint32_t kHeadDim, uint32_t kN, bool kMany>
__global__ void __launch_bounds__(kJoinThreads, kMany ? 6 : 1) attention_join_kernel(const __grid_constant__ AttentionParams p) {
    constexpr uint32_t kLanes = kHeadDim / 4, kShares = kJoinThreads / kLanes, kAhead = kMany ? 6 : 10;
    __shared__ float weight[kMaxCtas];
    __shared__ float4 sums[kShares][kLanes];
    __shared__ float wide[2][kJoinThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const JoinRecord record = p.records[blockIdx.x];
    const uint32_t group = p.query_heads / p.kv_heads, share = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, warp = threadIdx.x / 32;
    if (!join_record_ok(record, group, kN, p.rows, p.kv_heads, p.spans)) return;   // (a launch that gave up may have left anything)
    const uint32_t parts = record.last - record.first + 1;
    auto part = [&](uint32_t i) { return 2 * (record.first + i) + (i == 0 ? 1 : 0); };
    for (uint32_t query = blockIdx.y; query < record.tokens * group; query += gridDim.y) {
        // a part a thread: its weight 2^(reference - largest reference)
        float2 mine = make_float2(-INFINITY, 0.0f);
        if (threadIdx.x < parts) mine = reinterpret_cast<const float2*>(p.parts + static_cast<uint64_t>(2 * p.spans) * kN * kHeadDim)[part(threadIdx.x) * kN + query];
        // this thread's part of the outputs of the first parts, on their way meanwhile
        const float4* const from = reinterpret_cast<const float4*>(p.parts + static_cast<uint64_t>(query) * kHeadDim) + lane;
        float4 v[kAhead];
        auto load = [&](uint32_t first) {
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                v[i] = make_float4(0, 0, 0, 0);
                if (first + i * kShares < parts) v[i] = from[part(first + i * kShares) * (kN * kLanes)];
            }
        };
        load(share);
        float most = mine.x;
#pragma unroll
        for (uint32_t step = 16; step; step /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, step));
        if (threadIdx.x % 32 == 0) wide[0][warp] = most;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kJoinThreads / 32; ++w) most = fmaxf(most, wide[0][w]);
        // Parts of which the query sees nothing are passed over, whatever other queries' keys left in them. All others count, with a weight of zero too:
        // zero times a NaN is one, as in a pair that lies in one span.
        const bool sees = mine.x != -INFINITY;
        const float w = sees ? exp2_fast(mine.x - most) : 0.0f;
        weight[threadIdx.x] = sees ? w : -1.0f;
        float all = sees ? scaled_down(mine.y, mine.x - most) : 0.0f;
#pragma unroll
        for (uint32_t step = 16; step; step /= 2) all += __shfl_xor_sync(0xffffffffu, all, step);
        if (threadIdx.x % 32 == 0) wide[1][warp] = all;
        __syncthreads();
        float4 sum = make_float4(0, 0, 0, 0);
        for (uint32_t first = share; first < parts; first += kAhead * kShares) {
            if (first != share) load(first);
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                const float f = first + i * kShares < parts ? weight[first + i * kShares] : -1.0f;
                if (!(f < 0.0f)) sum.x = fmaf(f, v[i].x, sum.x), sum.y = fmaf(f, v[i].y, sum.y), sum.z = fmaf(f, v[i].z, sum.z), sum.w = fmaf(f, v[i].w, sum.w);
            }
        }
        sums[share][lane] = sum;
        __syncthreads();
        if (share == 0) {
#pragma unroll
            for (uint32_t i = 1; i < kShares; ++i) {
                const float4 x = sums[i][lane];
                sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
            }
            all = wide[1][0];
#pragma unroll
            for (uint32_t i = 1; i < kJoinThreads / 32; ++i) all += wide[1][i];
            const uint32_t token = query / group;
            const uint64_t place = static_cast<uint64_t>(record.row + token) * p.query_heads + record.head * group + (query - token * group), at = place * kHeadDim + 4 * lane;
            const float scale = 1.0f / all;
            const __nv_bfloat162 a = __floats2bfloat162_rn(all == 0.0f ? 0.0f : sum.x * scale, all == 0.0f ? 0.0f : sum.y * scale);
            const __nv_bfloat162 b = __floats2bfloat162_rn(all == 0.0f ? 0.0f : sum.z * scale, all == 0.0f ? 0.0f : sum.w * scale);
            *reinterpret_cast<uint2*>(p.output + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
        __syncthreads();   // the next query's values go to the same places
    }
}

template <uint32_t kHeadDim, uint32_t kN>
void launch_join(cudaStream_t stream, const AttentionParams& p) {
    const uint32_t queries = p.query_heads / p.kv_heads * p.max_new;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.stream = stream, config.attrs = &attribute, config.numAttrs = 1;
    const uint32_t rows = (kJoinCtas + p.joins - 1) / p.joins;
    config.gridDim = dim3(p.joins, queries < rows ? queries : rows), config.blockDim = dim3(kJoinThreads);
    const bool many = kN > 16 || config.gridDim.x * config.gridDim.y > 2 * p.spans;
    cudaLaunchKernelEx(&config, many ? attention_join_kernel<kHeadDim, kN, true> : attention_join_kernel<kHeadDim, kN, kN <= 16 ? false : true>, p);
}

uint32_t query_columns(uint32_t query_heads, uint32_t kv_heads, uint32_t max_new) {
    const uint32_t queries = query_heads / kv_heads * max_new;
    return queries <= 8 ? 8 : (queries + 15) / 16 * 16;
}
uint32_t launch_spans(uint32_t sm_count) { return sm_count < kMaxCtas ? sm_count : kMaxCtas; }

bool shape_ok(uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_new) {
    return kv_heads && kv_heads <= 1024 && query_heads && query_heads <= 1024 && query_heads % kv_heads == 0 && (head_dim == 128 || head_dim == 256) &&
           max_new >= 1 && max_new <= AUGUR_NVFP4_SM100_MAX_SMALL_TOKENS && query_heads / kv_heads * max_new <= kMaxQueries;
}

// The checks of an attention's descriptor; `ranges` (room for kAttentionRanges) are its tensors, the plan's scratch the last.
constexpr size_t kAttentionRanges = 6 + kKvRanges;
template <class Args>
bool attention_args_ok(int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_plan_v1* plan, const Args* a, Range* ranges, size_t* count, augur_cuda_result_v1* failure) {
    *failure = invalid();
    if (!header_ok(d, s, a)) {
        if (a && s && d >= 0 && s->ordinal == d && a->abi_version != AUGUR_CUDA_ABI_VERSION_V1) *failure = make_result(AUGUR_CUDA_STATUS_ABI_VERSION_MISMATCH);
        return false;
    }
    if (!plan_ok(plan, d, s) || !kv_layer_ok(a->layer) || !kv_batch_ok(a->batch) || a->reserved != 0) return false;
    if (static_cast<uint64_t>(a->batch.table_pages) * a->layer.page_tokens > (1u << kMaxTokensLog2)) return false;
    if (static_cast<uint64_t>(a->batch.sequences) * ((a->batch.table_pages * a->layer.page_tokens + kUnit - 1) / kUnit) * a->layer.kv_heads > INT32_MAX) return false;
    if (!shape_ok(a->query_heads, a->layer.kv_heads, a->layer.head_dim, a->max_new_tokens) || !std::isfinite(a->scale)) return false;
    const uint64_t bytes = static_cast<uint64_t>(a->batch.rows) * a->query_heads * a->layer.head_dim * 2;
    if (a->query_len_bytes != bytes || a->output_len_bytes != bytes) return false;
    size_t n = kv_ranges(a->layer, ranges);
    ranges[n++] = {a->query, a->query_len_bytes, 16}, ranges[n++] = {a->output, a->output_len_bytes, 16};
    ranges[n++] = {a->batch.page_table, a->batch.page_table_len_bytes, 4}, ranges[n++] = {a->batch.lengths, a->batch.lengths_len_bytes, 4};
    ranges[n++] = {a->batch.token_starts, a->batch.token_starts_len_bytes, 4}, ranges[n++] = plan_scratch_range(plan);
    *count = n;
    return all_disjoint(ranges, n);
}

// The same for those without a shared prefix, with the plan's scratch.
template <class Args>
bool check_attention(int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_plan_v1* plan, const Args* a, bool full, augur_cuda_result_v1* failure) {
    Range ranges[kAttentionRanges];
    size_t count;
    if (!attention_args_ok(d, s, plan, a, ranges, &count, failure)) return false;
    uint64_t need = 0;
    if (augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(a->query_heads, a->layer.kv_heads, a->layer.head_dim, a->max_new_tokens, plan->sm_count,
                                                                      &need).status != AUGUR_CUDA_STATUS_OK || plan->scratch_bytes < need) return false;
    return !full || inspect_device_ranges(d, ranges, count - 1, failure);
}

// What the launches get of a descriptor that passed.
template <class Args>
AttentionParams attention_params(const augur_cuda_nvfp4_sm100_plan_v1* plan, const Args* a) {
    AttentionParams p{};   // (pair_units stays 0 where the launch does not say more)
    p.query = reinterpret_cast<const __nv_bfloat16*>(a->query);
    p.output = reinterpret_cast<__nv_bfloat16*>(a->output);
    p.page_table = reinterpret_cast<const int32_t*>(a->batch.page_table);
    p.lengths = reinterpret_cast<const int32_t*>(a->batch.lengths);
    p.token_starts = reinterpret_cast<const int32_t*>(a->batch.token_starts);
    p.status_word = plan->status_word;
    p.rows = a->batch.rows, p.sequences = a->batch.sequences, p.table_pages = a->batch.table_pages, p.pages = a->layer.pages;
    p.query_heads = a->query_heads, p.kv_heads = a->layer.kv_heads, p.page_shift = static_cast<uint32_t>(__builtin_ctz(a->layer.page_tokens));
    p.max_new = a->max_new_tokens, p.spans = launch_spans(plan->sm_count);
    p.joins = static_cast<uint64_t>(p.sequences) * p.kv_heads < p.spans ? p.sequences * p.kv_heads : p.spans;
    p.scale_log2 = a->scale * 1.4426950408889634f;
    p.records = reinterpret_cast<JoinRecord*>(plan->scratch + kCounterBytes);
    p.parts = reinterpret_cast<float*>(p.records + p.spans);
    return p;
}

}  // namespace
}  // namespace augur_sm100
