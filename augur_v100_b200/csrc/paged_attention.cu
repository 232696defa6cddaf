// Attention of a step's 1..8 new tokens per sequence over a paged key-value cache on sm_100a.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale log2(e) q . k_j
//
// The cache is read once (4 kv_heads head_dim bytes a token) and that is the bound: for up to 64 queries per key-value head (new tokens x query
// heads that share it) the products are small change for the tensor cores. So no thread touches a key or a value: TMA brings pages
// into two rings in shared memory, and tcgen05.mma reads them there as the 128-row operand, the queries as the narrow one:
//
//   S^T[key][query]   = K Q^T          K as it lies in the pages (rows of head_dim: K-major), 128 keys a tile
//   O^T[dim][query]  += V^T P^T        V as it lies in the pages (the key is the k dimension: MN-major)
//
// A thread of the four softmax warps holds one key and, up to 16 at a time, the queries of S^T. The running maximum is a reference that only
// moves when a score passes it by more than 2^8: then O^T is scaled down in tensor memory; otherwise a tile costs a thread one comparison, one
// exponential and two 2-byte stores per query. p enters the second product as two BF16 terms, good to 2^-16 of it: with one its rounding was as
// large an error as the output's own. The terms lie side by side on the narrow operand, where they cost next to nothing (as products one
// behind the other a pass over V took the pipe twice: 64 ragged sequences 167 us against 155). The denominators are the same terms times ones.
//
// Work: the cached tokens of all (sequence, key-value head) pairs in units of 64, dealt out evenly as one span of units per SM. A pair
// that lies in several spans leaves an unnormalised part per span in the plan's scratch, and a second launch joins those, in
// the order of the spans. The spans follow from the lengths alone (read on the device, so that a captured call can be replayed).
#include <cfloat>

#include "kv_cache.cuh"
#include "kv_join_record.h"
#include "nvfp4_gemm.cuh"

namespace augur_sm100 {
namespace {
using namespace tc;

static_assert(sizeof(augur_cuda_nvfp4_sm100_paged_attention_args_v1) == 160, "attention ABI");

constexpr uint32_t kMaxQueries = 64;   // new tokens x query heads of a key-value head
constexpr uint32_t kMaxCtas = 256;     // spans that a launch deals out (the join has a thread for each)
constexpr uint32_t kUnit = 64;         // tokens of a unit of work
constexpr uint32_t kTile = 128;        // tokens of an MMA tile
constexpr uint32_t kSlotBytes = kTile * 128;   // 64 dims of a tile
constexpr uint32_t kMaxSequences = AUGUR_NVFP4_SM100_MAX_SEQUENCES;
constexpr uint32_t kOnesBytes = kTile * 32;    // 16 k of ones, as the 128-row operand
constexpr uint32_t kMaxTokensLog2 = 24;   // of a sequence
constexpr float kSlack = 8.0f;            // how far, in powers of two, a score may pass the reference maximum
constexpr float kNoNumber = -FLT_MAX;     // a part's reference where a query sees keys but no score above -infinity (-infinity: sees none)
constexpr uint32_t kStatusPage = 0x401, kStatusRows = 0x402;
constexpr uint32_t kStatusLoad = 0x411, kStatusMma = 0x412, kStatusScores = 0x413, kStatusValues = 0x414, kStatusQuery = 0x415, kStatusGroup = 0x416, kStatusProduct = 0x417;
constexpr uint32_t kThreads = 256;        // warp 0 loads keys, 1 MMA, 2 queries, 3 values, 4..7 softmax
constexpr uint32_t kSmemLimit = 227 * 1024;
constexpr uint32_t kInfos = 8;            // tiles that the loader is ahead of the softmax at most, rounded up

struct AttentionParams {
    const __nv_bfloat16* query;
    __nv_bfloat16* output;
    const int32_t *page_table, *lengths, *token_starts;
    uint32_t* status_word;
    JoinRecord* records;          // [joins]
    float* parts;                 // [spans][2][kN][head_dim], then [spans][2][kN] (reference maximum, denominator)
    uint32_t rows, sequences, table_pages, pages, query_heads, kv_heads, page_shift, max_new, spans, joins;
    float scale_log2;             // scale * log2(e)
};

// Small state of a CTA, behind the rings, the queries and the weights.
struct State {
    uint64_t full[16], empty[16];
    uint64_t scores_full[2], scores_empty[2], weights_full[2], weights_empty[2], query_full[2], query_empty[2], group, keys_first;
    uint32_t tmem, abort[1 + kThreads / 32];
    uint32_t needs[2];                 // a byte per softmax warp: a reference has to move
    uint32_t info[kInfos];             // of a tile: pages that are there, a bit per box
    uint32_t scan[kThreads / 32];
    float reference[kMaxQueries], factor[kMaxQueries];
    float4 wide[kMaxQueries];          // the largest score per query and softmax warp
    int32_t limit[kMaxQueries];        // keys that a query sees
    uint32_t units[kMaxSequences + 1]; // before sequence b, of one head
    uint32_t length[kMaxSequences];    // | new tokens << 25
    uint32_t row[kMaxSequences];       // the first token row
};

template <uint32_t kHeadDim, uint32_t kN>
struct Shape {
    static constexpr uint32_t kChunks = kHeadDim / 64, kHalves = kHeadDim / 128;
    // Columns of S^T (the MMA wants 16 at least), and of P^T and O^T: two BF16 terms of P side by side. kBlock of them are worked on at a time.
    static constexpr uint32_t kScores = kN < 16 ? 16 : kN, kTerms = 2 * kN, kBlock = kN < 16 ? kN : 16;
    static constexpr uint32_t kQueryBytes = kScores * kHeadDim * 2, kWeightBytes = kTerms * kTile * 2;
    static constexpr uint32_t fixed(uint32_t buffers) { return 1024 + kOnesBytes + sizeof(State) + buffers * kQueryBytes + 2 * kWeightBytes; }
    static constexpr uint32_t slots(uint32_t buffers) {
        const uint32_t fit = (kSmemLimit - fixed(buffers)) / kSlotBytes / 2 * 2;
        return fit < 16 ? fit : 16;
    }
    // A ring each for the keys and the values: a slot's uses then all belong to one of the two warps that load, which waits for them in turn. (With
    // slots that go from one warp to the other, a warp could take the end of the use before last for the end of the last one.)
    // The queries of a pair are held twice, so that the next pair's are there in time, but once where a tile of keys and one of values would not fit beside them: 48
    // and 64 columns of head size 256 (8 tokens of 6 heads each, 4 x 16385 tokens: 61.1 us with 4 + 4 slots, 69.3 with 2 + 4). Elsewhere the slots gained are
    // worth less than the second copy (one token of 4 heads of 128 each, 2 x 131071 tokens: 161.8 us with 4 + 6 slots, 171.6 with 6 + 6 and one copy; 8 tokens of
    // them, 4 x 16385: 61.9 with 4 + 4, 62.3 with 4 + 6 and one copy). The slots are even in number: an odd one, which went to the keys, was worth nothing (5 + 4
    // against 4 + 4: 5 tokens of 6 heads of 256 each 57.3 and 56.5 us; 3 + 4 against 2 + 4: 8 tokens of 8 heads of 128 95.6 and 94.1).
    static constexpr uint32_t kQueryBuffers = slots(2) < 2 * kChunks ? 1 : 2, kSlots = slots(kQueryBuffers), kFixed = fixed(kQueryBuffers);
    static constexpr uint32_t kValueSlots = (kSlots / 2 + 1) / 2 * 2, kKeySlots = kSlots - kValueSlots;   // (pairs of value slots are one operand)
    static constexpr uint32_t kSmem = kFixed + kSlots * kSlotBytes;
    // tensor memory: two of S^T, O^T in halves of 128 dims, the denominators
    static constexpr uint32_t kColumns = 2 * kScores + (kHalves + 1) * kTerms, kTmem = kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
    static_assert(kKeySlots >= 2 && kSlots % 2 == 0 && kValueSlots >= kChunks /* a tile's values are looked at before any is used */ && kSmem <= kSmemLimit && kColumns <= 512, "a CTA's memory");
};

template <uint32_t kHeadDim, uint32_t kN>
constexpr uint32_t kLayout = 100 * Shape<kHeadDim, kN>::kKeySlots + 10 * Shape<kHeadDim, kN>::kValueSlots + Shape<kHeadDim, kN>::kQueryBuffers;
static_assert(kLayout<128, 8> == 462 && kLayout<128, 16> == 462 && kLayout<128, 32> == 442 && kLayout<128, 48> == 442 && kLayout<128, 64> == 242 && kLayout<256, 8> == 462 &&
                  kLayout<256, 16> == 462 && kLayout<256, 32> == 442 && kLayout<256, 48> == 441 && kLayout<256, 64> == 241,
              "the slots that the figures above belong to");

// A CTA's way through its span: one (sequence, head) after the other, in each the keys [key, key_end).
struct Walk {
    uint32_t unit, end, sequence, head, key, key_end, length, tokens;
    bool starts, ends;   // the pair's first and last key are in the span

    __device__ void open(const State* st, const AttentionParams& p, uint32_t from, uint32_t to) {
        unit = from, end = to;
        uint32_t low = 0, high = p.sequences;   // the last sequence whose units start at or before `from`
        while (high - low > 1) {
            const uint32_t middle = (low + high) / 2;
            if (st->units[middle] * p.kv_heads <= from) low = middle;
            else high = middle;
        }
        sequence = low;
    }
    __device__ bool next(const State* st, const AttentionParams& p) {
        if (unit >= end) return false;
        while (unit >= st->units[sequence + 1] * p.kv_heads) ++sequence;
        const uint32_t count = st->units[sequence + 1] - st->units[sequence];
        const uint32_t at = unit - st->units[sequence] * p.kv_heads;
        head = at / count;
        const uint32_t first = at - head * count;
        const uint32_t take = end - unit < count - first ? end - unit : count - first;
        length = st->length[sequence] & ((1u << (kMaxTokensLog2 + 1)) - 1), tokens = st->length[sequence] >> (kMaxTokensLog2 + 1);
        starts = first == 0, ends = first + take == count;
        key = first * kUnit;
        const uint32_t stop = (first + take) * kUnit;
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
    __device__ void open(const State* st, const AttentionParams& p, uint32_t from, uint32_t to) {
        walk.open(st, p, from, to);
        seek(st, p);
    }
    __device__ void seek(const State* st, const AttentionParams& p) {
        do {
            valid = walk.next(st, p);
        } while (valid && walk.key >= walk.key_end);
        key = walk.key;
    }
    __device__ void advance(const State* st, const AttentionParams& p) {
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
__device__ __forceinline__ float warp_max(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
    return y;
}

template <uint32_t kHeadDim, uint32_t kN>
__global__ void __launch_bounds__(kThreads, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap map_keys, const __grid_constant__ CUtensorMap map_values, const __grid_constant__ AttentionParams p) {
    using S = Shape<kHeadDim, kN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const query_smem = smem + S::kSlots * kSlotBytes;
    uint8_t* const weight_smem = query_smem + S::kQueryBuffers * S::kQueryBytes;
    uint8_t* const ones_smem = weight_smem + 2 * S::kWeightBytes;
    State* const st = reinterpret_cast<State*>(ones_smem + kOnesBytes);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_u32(st->full), empty = smem_u32(st->empty), scores_full = smem_u32(st->scores_full), scores_empty = smem_u32(st->scores_empty);
    const uint32_t weights_full = smem_u32(st->weights_full), weights_empty = smem_u32(st->weights_empty);
    const uint32_t query_full = smem_u32(st->query_full), query_empty = smem_u32(st->query_empty), group_bar = smem_u32(&st->group);
    volatile uint32_t* abort_flag = st->abort;
    uint32_t* const status = p.status_word;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < S::kSlots; ++s) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1);
        for (uint32_t b = 0; b < 2; ++b) {
            mbar_init(scores_full + 8 * b, 1), mbar_init(scores_empty + 8 * b, 4);
            mbar_init(weights_full + 8 * b, 4), mbar_init(weights_empty + 8 * b, 1);
            mbar_init(query_full + 8 * b, 1), mbar_init(query_empty + 8 * b, 1);
        }
        mbar_init(group_bar, 4), mbar_init(smem_u32(&st->keys_first), 1);
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_keys) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_values) : "memory");
        for (uint32_t i = 0; i < 1 + kThreads / 32; ++i) st->abort[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&st->tmem)), "r"(S::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    for (uint32_t i = threadIdx.x; i < kOnesBytes / 16; i += kThreads) reinterpret_cast<uint4*>(ones_smem)[i] = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Everything above runs while the launch before this one drains; from here on its results are read.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // Units of every sequence, and their running sum.
    auto units_of = [&](uint32_t b) {
        const int32_t from = p.token_starts[b], to = p.token_starts[b + 1];
        int32_t length = p.lengths[b];
        const int32_t room = static_cast<int32_t>(p.table_pages << p.page_shift);
        const bool rows_fit = from >= 0 && to <= static_cast<int32_t>(p.rows) && to >= from && to - from <= static_cast<int32_t>(p.max_new);
        if (!rows_fit && blockIdx.x == 0) atomicCAS(status, 0u, kStatusRows);
        if (length > room) {
            length = room;
            if (blockIdx.x == 0) atomicCAS(status, 0u, kStatusPage);
        }
        if (length < 0) length = 0;
        const uint32_t tokens = rows_fit ? static_cast<uint32_t>(to - from) : 0;
        st->row[b] = static_cast<uint32_t>(from);
        st->length[b] = static_cast<uint32_t>(length) | tokens << (kMaxTokensLog2 + 1);
        if (!tokens && p.joins < p.spans && blockIdx.x == b % p.spans) {
            for (uint32_t h = 0; h < p.kv_heads; ++h) p.records[b * p.kv_heads + h] = JoinRecord{};   // an idle slot's
        }
        return !tokens ? 0 : length ? (static_cast<uint32_t>(length) + kUnit - 1) / kUnit : 1;   // a row that sees nothing is written too
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
    const uint32_t total = st->units[p.sequences] * p.kv_heads, spans = total < p.spans ? total : p.spans;
    const uint32_t base = spans ? total / spans : 0, extra = total - base * spans;   // spans of `base` units, the first `extra` of one more
    const uint32_t from = blockIdx.x * base + (blockIdx.x < extra ? blockIdx.x : extra), to = blockIdx.x < spans ? from + base + (blockIdx.x < extra ? 1 : 0) : from;
    const uint32_t tmem = st->tmem, tmem_out = tmem + 2 * S::kScores, tmem_sum = tmem_out + S::kHalves * S::kTerms;   // (one behind the other: scaled together)
    const uint32_t group = p.query_heads / p.kv_heads;

    if (warp == 0 || warp == 3) {
        // ---------------- pages: warp 0 the keys, warp 3 the values ----------------
        const uint32_t box_shift = p.page_shift < 6 ? p.page_shift : 6, boxes = kTile >> box_shift, box_bytes = 128u << box_shift;
        const CUtensorMap* const map = warp == 0 ? &map_keys : &map_values;
        Tiles tiles;
        tiles.open(st, p, from, to);
        bool alive = true;
        // The first tile's keys go before its values: the scores can be worked on while the values come.
        const uint32_t keys_first = smem_u32(&st->keys_first);
        if (warp == 3 && tiles.valid) alive = warp_look_wait(keys_first, 0, abort_flag, status, kStatusLoad);
        for (uint32_t tile = 0; alive && tiles.valid; ++tile) {
            // the row of the cache where this lane's box of the tile starts, and which lanes have one
            const uint32_t key = tiles.key + (lane << box_shift);
            uint32_t row = 0;
            bool there = false;
            if (lane < boxes && key < tiles.walk.key_end) {
                const int32_t page = __ldg(p.page_table + static_cast<uint64_t>(tiles.walk.sequence) * p.table_pages + (key >> p.page_shift));
                there = page >= 0 && static_cast<uint32_t>(page) < p.pages;
                if (there) row = ((static_cast<uint32_t>(page) * p.kv_heads + tiles.walk.head) << p.page_shift) + (key & ((1u << p.page_shift) - 1));
                else atomicCAS(status, 0u, kStatusPage);
            }
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            tiles.advance(st, p);
            if (warp == 0 && lane == 0) st->info[tile % kInfos] = mask;
            const uint32_t first_slot = warp == 0 ? 0 : S::kKeySlots, slots = warp == 0 ? S::kKeySlots : S::kValueSlots, use = S::kChunks * tile;
            uint32_t slot = first_slot + use % slots, phase = use / slots & 1 ^ 1;
            for (uint32_t c = 0; c < S::kChunks; ++c) {
                if (!warp_look_wait(empty + 8 * slot, phase, abort_flag, status, kStatusLoad)) {
                    alive = false;
                    break;
                }
                const uint32_t bar = full + 8 * slot;
                if (lane == 0) {
                    if (mask) mbar_expect_tx(bar, __popc(mask) * box_bytes);
                    else mbar_arrive(bar);
                }
                __syncwarp();
                if (there) tma_load_2d(smem_u32(smem) + slot * kSlotBytes + lane * box_bytes, map, c * 128, row, bar);
                __syncwarp();
                if (++slot == first_slot + slots) slot = first_slot, phase ^= 1;
            }
            if (warp == 0 && tile == 0 && lane == 0) mbar_arrive(keys_first);
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: S of a tile, then O of the tile before it ----------------
        constexpr uint32_t idesc_any = (1u << 4) | (1u << 7) | (1u << 10) | ((kTile >> 4) << 24);   // F32 += BF16 x BF16
        constexpr uint32_t idesc = idesc_any | ((S::kScores >> 3) << 17), idesc_sum = idesc_any | ((S::kTerms >> 3) << 17), idesc_values = idesc_sum | (1u << 15);                                                        // V is MN-major
        const uint32_t slots = low_word(smem_u32(smem), 16), slots_values = low_word(smem_u32(smem), kSlotBytes);
        const uint32_t queries = low_word(smem_u32(query_smem), 16), weights = low_word(smem_u32(weight_smem), 16), ones = low_word(smem_u32(ones_smem), 128);
        Tiles ahead, now;
        ahead.open(st, p, from, to);
        now = ahead;
        uint32_t key_slot = 0, key_phase = 0, slot = S::kKeySlots, phase = 0, scores = 0, products = 0, pair = 0;
        bool alive = true;
        auto scores_of_tile = [&]() {
            const uint32_t buffer = scores & 1, query = S::kQueryBuffers == 2 ? pair & 1 : 0;
            if (ahead.first() && !warp_look_wait(query_full + 8 * query, (S::kQueryBuffers == 2 ? pair >> 1 : pair) & 1, abort_flag, status, kStatusMma)) return false;
            if (!warp_look_wait(scores_empty + 8 * buffer, (scores >> 1 & 1) ^ 1, abort_flag, status, kStatusMma)) return false;
            for (uint32_t c = 0; c < S::kChunks; ++c) {
                if (!warp_look_wait(full + 8 * key_slot, key_phase, abort_flag, status, kStatusMma)) return false;
                tc_fence_after();
                mma_block<kHighSwizzled, 2>(tmem + buffer * S::kScores, slots + key_slot * (kSlotBytes >> 4), queries + ((query * S::kQueryBytes + c * S::kScores * 128) >> 4), idesc, c, 4);
                commit(empty + 8 * key_slot);
                if (++key_slot == S::kKeySlots) key_slot = 0, key_phase ^= 1;
            }
            commit(scores_full + 8 * buffer);
            if (ahead.last()) {
                commit(query_empty + 8 * query);
                ++pair;
            }
            ++scores;
            ahead.advance(st, p);
            return true;
        };
        if (ahead.valid) alive = scores_of_tile();
        while (alive && now.valid) {
            if (ahead.valid && !scores_of_tile()) break;
            const uint32_t buffer = products & 1, steps = (now.keys() + 15) / 16;
            if (!warp_look_wait(weights_full + 8 * buffer, products >> 1 & 1, abort_flag, status, kStatusProduct)) break;
            tc_fence_after();
            const uint32_t follows = !now.first(), weights_now = weights + ((buffer * S::kWeightBytes) >> 4);
            // denominators: the sum over the keys as one more product, into every lane
            mma_block<kHighPlain, 0>(tmem_sum, ones, weights_now, idesc_sum, follows, steps);
            if (steps > 4) mma_block<kHighPlain, 0>(tmem_sum, ones, weights_now + (S::kTerms * 128 >> 4), idesc_sum, 1, steps - 4);
            for (uint32_t h = 0; alive && h < S::kHalves; ++h) {
                for (uint32_t c = 0; c < 2; ++c) alive = alive && warp_look_wait(full + 8 * (slot + c), phase, abort_flag, status, kStatusProduct);
                if (!alive) break;
                tc_fence_after();
                // 16 keys: 16 rows of V, 32 bytes of a row of P
                const uint32_t a = slots_values + slot * (kSlotBytes >> 4), d = tmem_out + h * S::kTerms;
                mma_block<kHighSwizzled, (16 * 128 >> 4)>(d, a, weights_now, idesc_values, follows, steps);
                if (steps > 4) mma_block<kHighSwizzled, (16 * 128 >> 4)>(d, a + 4 * (16 * 128 >> 4), weights_now + (S::kTerms * 128 >> 4), idesc_values, 1, steps - 4);
                commit(empty + 8 * slot);
                commit(empty + 8 * (slot + 1));
                slot += 2;
                if (slot == S::kSlots) slot = S::kKeySlots, phase ^= 1;
            }
            if (!alive) break;
            commit(weights_empty + 8 * buffer);
            ++products;
            now.advance(st, p);
        }
    } else if (warp == 2) {
        // ---------------- queries of a pair, in the 128-byte swizzle of the operand; rows past the last are zero ----------------
        Walk walk;
        walk.open(st, p, from, to);
        uint32_t pair = 0;
        while (walk.next(st, p)) {
            if (walk.key >= walk.key_end) continue;
            const uint32_t buffer = S::kQueryBuffers == 2 ? pair & 1 : 0;
            const uint32_t first_row = st->row[walk.sequence], queries = walk.tokens * group;
            if (!warp_look_wait(query_empty + 8 * buffer, ((S::kQueryBuffers == 2 ? pair >> 1 : pair) & 1) ^ 1, abort_flag, status, kStatusQuery)) break;
            // 16 bytes a copy, all of them under way together (as loads and stores they waited for one another: 1000 cycles a row)
            constexpr uint32_t kPieces = kHeadDim / 8, kRows = 32 / kPieces;
            const uint32_t piece = lane % kPieces, to = smem_u32(query_smem) + buffer * S::kQueryBytes + (piece >> 3) * (S::kScores * 128);
            const __nv_bfloat16* const from_here = p.query + (static_cast<uint64_t>(first_row) * p.query_heads + walk.head * group) * kHeadDim + piece * 8;
            uint32_t token = 0, head = lane / kPieces;
            for (uint32_t row = lane / kPieces; row < S::kScores; row += kRows, head += kRows) {
                while (head >= group) head -= group, ++token;
                const bool live = row < queries;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + row * 128 + (((piece & 7) ^ (row & 7)) << 4)),
                             "l"(live ? from_here + (static_cast<uint64_t>(token) * p.query_heads + head) * kHeadDim : p.query), "r"(live ? 16 : 0)
                             : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(query_full + 8 * buffer);
            ++pair;
        }
    } else {
        // ---------------- softmax: thread = key of a tile, then dim of the output ----------------
        const uint32_t thread = threadIdx.x - 128, quadrant = warp & 3, lanes = (quadrant * 32) << 16;
        const uint32_t box_shift = p.page_shift < 6 ? p.page_shift : 6, boxes = kTile >> box_shift, all_boxes = (1u << boxes) - 1;
        constexpr uint32_t kBlock = S::kBlock;
        uint32_t tile = 0, meetings = 0;
        JoinRecord record{};
        // The four warps meet (a bounded wait, where a named barrier would hang on a warp that gave up).
        auto meet = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(group_bar);
            return warp_look_wait(group_bar, meetings++ & 1, abort_flag, status, kStatusGroup);
        };
        Walk walk;
        walk.open(st, p, from, to);
        bool alive = true;
        while (alive && walk.next(st, p)) {
            const uint32_t queries = walk.tokens * group;
            const uint32_t first_row = st->row[walk.sequence];
            if (thread < kN) {
                st->reference[thread] = -INFINITY;
                st->limit[thread] = thread < queries ? static_cast<int32_t>(walk.length) - static_cast<int32_t>(walk.tokens) + static_cast<int32_t>(thread / group) + 1 : 0;
            }
            if (!meet()) break;
            const int32_t seen_by_all = static_cast<int32_t>(walk.length) - static_cast<int32_t>(walk.tokens) + 1;
            for (uint32_t key = walk.key; key < walk.key_end; key += kTile, ++tile) {
                const uint32_t buffer = tile & 1;
                if (!warp_look_wait(scores_full + 8 * buffer, tile >> 1 & 1, abort_flag, status, kStatusScores)) {
                    alive = false;
                    break;
                }
                tc_fence_after();
                const uint32_t there = st->info[tile % kInfos];
                const uint32_t count = walk.key_end - key < kTile ? walk.key_end - key : kTile;
                const bool whole = count == kTile && there == all_boxes, masked = !whole || static_cast<int32_t>(key + kTile) > seen_by_all;
                const bool my_key = thread < count && (there >> (thread >> box_shift) & 1);
                // 16 queries' scores of this thread's key. Every step below goes through them again from tensor memory in a rolled loop: with all of 48
                // queries in registers and the loops unrolled, a tile cost 4200 cycles more, for want of instructions from their cache.
                float s[kBlock];
                auto scores = [&](uint32_t c0) {
                    if (kN == kBlock && c0 != 0) return;   // (there already)
                    load_columns<kBlock>(tmem + lanes + buffer * S::kScores + c0 % kN, reinterpret_cast<uint32_t*>(s));
                    tc_wait_ld();
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) s[i] *= p.scale_log2;
                    if (masked) {
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) s[i] = my_key && static_cast<int32_t>(key + thread) < st->limit[c0 % kN + i] ? s[i] : -INFINITY;
                    }
                };
                constexpr uint32_t kAgain = kN == kBlock ? kN : 0;   // up to 16 queries' stay in registers
                bool above = key == walk.key;   // a pair's first tile sets the references
                if (!above) {
#pragma unroll 1
                    for (uint32_t c = 0; c < kN; c += kBlock) {
                        scores(c);
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) above |= s[i] > st->reference[c + i] + kSlack;
                    }
                    above = __any_sync(0xffffffffu, above);
                    if (lane == 0) reinterpret_cast<uint8_t*>(&st->needs[buffer])[quadrant] = above;
                    if (!meet()) {
                        alive = false;
                        break;
                    }
                    above = *const_cast<volatile uint32_t*>(&st->needs[buffer]) != 0;
                } else {
                    scores(0);
                }
                if (above) {
                    // The references move up to the largest scores so far.
#pragma unroll 1
                    for (uint32_t c = 0; c < kN; c += kBlock) {
                        scores(c + kAgain);
                        float most = -INFINITY;
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) {
                            const float x = warp_max(s[i]);
                            if (lane == i) most = x;
                        }
                        if (lane < kBlock) reinterpret_cast<float*>(&st->wide[c + lane])[quadrant] = most;
                    }
                    if (!meet()) {
                        alive = false;
                        break;
                    }
                    if (thread < kN) {
                        const float old = st->reference[thread];
                        const float4 w = st->wide[thread];
                        const float now = fmaxf(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)), old);
                        st->factor[thread] = now == old ? 1.0f : exp2_fast(old - now);
                        st->reference[thread] = now;
                    }
                    if (!meet()) {
                        alive = false;
                        break;
                    }
                    if (key != walk.key) {
                        if (!warp_look_wait(weights_empty + 8 * (buffer ^ 1), (tile - 1) >> 1 & 1, abort_flag, status, kStatusProduct)) {
                            alive = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll 1
                        for (uint32_t c = 0; c < (S::kHalves + 1) * S::kTerms; c += 16) {
                            uint32_t v[16];
                            load_columns<16>(tmem_out + lanes + c, v);
                            tc_wait_ld();
#pragma unroll
                            for (uint32_t i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * st->factor[kN < 16 ? i % kN : c % kN + i]);
                            store_columns16(tmem_out + lanes + c, v);
                        }
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        tc_fence_before();
                    }
                }
                if (!warp_look_wait(weights_empty + 8 * buffer, (tile >> 1 & 1) ^ 1, abort_flag, status, kStatusProduct)) {
                    alive = false;
                    break;
                }
                uint8_t* const to_weights = weight_smem + buffer * S::kWeightBytes + (thread >> 6) * (S::kTerms * 128) + (thread & 7) * 2;
                const uint32_t unit = (thread & 63) >> 3;
#pragma unroll 1
                for (uint32_t c = 0; c < kN; c += kBlock) {
                    scores(c + kAgain);
                    float power[kBlock];   // all references before the first store, which the compiler would not move them across
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) power[i] = st->reference[c + i];
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) power[i] = exp2_fast(s[i] - (power[i] == -INFINITY ? 0.0f : power[i]));
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) {
                        uint8_t* const to = to_weights + (c + i) * 128 + ((unit ^ (i & 7)) << 4);
                        const __nv_bfloat16 high = __float2bfloat16_rn(power[i]);
                        *reinterpret_cast<__nv_bfloat16*>(to) = high;
                        *reinterpret_cast<__nv_bfloat16*>(to + kN * 128) = __float2bfloat16_rn(power[i] - __bfloat162float(high));
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(scores_empty + 8 * buffer);
                if (!whole) {
                    // Rows of V that are no token's are multiplied with weights of zero: whatever lies there, they must be numbers.
                    // These warps do not wait for every use of a slot, so they must not be more than one ahead: the tile before has to be through. (They
                    // took the end of the use before last for that of this one, and wrote their zeros into the values of the tile before.)
                    if (tile && !warp_look_wait(weights_empty + 8 * (buffer ^ 1), (tile - 1) >> 1 & 1, abort_flag, status, kStatusProduct)) {
                        alive = false;
                        break;
                    }
                    const uint32_t use = S::kChunks * tile;
                    uint32_t slot = S::kKeySlots + use % S::kValueSlots, phase = use / S::kValueSlots & 1;
                    for (uint32_t c = 0; alive && c < S::kChunks; ++c) {
                        if (!warp_look_wait(full + 8 * slot, phase, abort_flag, status, kStatusValues)) {
                            alive = false;
                            break;
                        }
                        if (!my_key && thread < (count + 15) / 16 * 16) {
                            uint4* row = reinterpret_cast<uint4*>(smem + slot * kSlotBytes + thread * 128);
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) row[i] = make_uint4(0, 0, 0, 0);
                        }
                        if (++slot == S::kSlots) slot = S::kKeySlots, phase ^= 1;
                    }
                    if (!alive) break;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(weights_full + 8 * buffer);
            }
            if (!alive) break;
            // ---- the pair's output, or its part ----
            const bool any = walk.key < walk.key_end;
            if (any) {
                if (!warp_look_wait(weights_empty + 8 * ((tile - 1) & 1), (tile - 1) >> 1 & 1, abort_flag, status, kStatusProduct)) break;
                tc_fence_after();
            }
            const bool alone = walk.starts && walk.ends;
            const uint32_t part = 2 * blockIdx.x + (walk.starts ? 1 : 0);
            float* const part_out = p.parts + static_cast<uint64_t>(part) * kN * kHeadDim + thread;
            __nv_bfloat16* const out = p.output + (static_cast<uint64_t>(first_row) * p.query_heads + walk.head * group) * kHeadDim + thread;
            const uint32_t next_token = (p.query_heads - group) * kHeadDim;   // from behind a token's queries to the next token's
            float2* const stats = reinterpret_cast<float2*>(p.parts + static_cast<uint64_t>(2 * p.spans) * kN * kHeadDim) + part * kN;
            uint32_t token_end = group;
            uint64_t skipped = 0;
            float2 mine = make_float2(0.0f, 0.0f);   // statistics of query `thread`
            // (No branch by query where 16 are there or a part is written, which has room for all columns: with one, 48 queries took 7000 cycles.)
            auto write = [&](const uint32_t (&v)[S::kHalves + 1][kBlock], uint32_t c0, uint32_t i) {
                const uint32_t c = c0 + i;
                if (c == token_end) token_end += group, skipped += next_token;
                const float all = __uint_as_float(v[S::kHalves][i]);
                float scale;
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(scale) : "f"(all));   // good to 2^-23
#pragma unroll
                for (uint32_t h = 0; h < S::kHalves; ++h) {
                    out[skipped + c * kHeadDim + h * 128] = __float2bfloat16_rn(all == 0.0f ? 0.0f : __uint_as_float(v[h][i]) * scale);
                }
            };
#pragma unroll 1
            for (uint32_t c0 = 0; c0 < queries; c0 += kBlock) {
                uint32_t v[S::kHalves + 1][kBlock], low[S::kHalves + 1][kBlock];   // both terms' sums; the last are the denominators
#pragma unroll
                for (uint32_t h = 0; h <= S::kHalves; ++h) {
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) v[h][i] = 0;
                }
                if (any) {
#pragma unroll
                    for (uint32_t h = 0; h <= S::kHalves; ++h) {
                        load_columns<kBlock>(tmem_out + lanes + h * S::kTerms + c0, v[h]);
                        load_columns<kBlock>(tmem_out + lanes + h * S::kTerms + kN + c0, low[h]);
                    }
                    tc_wait_ld();
#pragma unroll
                    for (uint32_t h = 0; h <= S::kHalves; ++h) {
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) v[h][i] = __float_as_uint(__uint_as_float(v[h][i]) + __uint_as_float(low[h][i]));
                    }
                }
                if (!alone) {
                    float* const to = part_out + c0 * kHeadDim;
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) {
#pragma unroll
                        for (uint32_t h = 0; h < S::kHalves; ++h) to[i * kHeadDim + h * 128] = __uint_as_float(v[h][i]);
                        if (thread == c0 + i) mine.y = __uint_as_float(v[S::kHalves][i]);
                    }
                } else if (c0 + kBlock <= queries) {
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) write(v, c0, i);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) {
                        if (c0 + i < queries) write(v, c0, i);
                    }
                }
            }
            if (!alone && thread < queries) {
                // A part all of whose scores are NaN or -infinity has the reference -infinity too, but counts: its sums may be NaN.
                mine.x = st->reference[thread];
                if (mine.x == -INFINITY && st->limit[thread] > static_cast<int32_t>(walk.key)) mine.x = kNoNumber;
                stats[thread] = mine;
            }
            if (any) tc_fence_before();
            if (!alone) {
                if (walk.starts) {
                    const uint32_t units = st->units[walk.sequence + 1] - st->units[walk.sequence], longer = extra * (base + 1);
                    const uint32_t last = st->units[walk.sequence] * p.kv_heads + (walk.head + 1) * units - 1;   // the pair's last unit
                    record.row = first_row, record.tokens = walk.tokens, record.head = walk.head, record.first = blockIdx.x;
                    record.last = last < longer ? last / (base + 1) : extra + (last - longer) / base;
                }
            }
            if (p.joins < p.spans && walk.starts && thread == 0) p.records[walk.sequence * p.kv_heads + walk.head] = alone ? JoinRecord{} : record;
        }
        if (p.joins == p.spans && thread == 0) p.records[blockIdx.x] = record;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmem) : "memory");
    }
}

// Joins the parts of one pair, in the order of their spans. A CTA takes queries blockIdx.y, blockIdx.y + gridDim.y, ...; four outputs a
// thread, and the threads of a query's outputs as many times over as there are, each with every so many-th part.
constexpr uint32_t kJoinThreads = 256, kJoinCtas = 1184;   // about as many as run at once
// Few queries have few CTAs, and as many loads under way as the parts of one sequence want; many queries more CTAs at once.
template <uint32_t kHeadDim, uint32_t kN>
__global__ void __launch_bounds__(kJoinThreads, kN <= 16 ? 1 : 6) attention_join_kernel(const __grid_constant__ AttentionParams p) {
    constexpr uint32_t kLanes = kHeadDim / 4, kShares = kJoinThreads / kLanes, kAhead = kN <= 16 ? 10 : 6;
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
        float all = sees ? w * mine.y : 0.0f;
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
            const float scale = 1.0f / all;
            const __nv_bfloat162 a = __floats2bfloat162_rn(all == 0.0f ? 0.0f : sum.x * scale, all == 0.0f ? 0.0f : sum.y * scale);
            const __nv_bfloat162 b = __floats2bfloat162_rn(all == 0.0f ? 0.0f : sum.z * scale, all == 0.0f ? 0.0f : sum.w * scale);
            const uint32_t token = query / group;
            const uint64_t at = (static_cast<uint64_t>(record.row + token) * p.query_heads + record.head * group + (query - token * group)) * kHeadDim + 4 * lane;
            *reinterpret_cast<uint2*>(p.output + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
        __syncthreads();   // the next query's values go to the same places
    }
}

uint32_t query_columns(uint32_t query_heads, uint32_t kv_heads, uint32_t max_new) {
    const uint32_t queries = query_heads / kv_heads * max_new;
    return queries <= 8 ? 8 : (queries + 15) / 16 * 16;
}
uint32_t launch_spans(uint32_t sm_count) { return sm_count < kMaxCtas ? sm_count : kMaxCtas; }

template <uint32_t kHeadDim, uint32_t kN>
void launch_attention(cudaStream_t stream, const CUtensorMap& keys, const CUtensorMap& values, const AttentionParams& p) {
    using S = Shape<kHeadDim, kN>;
    launch_dependent(stream, paged_attention_kernel<kHeadDim, kN>, p.spans, kThreads, S::kSmem, keys, values, p);
    const uint32_t queries = p.query_heads / p.kv_heads * p.max_new;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.stream = stream, config.attrs = &attribute, config.numAttrs = 1;
    const uint32_t rows = (kJoinCtas + p.joins - 1) / p.joins;
    config.gridDim = dim3(p.joins, queries < rows ? queries : rows), config.blockDim = dim3(kJoinThreads);
    cudaLaunchKernelEx(&config, attention_join_kernel<kHeadDim, kN>, p);
    count_launch(2);
}

using Launch = void (*)(cudaStream_t, const CUtensorMap&, const CUtensorMap&, const AttentionParams&);
template <uint32_t kHeadDim>
Launch launch_of(uint32_t columns) {
    switch (columns) {
        case 8: return launch_attention<kHeadDim, 8>;
        case 16: return launch_attention<kHeadDim, 16>;
        case 32: return launch_attention<kHeadDim, 32>;
        case 48: return launch_attention<kHeadDim, 48>;
        default: return launch_attention<kHeadDim, 64>;
    }
}

template <uint32_t kHeadDim>
cudaError_t configure() {
    constexpr cudaFuncAttribute kSmem = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 8>, kSmem, Shape<kHeadDim, 8>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 16>, kSmem, Shape<kHeadDim, 16>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 32>, kSmem, Shape<kHeadDim, 32>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 48>, kSmem, Shape<kHeadDim, 48>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 64>, kSmem, Shape<kHeadDim, 64>::kSmem);
    return e;
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
    if (static_cast<uint64_t>(a->batch.table_pages) * a->layer.page_tokens > (1u << kMaxTokensLog2)) return false;
    if (static_cast<uint64_t>(a->batch.sequences) * ((a->batch.table_pages * a->layer.page_tokens + kUnit - 1) / kUnit) * a->layer.kv_heads > INT32_MAX) return false;
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

cudaError_t attention_configure_device() {
    const cudaError_t e = configure<128>();
    return e == cudaSuccess ? configure<256>() : e;
}

}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_paged_attention_scratch_extent_host_v1(
    uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_new_tokens, uint32_t sm_count, uint64_t* out_bytes) {
    if (!out_bytes || !shape_ok(query_heads, kv_heads, head_dim, max_new_tokens) || !sm_count || sm_count > 4096) return invalid();
    // the counter regions of the plan's scratch stay as they are; behind them the records and the parts
    const uint64_t spans = launch_spans(sm_count), columns = query_columns(query_heads, kv_heads, max_new_tokens);
    *out_bytes = kCounterBytes + spans * sizeof(JoinRecord) + 2 * spans * columns * (head_dim + 2) * sizeof(float);
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
    const uint32_t head_dim = a->layer.head_dim, box = a->layer.page_tokens < kUnit ? a->layer.page_tokens : kUnit;
    const uint64_t cache_rows = static_cast<uint64_t>(a->layer.pages) * a->layer.kv_heads * a->layer.page_tokens;
    CUtensorMap keys, values;   // rows of head_dim * 2 bytes, as a map of packed codes with four times the columns
    if (!make_code_map(&keys, a->layer.keys, cache_rows, head_dim * 4, box) || !make_code_map(&values, a->layer.values, cache_rows, head_dim * 4, box)) {
        return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE);
    }
    const uint32_t columns = query_columns(a->query_heads, a->layer.kv_heads, a->max_new_tokens);
    auto launch = head_dim == 256 ? launch_of<256>(columns) : launch_of<128>(columns);
    launch(s->stream, keys, values, p);
    return submitted();
}
