// Attention of a step's 1..8 new tokens per sequence over a paged cache of E4M3 codes on sm_100a.
//
//   o = sum_j 2^(s_j - m) 2^f_j v_j / sum_j 2^(s_j - m),  s_j = scale log2(e) 2^e_j q . k_j,  k_j, v_j codes, 2^e_j, 2^f_j their scales
//
// The cache is read once, 2 kv_heads (head_dim + 1) bytes a token, half of what the BF16 cache takes; that is the bound. As there, no thread touches a
// key or a value: TMA brings the pages into two rings, and tcgen05.mma (kind::f8f6f4) reads them there as the 128-row operand:
//
//   S^T[key][query]   = K Q^T          K as it lies in the pages (K-major), 128 keys a tile
//   O^T[dim][query]  += V^T W^T        V as it lies in the pages (the key is the k dimension: MN-major)
//
// That unit takes two operands of 8 bits, so what goes with the codes is split into terms of 8 bits:
//   q in two E4M3 terms, in units in which its largest element is 224 at least: a BF16 element above 2^-9 of the largest is met exactly, a smaller one to
//     2^-17 of the largest. Both terms add into the same S^T: two passes over K, for which the pipe has the time (side by side they would double
//     what the softmax reads);
//   w = 2^(s_j + f_j - m), rounded to half precision, in three E5M2 terms, each in units a sixteenth of the one before it: exact, since a term has the half's exponents
//     and takes four bits of its eleven, the sign's among them. Side by side on the narrow operand, whose terms' sums are added at the end. The weight that sets the
//     reference is 2^7: weights down to 2^-21 of it are good to 2^-11 of themselves, smaller ones to 2^-32 of it, which 2^24 tokens add up to 2^-8. (E4M3 terms with the
//     reference at 1 end at 2^-17 and lose every weight below 2^-18 from the numerator alone: one key and 131071 of 2^-18.5 of its weight, all values 1, gave 0.74.)
// A scale is a power of two, so that a value's is part of the weight's exponent: the reference m follows the largest s_j + f_j, and the weights that enter the
// product lie below 2^8 whatever the scales are. The denominator sums w 2^-f_j in F32, a part of it in each softmax thread.
//
// A thread of the softmax warps (four, or two times four that share the queries) holds one key and, up to 16 at a time, the queries of S^T; it writes 16 weights' terms as three
// 16-byte stores (W^T is MN-major: a key's row holds all queries). The reference moves only when a weight would pass 2^8, which is found out while the weights are
// formed; then O^T is scaled down in tensor memory. Spans, parts and their join are those of the BF16 cache's kernel.
#include "paged_attention.cuh"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_paged_attention_e4m3_args_v1) == 176, "attention ABI");

// Weights are formed 2^kLift times too large and brought down to 2^kTop times where they become half precision: the denominator divides by the value's scale again, and wants those of
// small scales down to 2^-30 of the largest. 2^(8 + kLift) * 2^60 and 2^-126 are 2^(30 + 60 + 60 + 8) apart at least, and as much lies between.
constexpr float kLift = 48.0f;
constexpr int kTop = 7;                        // the product's weights reach 2^(kTop + kRoom) = 2^15: a half, and what a term leaves of it, times 16, an E5M2 number
constexpr float kNoReference = 1e30f;         // where a query has seen no key yet: whatever is added, but -infinity, passes
constexpr float kFar = -100.0f, kFarFactor = 0x1p-100f;   // the least first factor, where a reference moves further
constexpr float kRoom = 8.0f;                  // how far, in powers of two, a weight may pass 1, which was the largest when the reference moved
constexpr uint32_t kTileInfos = 16;            // tiles that the loader is ahead of the softmax at most (a ring of keys and three more), rounded up
constexpr uint32_t kWeightAtom = kTile * 32;   // 32 columns of a tile's weights

// Small state of a CTA, behind the rings, the queries and the weights.
struct StateE4m3 : BatchState {
    uint64_t full[16], empty[16], scales_full[kTileInfos];
    uint64_t scores_full[2], scores_empty[2], weights_full[2], weights_empty[2], query_full[2], query_empty[2], group[2], keys_first;
    uint32_t tmem, abort[1 + kMaxWarps];
    uint32_t needs[2][2];              // by group, a byte per softmax warp: a reference has to move
    uint32_t info[kTileInfos];         // of a tile: pages that are there, a bit per box
    float reference[kMaxQueries], factor[2][kMaxQueries], total[kMaxQueries];
    alignas(16) float minus[kMaxQueries];            // the references with the sign changed, kNoReference for -infinity
    alignas(16) float query_scale[2][kMaxQueries];   // (read four at a time)
    float4 wide[kMaxQueries];          // by softmax warp: the largest score, or the sum of the weights
    int32_t limit[kMaxQueries];        // keys that a query sees
    alignas(16) uint16_t scales[kTileInfos][kTile];   // of a tile's keys: the key's, the value's << 8
};

template <uint32_t kHeadDim, uint32_t kN>
struct ShapeE4m3 {
    static constexpr uint32_t kChunks = kHeadDim / 128;
    // Columns of S^T (the MMA wants 16 at least), and of W^T and O^T: three terms side by side, in steps of 16. A softmax warp works on kBlock queries at a time.
    static constexpr uint32_t kScores = kN < 16 ? 16 : kN, kTerms = (3 * kN + 15) / 16 * 16, kAtoms = (kTerms + 31) / 32;
    // From 32 queries on two groups of softmax warps, each for half of them: independent of one another but for where they say that a tile's weights are there. (One group: 3200
    // cycles a tile of 48 queries, more than HBM takes to bring it: 8 tokens of four sequences at 16385 49 us, with two groups 46.)
    static constexpr uint32_t kGroups = kN < 32 ? 1 : 2, kMine = kN / kGroups, kBlock = kMine % 16 == 0 ? 16 : 8, kThreads = 128 + 128 * kGroups;
    static constexpr uint32_t kTermBytes = kScores * kHeadDim, kQueryBytes = 2 * kTermBytes, kWeightBytes = kAtoms * kWeightAtom;
    // The denominators' sums: in registers for one block of queries, else in shared memory.
    static constexpr uint32_t kSumBytes = kMine == kBlock ? 0 : kN * kTile * 4;
    static constexpr uint32_t fixed(uint32_t buffers) { return 1024 + sizeof(StateE4m3) + buffers * kQueryBytes + 2 * kWeightBytes + kSumBytes; }
    static constexpr uint32_t slots(uint32_t buffers) {
        const uint32_t fit = (kSmemLimit - fixed(buffers)) / kSlotBytes / 2 * 2;
        return fit < 16 ? fit : 16;
    }
    // A ring each for the keys and the values, as many slots of 16 KB each as there is room for; the queries of a pair twice where two tiles of both fit beside them, so that a
    // warp of its own can split the next pair's in time. Else the softmax warps split them, all of them, once the last pair's are no longer read.
    static constexpr uint32_t kQueryBuffers = slots(2) < 4 * kChunks ? 1 : 2, kSlots = slots(kQueryBuffers), kFixed = fixed(kQueryBuffers);
    static constexpr uint32_t kKeySlots = kSlots / 2, kValueSlots = kSlots - kKeySlots;
    static constexpr uint32_t kSmem = kFixed + kSlots * kSlotBytes;
    // tensor memory: two of S^T, O^T in parts of 128 dims
    static constexpr uint32_t kColumns = 2 * kScores + kChunks * kTerms, kTmem = kColumns <= 64 ? 64 : kColumns <= 128 ? 128 : kColumns <= 256 ? 256 : 512;
    static_assert(kKeySlots >= kChunks && kValueSlots >= kChunks && kKeySlots / kChunks + 3 <= kTileInfos && kSmem <= kSmemLimit && kColumns <= 512, "a CTA's memory");
};

// Up to four MMAs of 32 k of a converged warp, as mma_block of the BF16 kernel: the 128-row operand kStep (of 16 bytes) further each time, the narrow one kNarrow.
// The narrow operand MN-major in the 32-byte swizzle: 32 bytes are 32 columns of one key, 8 keys 256 bytes, the next 32 columns kWeightAtom further.
constexpr uint32_t kHighWeights = (256 >> 4) | (1u << 14) | (6u << 29);
template <uint32_t kHighNarrow, uint32_t kStep, uint32_t kNarrow>
__device__ __forceinline__ void mma_block_e4m3(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate, uint32_t steps) {
    asm volatile(
        "{\n.reg .pred e, p, q, e1, e2, e3;\n.reg .b64 a0, a1, a2, a3, b0, b1, b2, b3;\n.reg .b32 l1, l2, l3, m1, m2, m3;\n"
        "elect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\nsetp.eq.u32 q, 0, 0;\n"
        "setp.gt.and.u32 e1, %5, 1, e;\nsetp.gt.and.u32 e2, %5, 2, e;\nsetp.gt.and.u32 e3, %5, 3, e;\n"
        "add.s32 l1, %1, %8;\nadd.s32 l2, l1, %8;\nadd.s32 l3, l2, %8;\nadd.s32 m1, %2, %9;\nadd.s32 m2, m1, %9;\nadd.s32 m3, m2, %9;\n"
        "mov.b64 a0, {%1, %6};\nmov.b64 a1, {l1, %6};\nmov.b64 a2, {l2, %6};\nmov.b64 a3, {l3, %6};\n"
        "mov.b64 b0, {%2, %7};\nmov.b64 b1, {m1, %7};\nmov.b64 b2, {m2, %7};\nmov.b64 b3, {m3, %7};\n"
        "@e tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a0, b0, %3, p;\n"
        "@e1 tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a1, b1, %3, q;\n"
        "@e2 tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a2, b2, %3, q;\n"
        "@e3 tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a3, b3, %3, q;\n}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(steps), "r"(kHighSwizzled), "r"(kHighNarrow), "n"(kStep), "n"(kNarrow)
        : "memory");
}

template <uint32_t kCount>
__device__ __forceinline__ void store_columns(uint32_t taddr, const uint32_t* v) {
    if constexpr (kCount == 16) {
        store_columns16(taddr, v);
    } else {
        static_assert(kCount == 8, "columns at a time");
        asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};"
                     ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(taddr)
                     : "memory");
    }
}
__device__ __forceinline__ uint32_t half2_of(float low, float high) {
    uint32_t x;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(x) : "f"(high), "f"(low));
    return x;
}
// A weight's term and what it stands for (E5M2).
__device__ __forceinline__ uint16_t term_of(uint32_t halves) {
    uint16_t x;
    asm("cvt.rn.satfinite.e5m2x2.f16x2 %0, %1;" : "=h"(x) : "r"(halves));
    return x;
}
__device__ __forceinline__ uint32_t halves_of_term(uint16_t codes) {
    uint32_t x;
    asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(x) : "h"(codes));
    return x;
}
__device__ __forceinline__ uint32_t halves_of(uint16_t codes) {
    uint32_t x;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(x) : "h"(codes));
    return x;
}
// (x - y) * 16 of both halves, exact where y is x to the nearest E5M2 number and x at most 2^15.
__device__ __forceinline__ uint32_t rest16(uint32_t x, uint32_t y) {
    const __half2 r = __hmul2(__hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y)), __float2half2_rn(16.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t byte) { return byte < kE4m3LeastScale ? kE4m3LeastScale : byte > kE4m3LargestScale ? kE4m3LargestScale : byte; }

// A pair's queries as two terms, in the 128-byte swizzle of the operand; rows past the last are zero. Each of `warps` warps takes every so many-th round of kRows * kAhead rows.
template <uint32_t kHeadDim, uint32_t kN>
struct SplitQueries {
    using S = ShapeE4m3<kHeadDim, kN>;
    static constexpr uint32_t kLanes = kHeadDim / 8, kRows = 32 / kLanes, kAhead = S::kQueryBuffers == 1 ? 4 : 8;   // lanes for a row, rows at a time, loads under way
    static_assert(S::kScores % (kRows * kAhead) == 0, "rows of a round");
    // A round's rows are on their way while the round before is split, the first of them while the buffer's last pair is still in use. (The place of a row follows from
    // the one before: a division for each made eight loads 1500 cycles.)
    uint4 next[kAhead];
    const __nv_bfloat16* ahead;
    uint32_t row_ahead, within, queries, group, query_heads, first, step;

    __device__ __forceinline__ void load() {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            next[i] = make_uint4(0, 0, 0, 0);
            if (row_ahead < queries) next[i] = *reinterpret_cast<const uint4*>(ahead);
            move(kRows);
        }
    }
    __device__ __forceinline__ void move(uint32_t rows) {
        row_ahead += rows, within += rows, ahead += rows * kHeadDim;
        while (within >= group) within -= group, ahead += (query_heads - group) * kHeadDim;
    }
    __device__ __forceinline__ void open(const __nv_bfloat16* from, uint32_t pair_queries, uint32_t pair_group, uint32_t all_heads, uint32_t warp, uint32_t warps, uint32_t lane) {
        queries = pair_queries, group = pair_group, query_heads = all_heads, first = warp * kRows * kAhead, step = warps * kRows * kAhead;
        row_ahead = within = 0, ahead = from;
        move(first + lane / kLanes);
        load();
    }
    __device__ __forceinline__ void run(uint8_t* to, float* scales, uint32_t lane) {
        const uint32_t piece = lane % kLanes, unit = (piece & 15) >> 1;
        uint8_t* const to_here = to + (piece >> 4) * (S::kScores * 128) + (piece & 1) * 8;
#pragma unroll 1
        for (; first < S::kScores; first += step) {
            uint4 raw[kAhead];
            uint32_t most[kAhead];   // of the magnitudes' bits
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) raw[i] = next[i];
            if (step > kRows * kAhead) move(step - kRows * kAhead);
            load();
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                const uint32_t two = __vmaxu2(__vmaxu2(raw[i].x & 0x7fff7fffu, raw[i].y & 0x7fff7fffu), __vmaxu2(raw[i].z & 0x7fff7fffu, raw[i].w & 0x7fff7fffu));
                most[i] = max(two >> 16, two & 0xffffu);
            }
            if constexpr (kLanes == 32) {
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i) most[i] = __reduce_max_sync(0xffffffffu, most[i]);
            } else {   // a row in either half of the warp: step by step, the rows side by side
#pragma unroll
                for (uint32_t step = kLanes / 2; step; step /= 2) {
#pragma unroll
                    for (uint32_t i = 0; i < kAhead; ++i) most[i] = max(most[i], __shfl_xor_sync(0xffffffffu, most[i], step));
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < kAhead; ++i) {
                const uint32_t row = first + i * kRows + lane / kLanes;
                // the smallest power of two (a normal number) with which the largest is at most 448 = 1.75 * 2^8; a row that is not finite: codes of zero, a scale of NaN
                const bool finite = most[i] < 0x7f80u;
                const uint32_t exponent = (most[i] >> 7) + ((most[i] & 0x7fu) > 0x60u ? 1 : 0), byte = exponent < 9 ? 1 : exponent - 8;
                const float inverse = __uint_as_float((254 - byte) << 23);
                const uint32_t word[4] = {finite ? raw[i].x : 0, finite ? raw[i].y : 0, finite ? raw[i].z : 0, finite ? raw[i].w : 0};
                uint32_t high[4], low[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const float x0 = __uint_as_float(word[e] << 16) * inverse, x1 = __uint_as_float(word[e] & 0xffff0000u) * inverse;
                    uint16_t code;
                    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(code) : "f"(x1), "f"(x0));
                    const uint32_t back = halves_of(code);
                    const float2 met = __half22float2(*reinterpret_cast<const __half2*>(&back));
                    high[e] = code;
                    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(code) : "f"(x1 - met.y), "f"(x0 - met.x));
                    low[e] = code;
                }
                uint8_t* const at = to_here + row * 128 + ((unit ^ (row & 7)) << 4);
                *reinterpret_cast<uint2*>(at) = make_uint2(high[0] | high[1] << 16, high[2] | high[3] << 16);
                *reinterpret_cast<uint2*>(at + S::kTermBytes) = make_uint2(low[0] | low[1] << 16, low[2] | low[3] << 16);
                if (piece == 0 && row < kN) scales[row] = finite ? __uint_as_float(byte << 23) : __uint_as_float(0x7fc00000u);
            }
        }
    }
};

template <uint32_t kHeadDim, uint32_t kN>
__global__ void __launch_bounds__(ShapeE4m3<kHeadDim, kN>::kThreads, 1)
paged_attention_e4m3_kernel(const __grid_constant__ CUtensorMap map_keys, const __grid_constant__ CUtensorMap map_values, const __grid_constant__ AttentionParams p) {
    using S = ShapeE4m3<kHeadDim, kN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const query_smem = smem + S::kSlots * kSlotBytes;
    uint8_t* const weight_smem = query_smem + S::kQueryBuffers * S::kQueryBytes;
    float4* const sum_smem = reinterpret_cast<float4*>(weight_smem + 2 * S::kWeightBytes);   // [kN / 4][kTile]
    StateE4m3* const st = reinterpret_cast<StateE4m3*>(weight_smem + 2 * S::kWeightBytes + S::kSumBytes);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_u32(st->full), empty = smem_u32(st->empty), scores_full = smem_u32(st->scores_full), scores_empty = smem_u32(st->scores_empty);
    const uint32_t weights_full = smem_u32(st->weights_full), weights_empty = smem_u32(st->weights_empty), scales_full = smem_u32(st->scales_full);
    const uint32_t query_full = smem_u32(st->query_full), query_empty = smem_u32(st->query_empty), group_bar = smem_u32(st->group);
    volatile uint32_t* abort_flag = st->abort;
    uint32_t* const status = p.status_word;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < S::kSlots; ++s) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1);
        for (uint32_t i = 0; i < kTileInfos; ++i) mbar_init(scales_full + 8 * i, 1);
        for (uint32_t b = 0; b < 2; ++b) {
            mbar_init(scores_full + 8 * b, 1), mbar_init(scores_empty + 8 * b, 4 * S::kGroups), mbar_init(group_bar + 8 * b, 4);
            mbar_init(weights_full + 8 * b, 4 * S::kGroups), mbar_init(weights_empty + 8 * b, 1);
            mbar_init(query_full + 8 * b, S::kQueryBuffers == 1 ? 4 * S::kGroups : 1), mbar_init(query_empty + 8 * b, 1 + 4 * S::kGroups);   // the MMAs, and the softmax warps with the queries' scales
        }
        mbar_init(smem_u32(&st->keys_first), 1);
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_keys) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_values) : "memory");
        for (uint32_t i = 0; i < 1 + kMaxWarps; ++i) st->abort[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&st->tmem)), "r"(S::kTmem) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Everything above runs while the launch before this one drains; from here on its results are read.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    scan_units(st, p, warp, lane);
    const uint32_t total = st->units[p.sequences] * p.kv_heads, spans = total < p.spans ? total : p.spans;
    const uint32_t base = spans ? total / spans : 0, extra = total - base * spans;   // spans of `base` units, the first `extra` of one more
    const auto cut = [&](uint32_t span) { return Walk::cut(st, p, span * base + (span < extra ? span : extra)); };
    const uint32_t from = blockIdx.x < spans ? cut(blockIdx.x) : 0, to = blockIdx.x < spans ? cut(blockIdx.x + 1) : 0;
    const uint32_t tmem = st->tmem, tmem_out = tmem + 2 * S::kScores;
    const uint32_t group = p.query_heads / p.kv_heads;

    if (warp == 0 || warp == 3) {
        // ---------------- pages: warp 0 the keys and the scales, warp 3 the values ----------------
        const uint32_t box_shift = p.page_shift < 6 ? p.page_shift : 6, boxes = kTile >> box_shift, box_bytes = 128u << box_shift;
        const CUtensorMap* const map = warp == 0 ? &map_keys : &map_values;
        Tiles tiles;
        tiles.open(st, p, from, to);
        bool alive = true;
        // The page of this lane's box of a tile, looked up while the tile before waits for its slots.
        auto page_of = [&]() {
            const uint32_t key = tiles.key + (lane << box_shift);
            return tiles.valid && lane < boxes && key < tiles.walk.key_end
                       ? __ldg(p.page_table + static_cast<uint64_t>(tiles.walk.sequence) * p.table_pages + (key >> p.page_shift)) : INT32_MIN;
        };
        int32_t page = page_of();
        // The first tile's keys go before its values: the scores can be worked on while the values come.
        const uint32_t keys_first = smem_u32(&st->keys_first);
        if (warp == 3 && tiles.valid) alive = warp_look_suspended(keys_first, 0, abort_flag, status, kStatusLoad);
        for (uint32_t tile = 0; alive && tiles.valid; ++tile) {
            // the row of the cache where this lane's box of the tile starts, and which lanes have one
            const bool there = page >= 0 && static_cast<uint32_t>(page) < p.pages;
            if (!there && page != INT32_MIN) atomicCAS(status, 0u, kStatusPage);
            const uint32_t row = there ? ((static_cast<uint32_t>(page) * p.kv_heads + tiles.walk.head) << p.page_shift) + ((tiles.key + (lane << box_shift)) & ((1u << p.page_shift) - 1)) : 0;
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            tiles.advance(st, p);
            page = page_of();
            if (warp == 0) {
                const uint32_t at = tile % kTileInfos, bar = scales_full + 8 * at;
                if (lane == 0) {
                    st->info[at] = mask;
                    if (mask) mbar_expect_tx(bar, __popc(mask) * (2u << box_shift));
                    else mbar_arrive(bar);
                }
                __syncwarp();
                if (there) bulk_load(smem_u32(st->scales[at]) + (lane << box_shift) * 2, p.scales + static_cast<uint64_t>(row) * 2, 2u << box_shift, bar);
            }
            const uint32_t first_slot = warp == 0 ? 0 : S::kKeySlots, slots = warp == 0 ? S::kKeySlots : S::kValueSlots, use = S::kChunks * tile;
            uint32_t slot = first_slot + use % slots, phase = use / slots & 1 ^ 1;
            for (uint32_t c = 0; c < S::kChunks; ++c) {
                if (!warp_look_suspended(empty + 8 * slot, phase, abort_flag, status, kStatusLoad)) {
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
        constexpr uint32_t idesc_any = (1u << 4) | ((kTile >> 4) << 24);   // F32 += E4M3 x E4M3, or (1 << 10) x E5M2
        constexpr uint32_t idesc = idesc_any | ((S::kScores >> 3) << 17), idesc_values = idesc_any | (1u << 10) | ((S::kTerms >> 3) << 17) | (1u << 15) | (1u << 16);   // V and W MN-major
        const uint32_t slots = low_word(smem_u32(smem), 16);
        const uint32_t queries = low_word(smem_u32(query_smem), 16), weights = low_word(smem_u32(weight_smem), kWeightAtom);
        Tiles ahead, now;
        ahead.open(st, p, from, to);
        now = ahead;
        uint32_t key_slot = 0, key_phase = 0, slot = S::kKeySlots, phase = 0, scores = 0, products = 0, pair = 0;
        bool alive = true;
        auto scores_of_tile = [&]() {
            const uint32_t buffer = scores & 1, query = S::kQueryBuffers == 2 ? pair & 1 : 0;
            if (ahead.first() && !warp_look_suspended(query_full + 8 * query, (S::kQueryBuffers == 2 ? pair >> 1 : pair) & 1, abort_flag, status, kStatusMma)) return false;
            if (!warp_look_suspended(scores_empty + 8 * buffer, (scores >> 1 & 1) ^ 1, abort_flag, status, kStatusMma)) return false;
            for (uint32_t c = 0; c < S::kChunks; ++c) {
                if (!warp_look_suspended(full + 8 * key_slot, key_phase, abort_flag, status, kStatusMma)) return false;
                tc_fence_after();
                const uint32_t a = slots + key_slot * (kSlotBytes >> 4), b = queries + ((query * S::kQueryBytes + c * S::kScores * 128) >> 4);
                mma_block_e4m3<kHighSwizzled, 2, 2>(tmem + buffer * S::kScores, a, b, idesc, c, 4);
                mma_block_e4m3<kHighSwizzled, 2, 2>(tmem + buffer * S::kScores, a, b + (S::kTermBytes >> 4), idesc, 1, 4);
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
        auto product_of_tile = [&]() {
            const uint32_t buffer = products & 1, steps = (now.keys() + 31) / 32;
            if (!warp_look_suspended(weights_full + 8 * buffer, products >> 1 & 1, abort_flag, status, kStatusProduct)) return false;
            for (uint32_t h = 0; h < S::kChunks; ++h) {
                if (!warp_look_suspended(full + 8 * slot, phase, abort_flag, status, kStatusProduct)) return false;
                tc_fence_after();
                // 32 keys: 32 rows of 128 bytes of V, of 32 bytes of W
                mma_block_e4m3<kHighWeights, (32 * 128 >> 4), (32 * 32 >> 4)>(tmem_out + h * S::kTerms, slots + slot * (kSlotBytes >> 4), weights + ((buffer * S::kWeightBytes) >> 4),
                                                                              idesc_values, !now.first(), steps);
                commit(empty + 8 * slot);
                if (++slot == S::kSlots) slot = S::kKeySlots, phase ^= 1;
            }
            commit(weights_empty + 8 * buffer);
            ++products;
            now.advance(st, p);
            return true;
        };
        // The scores of a tile are formed once the softmax is done with those of two tiles before, ahead of that tile's product: behind it, the softmax waited for them. (Whichever
        // can go next, found out by polling: two documents of 131071 tokens 121 us, so 102.) A new pair's queries may be waiting for the products of the pair before.
        while (alive && now.valid) {
            while (alive && ahead.valid && scores < products + 3) {
                if (ahead.first() && scores != products) {
                    const uint32_t query = S::kQueryBuffers == 2 ? pair & 1 : 0, query_phase = (S::kQueryBuffers == 2 ? pair >> 1 : pair) & 1;
                    if (!__all_sync(0xffffffffu, mbar_test(query_full + 8 * query, query_phase))) break;
                }
                alive = scores_of_tile();
            }
            alive = alive && product_of_tile();
        }
    } else if (warp == 2) {
        // ---------------- queries of a pair as two terms, in the 128-byte swizzle of the operand; rows past the last are zero ----------------
        constexpr uint32_t kLanes = kHeadDim / 8, kRows = 32 / kLanes;   // lanes for a row, rows at a time
        Walk walk;
        walk.open(st, p, from, to);
        uint32_t pair = 0;
        while (walk.next(st, p)) {
            if (walk.key >= walk.key_end) continue;
            const uint32_t buffer = S::kQueryBuffers == 2 ? pair & 1 : 0;
            const uint32_t first_row = st->row[walk.sequence], queries = walk.tokens * group;
            const __nv_bfloat16* const from_here = p.query + (static_cast<uint64_t>(first_row) * p.query_heads + walk.head * group) * kHeadDim + lane % kLanes * 8;
            if constexpr (S::kQueryBuffers == 1) {   // the softmax warps split them; here they are only brought nearer
                for (uint32_t row = lane / kLanes; row < queries; row += kRows) {
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(from_here + (static_cast<uint64_t>(row / group) * p.query_heads + row % group) * kHeadDim));
                }
                continue;
            }
            SplitQueries<kHeadDim, kN> split;
            split.open(from_here, queries, group, p.query_heads, 0, 1, lane);
            if (!warp_look_suspended(query_empty + 8 * buffer, (pair >> 1 & 1) ^ 1, abort_flag, status, kStatusQuery)) break;
            split.run(query_smem + buffer * S::kQueryBytes, st->query_scale[buffer], lane);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(query_full + 8 * buffer);
            ++pair;
        }
    } else {
        // ---------------- softmax: thread = key of a tile, then dim of the output ----------------
        const uint32_t thread = threadIdx.x & 127, quadrant = warp & 3, lanes = (quadrant * 32) << 16;
        const uint32_t half = S::kGroups == 1 ? 0 : (warp - 4) / 4, first = half * S::kMine, behind = first + S::kMine;   // the group, its queries
        const uint32_t box_shift = p.page_shift < 6 ? p.page_shift : 6, boxes = kTile >> box_shift, all_boxes = (1u << boxes) - 1;
        constexpr uint32_t kBlock = S::kBlock;
        constexpr bool kOneBlock = S::kMine == kBlock;
        uint32_t tile = 0, meetings = 0, pair = 0;
        JoinRecord record{};
        // The four warps of a group meet (a bounded wait, where a named barrier would hang on a warp that gave up).
        auto come = [&]() {
            __syncwarp();
            if (lane == 0) mbar_arrive(group_bar + 8 * half);
        };
        auto all_came = [&]() { return warp_look_suspended(group_bar + 8 * half, meetings++ & 1, abort_flag, status, kStatusGroup); };
        auto meet = [&]() {
            come();
            return all_came();
        };
        Walk walk;
        walk.open(st, p, from, to);
        bool alive = true;
        while (alive && walk.next(st, p)) {
            const uint32_t queries = walk.tokens * group;
            const uint32_t first_row = st->row[walk.sequence];
            const bool any = walk.key < walk.key_end;
            const uint32_t mine = first + thread;   // the query whose reference this thread keeps
            if (thread < S::kMine) {
                st->reference[mine] = -INFINITY;
                st->limit[mine] = mine < queries ? static_cast<int32_t>(walk.length) - static_cast<int32_t>(walk.tokens) + static_cast<int32_t>(mine / group) + 1 : 0;
            }
            if (!meet()) break;
            const uint32_t query_buffer = S::kQueryBuffers == 2 ? pair & 1 : 0;
            const float* const query_scale = st->query_scale[query_buffer];
            if (S::kQueryBuffers == 1 && any) {
                SplitQueries<kHeadDim, kN> split;
                split.open(p.query + (static_cast<uint64_t>(first_row) * p.query_heads + walk.head * group) * kHeadDim + lane % (kHeadDim / 8) * 8, queries, group, p.query_heads, warp - 4, 4 * S::kGroups, lane);
                if (!warp_look_suspended(query_empty, (pair & 1) ^ 1, abort_flag, status, kStatusQuery)) break;
                split.run(query_smem, st->query_scale[0], lane);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(query_full);
            }
            if (any && !warp_look_suspended(query_full + 8 * query_buffer, (S::kQueryBuffers == 2 ? pair >> 1 : pair) & 1, abort_flag, status, kStatusQuery)) break;
            const int32_t seen_by_all = static_cast<int32_t>(walk.length) - static_cast<int32_t>(walk.tokens) + 1;
            float sum[kBlock];   // this thread's part of the denominators
#pragma unroll
            for (uint32_t i = 0; i < kBlock; ++i) sum[i] = 0.0f;
            // A tile's pages and scales, asked for while the warps wait for one another over the tile before.
            uint32_t next_there = 0, next_bytes = 0;
            auto fetch = [&](uint32_t t) {
                const uint32_t at = t % kTileInfos;
                if (!warp_look_suspended(scales_full + 8 * at, t / kTileInfos & 1, abort_flag, status, kStatusScores)) return false;
                next_there = st->info[at], next_bytes = st->scales[at][thread];
                return true;
            };
            if (any && !fetch(tile)) break;
            for (uint32_t key = walk.key; key < walk.key_end; key += kTile, ++tile) {
                const uint32_t buffer = tile & 1, there = next_there;
                const uint32_t count = walk.key_end - key < kTile ? walk.key_end - key : kTile;
                const bool whole = count == kTile && there == all_boxes, masked = !whole || static_cast<int32_t>(key + kTile) > seen_by_all;
                const bool my_key = thread < count && (there >> (thread >> box_shift) & 1);
                const uint32_t bytes = my_key ? next_bytes : 0x7f7fu, key_byte = scale_byte(bytes & 0xff), value_byte = scale_byte(bytes >> 8);
                const float key_scale = (bytes & 0xff) == 0xff ? __uint_as_float(0x7fc00000u) : __uint_as_float(key_byte << 23) * p.scale_log2;
                const float value_power = bytes >> 8 == 0xff ? __uint_as_float(0x7fc00000u) : static_cast<float>(static_cast<int32_t>(value_byte) - 127);
                const float value_inverse = __uint_as_float((254 - 60 - value_byte) << 23);   // 2^-60 of it, which the total makes up for
                // 16 queries' s + f of this thread's key. More than 16 queries are gone through 16 at a time, in rolled loops, from tensor memory each time; up to 16
                // queries' stay in registers.
                float s[kBlock];
                auto scores = [&](uint32_t c0) {
                    load_columns<kBlock>(tmem + lanes + buffer * S::kScores + c0, reinterpret_cast<uint32_t*>(s));
                    float scale[kBlock];
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; i += 4) *reinterpret_cast<float4*>(scale + i) = *reinterpret_cast<const float4*>(query_scale + c0 + i);
                    tc_wait_ld();
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) s[i] = fmaf(s[i] * scale[i], key_scale, value_power);
                    if (masked) {
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) s[i] = my_key && static_cast<int32_t>(key + thread) < st->limit[c0 + i] ? s[i] : -INFINITY;
                    }
                };
                // Their weights under the references as they stand, and whether one of them would pass 2^kRoom (it is held there).
                auto weights = [&](uint32_t c0, float (&w)[kBlock]) {
                    bool passes = false;
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; i += 4) *reinterpret_cast<float4*>(w + i) = *reinterpret_cast<const float4*>(st->minus + c0 + i);
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) {
                        w[i] += s[i];
                        passes |= w[i] > kRoom + kLift;
                        asm("min.NaN.f32 %0, %0, %1;" : "+f"(w[i]) : "f"(kRoom + kLift));
                    }
                    return passes;
                };
                if (!warp_look_suspended(weights_empty + 8 * buffer, (tile >> 1 & 1) ^ 1, abort_flag, status, kStatusProduct) ||
                    !warp_look_suspended(scores_full + 8 * buffer, tile >> 1 & 1, abort_flag, status, kStatusScores)) {
                    alive = false;
                    break;
                }
                tc_fence_after();
                if (kOneBlock) scores(first);
                // The weights are formed and stored under the references as they stand, and stand if no warp finds one that passes 2^kRoom; else the references
                // move and the weights are formed anew. (Asked first and formed then, a tile of eight queries took 400 cycles more, which the warps waited for one another.)
                bool move = key == walk.key;   // a pair's first tile sets the references
                for (bool again = false;; again = true) {
                    if (move) {
                        if (again) {   // the sums as they were
#pragma unroll 1
                            for (uint32_t c = first; c < behind; c += kBlock) {
                                if (!kOneBlock) scores(c);
                                float w[kBlock];
                                weights(c, w);
#pragma unroll
                                for (uint32_t i = 0; i < kBlock; ++i) w[i] = exp2_fast(w[i]);
                                if constexpr (kOneBlock) {
#pragma unroll
                                    for (uint32_t i = 0; i < kBlock; ++i) sum[i] = fmaf(-w[i], value_inverse, sum[i]);
                                } else {
#pragma unroll
                                    for (uint32_t i = 0; i < kBlock; i += 4) {
                                        float4& x = sum_smem[(c + i) / 4 * kTile + thread];
                                        x = make_float4(fmaf(-w[i], value_inverse, x.x), fmaf(-w[i + 1], value_inverse, x.y), fmaf(-w[i + 2], value_inverse, x.z), fmaf(-w[i + 3], value_inverse, x.w));
                                    }
                                }
                            }
                        }
                        // The references move up to the largest so far.
#pragma unroll 1
                        for (uint32_t c = first; c < behind; c += kBlock) {
                            if (!kOneBlock) scores(c);
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
                        if (thread < S::kMine) {
                            const float old = st->reference[mine];
                            const float4 w = st->wide[mine];
                            const float now = fmaxf(fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)), old);
                            // What the sums shrink by, in two factors: denominators of values of small scales still count where 2^(old - now) is zero.
                            st->factor[0][mine] = now == old ? 1.0f : exp2_fast(fmaxf(old - now, kFar));
                            st->factor[1][mine] = now == old ? 1.0f : exp2_fast(fminf(old - now - kFar, 0.0f));
                            st->reference[mine] = now;
                            st->minus[mine] = now == -INFINITY ? kNoReference : kLift - now;
                        }
                        if (!meet()) {
                            alive = false;
                            break;
                        }
                        if (again) {
                            if (!warp_look_suspended(weights_empty + 8 * (buffer ^ 1), (tile - 1) >> 1 & 1, abort_flag, status, kStatusProduct)) {
                                alive = false;
                                break;
                            }
                            tc_fence_after();
#pragma unroll 1
                            for (uint32_t part = 0, far = 0; part <= far; ++part) {   // by the second factor where the first is its least
#pragma unroll 1
                                for (uint32_t c = first; c < behind; c += kBlock) {   // 16 queries' columns (or eight), if one of them has moved
                                    float factor[kBlock];
                                    bool moved = false;
#pragma unroll
                                    for (uint32_t i = 0; i < kBlock; ++i) factor[i] = st->factor[part][c + i], moved |= factor[i] != 1.0f, far |= factor[i] <= kFarFactor;
                                    if (!moved) continue;
#pragma unroll 1
                                    for (uint32_t column = c; column < S::kChunks * S::kTerms; column = column % S::kTerms + kN < 3 * kN ? column + kN : column / S::kTerms * S::kTerms + S::kTerms + c) {
                                        uint32_t v[kBlock];
                                        load_columns<kBlock>(tmem_out + lanes + column, v);
                                        tc_wait_ld();
#pragma unroll
                                        for (uint32_t i = 0; i < kBlock; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * factor[i]);
                                        store_columns<kBlock>(tmem_out + lanes + column, v);
                                    }
                                    if constexpr (kOneBlock) {
#pragma unroll
                                        for (uint32_t i = 0; i < kBlock; ++i) sum[i] *= factor[i];
                                    } else {
#pragma unroll
                                        for (uint32_t i = 0; i < kBlock; i += 4) {
                                            float4& x = sum_smem[(c + i) / 4 * kTile + thread];
                                            x = make_float4(x.x * factor[i], x.y * factor[i + 1], x.z * factor[i + 2], x.w * factor[i + 3]);
                                        }
                                    }
                                }
                                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                            }
                            tc_fence_before();
                        }
                    }
                    // a key's row of a column's atom, and the halves of it in the 32-byte swizzle
                    uint8_t* const to_weights = weight_smem + buffer * S::kWeightBytes + thread * 32;
                    const uint32_t turned = (thread & 7) >> 2;
                    auto store = [&](uint32_t column, uint4 sixteen) { *reinterpret_cast<uint4*>(to_weights + column / 32 * kWeightAtom + ((column / 16 % 2 ^ turned) << 4)) = sixteen; };
                    bool passes = false;
#pragma unroll 1
                    for (uint32_t c = first; c < behind; c += kBlock) {
                        if (!kOneBlock) scores(c);
                        if constexpr (!kOneBlock) {
                            if (key != walk.key) {
#pragma unroll
                                for (uint32_t i = 0; i < kBlock; i += 4) *reinterpret_cast<float4*>(sum + i) = sum_smem[(c + i) / 4 * kTile + thread];
                            } else {
#pragma unroll
                                for (uint32_t i = 0; i < kBlock; ++i) sum[i] = 0.0f;
                            }
                        }
                        float w[kBlock];
                        passes |= weights(c, w);
                        if (!move && c + kBlock == behind) {   // say so, and go on
                            passes = __any_sync(0xffffffffu, passes);
                            if (lane == 0) reinterpret_cast<uint8_t*>(&st->needs[half][buffer])[quadrant] = passes;
                            come();
                        }
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) w[i] = exp2_fast(w[i]);
                        constexpr float kDown = 1.0f / (1ull << (static_cast<int>(kLift) - kTop));
                        uint32_t term[3][kBlock / 4];   // four codes each
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; i += 4) {
                            uint16_t code[3][2];
#pragma unroll
                            for (uint32_t j = 0; j < 2; ++j) {
                                uint32_t x = half2_of(w[i + 2 * j] * kDown, w[i + 2 * j + 1] * kDown);
                                code[0][j] = term_of(x);
                                x = rest16(x, halves_of_term(code[0][j]));
                                code[1][j] = term_of(x);
                                code[2][j] = term_of(rest16(x, halves_of_term(code[1][j])));
                            }
#pragma unroll
                            for (uint32_t t = 0; t < 3; ++t) term[t][i / 4] = code[t][0] | static_cast<uint32_t>(code[t][1]) << 16;
                        }
                        if constexpr (kBlock == 16) {
#pragma unroll
                            for (uint32_t t = 0; t < 3; ++t) store(t * kN + c, make_uint4(term[t][0], term[t][1], term[t][2], term[t][3]));
                        } else if constexpr (kN == 8) {
                            store(0, make_uint4(term[0][0], term[0][1], term[1][0], term[1][1]));
                            store(16, make_uint4(term[2][0], term[2][1], 0, 0));
                        } else {
#pragma unroll
                            for (uint32_t t = 0; t < 3; ++t) {
                                const uint32_t column = t * kN + c;
                                *reinterpret_cast<uint2*>(to_weights + column / 32 * kWeightAtom + ((column / 16 % 2 ^ turned) << 4) + column % 16) = make_uint2(term[t][0], term[t][1]);
                            }
                        }
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) sum[i] = fmaf(w[i], value_inverse, sum[i]);
                        if constexpr (!kOneBlock) {
#pragma unroll
                            for (uint32_t i = 0; i < kBlock; i += 4) sum_smem[(c + i) / 4 * kTile + thread] = *reinterpret_cast<const float4*>(sum + i);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    if (!again && key + kTile < walk.key_end && !fetch(tile + 1)) {
                        alive = false;
                        break;
                    }
                    if (move) break;
                    if (!all_came()) {
                        alive = false;
                        break;
                    }
                    move = *const_cast<volatile uint32_t*>(&st->needs[half][buffer]) != 0;
                    if (!move) break;
                }
                if (!alive) break;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(scores_empty + 8 * buffer);
                if (!whole) {
                    // Rows of V that are no token's are multiplied with weights of zero: whatever lies there, they must be numbers.
                    // These warps do not wait for every use of a slot, so they must not be more than one ahead: the tile before has to be through.
                    if (tile && !warp_look_suspended(weights_empty + 8 * (buffer ^ 1), (tile - 1) >> 1 & 1, abort_flag, status, kStatusProduct)) {
                        alive = false;
                        break;
                    }
                    const uint32_t use = S::kChunks * tile;
                    uint32_t slot = S::kKeySlots + use % S::kValueSlots, phase = use / S::kValueSlots & 1;
                    for (uint32_t c = 0; alive && c < S::kChunks; ++c) {
                        if (!warp_look_suspended(full + 8 * slot, phase, abort_flag, status, kStatusValues)) {
                            alive = false;
                            break;
                        }
                        if (half == 0 && !my_key && thread < (count + 31) / 32 * 32) {
                            uint4* row = reinterpret_cast<uint4*>(smem + slot * kSlotBytes + thread * 128);
#pragma unroll
                            for (uint32_t i = 0; i < 8; ++i) row[i] = make_uint4(0, 0, 0, 0);
                        }
                        if (++slot == S::kSlots) slot = S::kKeySlots, phase ^= 1;
                    }
                    if (!alive) break;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(weights_full + 8 * buffer);
            }
            if (!alive) break;
            // ---- the pair's output, or its part ----
            if (any) {
                if (lane == 0) mbar_arrive(query_empty + 8 * query_buffer);
                ++pair;
                // The denominators: over the lanes, halving the queries that a lane holds as long as it holds more than one, then over the warps.
#pragma unroll 1
                for (uint32_t c = first; c < behind; c += kBlock) {
                    if constexpr (!kOneBlock) {
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; i += 4) *reinterpret_cast<float4*>(sum + i) = sum_smem[(c + i) / 4 * kTile + thread];
                    }
                    uint32_t query = 0;
#pragma unroll
                    for (uint32_t step = 16, held = kBlock / 2; step; step /= 2, held /= 2) {
                        const bool upper = lane & step;
                        if (held) {
#pragma unroll
                            for (uint32_t i = 0; i < kBlock / 2; ++i) {
                                if (i < held) {
                                    const float give = upper ? sum[i] : sum[i + held], keep = upper ? sum[i + held] : sum[i];
                                    sum[i] = keep + __shfl_xor_sync(0xffffffffu, give, step);
                                }
                            }
                            if (upper) query += held;
                        } else {
                            sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], step);
                        }
                    }
                    if (lane % (32 / kBlock) == 0) reinterpret_cast<float*>(&st->wide[c + query])[quadrant] = sum[0];
                }
                if (!meet()) break;
                if (thread < S::kMine) st->total[mine] = ((st->wide[mine].x + st->wide[mine].y) + (st->wide[mine].z + st->wide[mine].w)) * static_cast<float>(1ull << (60 + kTop - static_cast<int>(kLift)));
                if (!meet()) break;
                if (!warp_look_suspended(weights_empty + 8 * ((tile - 1) & 1), (tile - 1) >> 1 & 1, abort_flag, status, kStatusProduct)) break;
                tc_fence_after();
            }
            const bool alone = walk.starts && walk.ends;
            const uint32_t part = 2 * blockIdx.x + (walk.starts ? 1 : 0);
            float* const part_out = p.parts + static_cast<uint64_t>(part) * kN * kHeadDim + thread;
            __nv_bfloat16* const out = p.output + (static_cast<uint64_t>(first_row) * p.query_heads + walk.head * group) * kHeadDim + thread;
            const uint32_t next_token = (p.query_heads - group) * kHeadDim;   // from behind a token's queries to the next token's
            float2* const stats = reinterpret_cast<float2*>(p.parts + static_cast<uint64_t>(2 * p.spans) * kN * kHeadDim) + part * kN;
            uint32_t token_end = (first / group + 1) * group;
            uint64_t skipped = static_cast<uint64_t>(first / group) * next_token;
            auto write = [&](const uint32_t (&v)[S::kChunks][kBlock], uint32_t c0, uint32_t i) {
                const uint32_t c = c0 + i;
                if (c == token_end) token_end += group, skipped += next_token;
                const float all = any ? st->total[c] : 0.0f;
                float scale;
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(scale) : "f"(all));   // good to 2^-23
#pragma unroll
                for (uint32_t h = 0; h < S::kChunks; ++h) {
                    out[skipped + c * kHeadDim + h * 128] = __float2bfloat16_rn(all == 0.0f ? 0.0f : __uint_as_float(v[h][i]) * scale);
                }
            };
#pragma unroll 1
            for (uint32_t c0 = first; c0 < (queries < behind ? queries : behind); c0 += kBlock) {
                uint32_t v[S::kChunks][kBlock], middle[S::kChunks][kBlock], low[S::kChunks][kBlock];   // the terms' sums
#pragma unroll
                for (uint32_t h = 0; h < S::kChunks; ++h) {
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) v[h][i] = 0;
                }
                if (any) {
#pragma unroll
                    for (uint32_t h = 0; h < S::kChunks; ++h) {
                        load_columns<kBlock>(tmem_out + lanes + h * S::kTerms + c0, v[h]);
                        load_columns<kBlock>(tmem_out + lanes + h * S::kTerms + kN + c0, middle[h]);
                        load_columns<kBlock>(tmem_out + lanes + h * S::kTerms + 2 * kN + c0, low[h]);
                    }
                    tc_wait_ld();
#pragma unroll
                    for (uint32_t h = 0; h < S::kChunks; ++h) {
#pragma unroll
                        for (uint32_t i = 0; i < kBlock; ++i) {
                            v[h][i] = __float_as_uint(fmaf(fmaf(__uint_as_float(low[h][i]), 0.0625f, __uint_as_float(middle[h][i])), 0.0625f, __uint_as_float(v[h][i])));
                        }
                    }
                }
                if (!alone) {
                    float* const to = part_out + c0 * kHeadDim;
#pragma unroll
                    for (uint32_t i = 0; i < kBlock; ++i) {
#pragma unroll
                        for (uint32_t h = 0; h < S::kChunks; ++h) to[i * kHeadDim + h * 128] = __uint_as_float(v[h][i]);
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
            if (!alone && thread < S::kMine && mine < queries) {
                // A part all of whose scores are NaN or -infinity has the reference -infinity too, but counts: its sums may be NaN.
                float2 stat = make_float2(st->reference[mine], any ? st->total[mine] : 0.0f);
                if (stat.x == -INFINITY && st->limit[mine] > static_cast<int32_t>(walk.key)) stat.x = kNoNumber;
                stats[mine] = stat;
            }
            if (any) tc_fence_before();
            if (!alone) {
                if (walk.starts) {
                    const uint32_t units = st->units[walk.sequence + 1] - st->units[walk.sequence], longer = extra * (base + 1);
                    const uint32_t last = st->units[walk.sequence] * p.kv_heads + (walk.head + 1) * units - p.pair_units - 1;   // the pair's last unit
                    record.row = first_row, record.tokens = walk.tokens, record.head = walk.head, record.first = blockIdx.x;
                    record.last = last < longer ? last / (base + 1) : extra + (last - longer) / base;
                }
            }
            if (p.joins < p.spans && walk.starts && thread == 0 && half == 0) p.records[walk.sequence * p.kv_heads + walk.head] = alone ? JoinRecord{} : record;
        }
        if (p.joins == p.spans && thread == 0 && half == 0) p.records[blockIdx.x] = record;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmem) : "memory");
    }
}

template <uint32_t kHeadDim, uint32_t kN>
void launch_attention(cudaStream_t stream, const CUtensorMap& keys, const CUtensorMap& values, const AttentionParams& p) {
    launch_dependent(stream, paged_attention_e4m3_kernel<kHeadDim, kN>, p.spans, ShapeE4m3<kHeadDim, kN>::kThreads, ShapeE4m3<kHeadDim, kN>::kSmem, keys, values, p);
    launch_join<kHeadDim, kN>(stream, p);
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
    cudaError_t e = cudaFuncSetAttribute(paged_attention_e4m3_kernel<kHeadDim, 8>, kSmem, ShapeE4m3<kHeadDim, 8>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_e4m3_kernel<kHeadDim, 16>, kSmem, ShapeE4m3<kHeadDim, 16>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_e4m3_kernel<kHeadDim, 32>, kSmem, ShapeE4m3<kHeadDim, 32>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_e4m3_kernel<kHeadDim, 48>, kSmem, ShapeE4m3<kHeadDim, 48>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_e4m3_kernel<kHeadDim, 64>, kSmem, ShapeE4m3<kHeadDim, 64>::kSmem);
    return e;
}

}  // namespace

cudaError_t attention_e4m3_configure_device() {
    const cudaError_t e = configure<128>();
    return e == cudaSuccess ? configure<256>() : e;
}

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
    const uint32_t columns = query_columns(a->query_heads, a->layer.kv_heads, a->max_new_tokens);
    // A pair's beginning and end take about 2 us where a unit of head size 256 streams in 0.7 us, of 128 in 0.4; of many queries about 6 us. (64 ragged sequences, spans of as
    // many units each: those of one pair done after 72 us, those of six after 84.)
    p.pair_units = columns > 16 ? 8 : a->layer.head_dim == 256 ? 3 : 5;
    const uint32_t head_dim = a->layer.head_dim, box = a->layer.page_tokens < kUnit ? a->layer.page_tokens : kUnit;
    const uint64_t cache_rows = static_cast<uint64_t>(a->layer.pages) * a->layer.kv_heads * a->layer.page_tokens;
    CUtensorMap keys, values;   // rows of head_dim bytes, as a map of packed codes with twice the columns
    if (!make_code_map(&keys, a->layer.keys, cache_rows, head_dim * 2, box) || !make_code_map(&values, a->layer.values, cache_rows, head_dim * 2, box)) {
        return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE);
    }
    auto launch = head_dim == 256 ? launch_of<256>(columns) : launch_of<128>(columns);
    launch(s->stream, keys, values, p);
    return submitted();
}
