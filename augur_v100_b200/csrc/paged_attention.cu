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
#include "paged_attention.cuh"

namespace augur_sm100 {
namespace {

constexpr uint32_t kOnesBytes = kTile * 32;    // 16 k of ones, as the 128-row operand
constexpr uint32_t kInfos = 8;                 // tiles that the loader is ahead of the softmax at most, rounded up

static_assert(sizeof(augur_cuda_nvfp4_sm100_paged_attention_args_v1) == 160, "attention ABI");

// Small state of a CTA, behind the rings, the queries and the weights.
struct State : BatchState {
    uint64_t full[16], empty[16];
    uint64_t scores_full[2], scores_empty[2], weights_full[2], weights_empty[2], query_full[2], query_empty[2], group, keys_first;
    uint32_t tmem, abort[1 + kThreads / 32];
    uint32_t needs[2];                 // a byte per softmax warp: a reference has to move
    uint32_t info[kInfos];             // of a tile: pages that are there, a bit per box
    float reference[kMaxQueries], factor[kMaxQueries];
    float4 wide[kMaxQueries];          // the largest score per query and softmax warp
    int32_t limit[kMaxQueries];        // keys that a query sees
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
    scan_units(st, p, warp, lane);
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

template <uint32_t kHeadDim, uint32_t kN>
void launch_attention(cudaStream_t stream, const CUtensorMap& keys, const CUtensorMap& values, const AttentionParams& p) {
    launch_dependent(stream, paged_attention_kernel<kHeadDim, kN>, p.spans, kThreads, Shape<kHeadDim, kN>::kSmem, keys, values, p);
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
    cudaError_t e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 8>, kSmem, Shape<kHeadDim, 8>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 16>, kSmem, Shape<kHeadDim, 16>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 32>, kSmem, Shape<kHeadDim, 32>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 48>, kSmem, Shape<kHeadDim, 48>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(paged_attention_kernel<kHeadDim, 64>, kSmem, Shape<kHeadDim, 64>::kSmem);
    return e;
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
    AttentionParams p = attention_params(plan, a);
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
