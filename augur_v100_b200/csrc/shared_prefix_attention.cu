// Attention of a step's new tokens over a paged BF16 cache whose sequences share a prefix, on sm_100a.
//
//   o = (sum over the prefix + sum over a row's own tokens) of 2^(s_j - m) v_j, over the same sum of 2^(s_j - m),  s_j = scale log2(e) q . k_j
//
// The prefix's keys and values are the same for every row, so its part is two dense products of all rows' queries: 4 head_dim operations
// per query and token against 4 head_dim bytes per token, that is: bound by HBM up to some 250 queries of a key-value head, by the matrix units and what
// feeds them above. Three launches: the rows' own tokens, in small CTAs (own_attention_kernel); the prefix; the join of both.
//
// For the prefix a CTA takes 128 queries of a key-value head (token rows x the heads that share it, packed) through a run of its tiles:
//
//   S[query][key]  = Q K^T           both from shared memory, S in tensor memory
//   O[query][dim] += P V             P from tensor memory, where it takes the place of the S that it came from; V as it lies in the pages (MN-major)
//
// A softmax thread holds one query, so nothing of the softmax passes between threads. Its reference maximum moves when a score passes it by more than 2^8 (then
// O is scaled in tensor memory). P is one BF16 term (2^-8 of each weight at most; the denominator sums the same terms): a second one would
// cost half as much again of the product that bounds the kernel.
//
// Head size 256: one group of softmax warps, 128 keys a tile, two S; 2800 cycles a tile where the products alone take 2048 (84 GB/s and SM from L2): a tile's scores wait for the
// product of two tiles before, whose P lies in their place, and that for 2050 cycles of softmax, 1024 of them exponentials; and Q and K of the first product are both read from
// shared memory, 128 bytes a cycle with the copies coming in.
// Head size 128: two groups that take tiles of 64 keys in turn, each with an O and two S of its own: one group's exponentials take as long as a tile's products.
// Twelve sequences of eight tokens on 65536 tokens (24 / 4 heads of 256): 160 to 165 us in bursts of some ms (0.94 to 0.97 PFLOP/s), 188 to 194 without a pause, where the power cap leaves
// 1537 MHz (0.81).
#include "paged_attention.cuh"

namespace augur_sm100 {

namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_shared_prefix_attention_args_v1) == 192, "attention ABI");

constexpr uint32_t kRowsM = 128;               // queries of a CTA
constexpr uint32_t kRounds = 3;                // a device's worth of CTAs, at most so many times, where the prefix is split for it
constexpr uint32_t kMaxSplit = 256, kMaxChunks = 32;   // of the prefix, and of a sequence's own tokens
constexpr uint32_t kInfoRing = 16, kMaxSlots = 12, kMaxBuffers = 4;
constexpr uint32_t kStatusPrefixLoad = 0x421, kStatusPrefixMma = 0x422, kStatusPrefixScores = 0x423, kStatusPrefixQuery = 0x424, kStatusPrefixProduct = 0x425, kStatusPrefixInfo = 0x426;

struct PrefixParams {
    AttentionParams a;
    const int32_t *prefix_table, *prefix_tokens;
    float* parts;              // [items][streams][head_dim / 4][kRowsM][4], then [items][streams][kRowsM] (reference maximum, denominator)
    float* own_parts;          // [rows][query_heads][chunks][head_dim]
    float2* own_stats;         // [rows][query_heads][chunks]
    uint32_t prefix_pages;
    uint32_t max_items;        // that there is room for
    uint32_t tiles;            // of kRowsM queries
    uint32_t chunks;           // that the tokens of a sequence are cut into
};

// The shared tokens that are read from the prefix's pages: whole pages, as many as there are.
__device__ __forceinline__ uint32_t shared_tokens(const PrefixParams& p) {
    const int32_t tokens = *p.prefix_tokens;
    const uint32_t whole = tokens > 0 ? static_cast<uint32_t>(tokens) >> p.a.page_shift : 0;
    return (whole < p.prefix_pages ? whole : p.prefix_pages) << p.a.page_shift;
}

template <uint32_t kHeadDim>
struct PrefixShape {
    static constexpr uint32_t kParts = kHeadDim / 128, kStreams = kHeadDim == 128 ? 2 : 1;
    // Keys of a tile, and S in tensor memory: 256 columns of it. With two streams each has two, so that the next scores are formed while its softmax is at work (of 128 keys
    // and one each, the weights' product and the next scores behind it were waited for: 2300 cycles a tile. What bounds it now with pages of 16 tokens is
    // the copies' issue, 100 cycles each: 1120 cycles for 64 keys).
    static constexpr uint32_t kKeys = kHeadDim == 128 ? 64 : 128, kBuffers = 256 / kKeys, kSlot = kKeys * 256;   // a slot: 128 dims of a tile, as two halves of 128 bytes a key
    static constexpr uint32_t kThreads = 128 + 128 * kStreams;   // warp 0 loads keys, 1 and 2 MMA, 3 values, then the softmax
    static constexpr uint32_t kQueryBytes = kRowsM * kHeadDim * 2, kSlots = (224 * 1024 - kQueryBytes) / kSlot;
    // A ring each for the keys and the values, so that two warps deal out the copies: one alone took 80 cycles a copy, and pages of 16 tokens are up to 16 copies a slot.
    static constexpr uint32_t kValueSlots = kSlots / 2, kKeySlots = kSlots - kValueSlots;
    static constexpr uint32_t kSmem = 1024 + kQueryBytes + kSlots * kSlot + 1024;
    static constexpr uint32_t kScoresAt = 0, kOutAt = 256;       // tensor memory: S, then one O per stream
    static_assert(kSlots <= kMaxSlots && kKeySlots / kParts + kBuffers + 1 <= kInfoRing && kKeySlots >= kParts && kValueSlots >= kParts && kSmem <= kSmemLimit && kOutAt + kStreams * kHeadDim == 512, "a CTA's memory");
};

struct PrefixState {
    uint64_t full[kMaxSlots], empty[kMaxSlots], scores_full[kMaxBuffers], weights_full[kMaxBuffers], products[kMaxBuffers], query_full, query_empty, info_full[kInfoRing];
    uint32_t tmem, abort[1 + 12], info[kInfoRing];
};
static_assert(sizeof(PrefixState) <= 1024, "the state's room");

// An item is 128 queries of a key-value head over a `split`-th of the prefix's tiles. Items are dealt out round by round, those of the same keys next to one
// another, so that the keys come from L2 for all but the first.
struct Items {
    uint32_t key_tiles, split, tokens;
    uint32_t count;
    __device__ __forceinline__ void locate(const PrefixParams& p, uint32_t item, uint32_t* head, uint32_t* tile, uint32_t* first, uint32_t* last) const {
        const uint32_t rest = item / p.tiles;
        *tile = item - rest * p.tiles;
        *head = rest / split;
        const uint32_t part = rest - *head * split;
        *first = part * key_tiles / split, *last = (part + 1) * key_tiles / split;   // (at most 2^8 * 2^18)
    }
};
// The split that a simple model takes for quickest: rounds of items, each its keys and 512 for beginning and end, and four keys for every part to be joined. A warp together.
template <uint32_t kKeys>
__device__ __forceinline__ Items items_of(const PrefixParams& p, uint32_t ctas) {
    Items x;
    x.tokens = shared_tokens(p);
    x.key_tiles = (x.tokens + kKeys - 1) / kKeys;
    const uint32_t pairs = p.a.kv_heads * p.tiles, room = p.max_items / pairs;
    uint32_t most = x.key_tiles < room ? x.key_tiles : room;
    most = most < kMaxSplit ? most : kMaxSplit;
    uint64_t best = UINT64_MAX;
    for (uint32_t split = 1 + threadIdx.x % 32; split <= most; split += 32) {
        const uint32_t items = pairs * split;   // at most max_items
        const uint64_t cost = static_cast<uint64_t>((items + ctas - 1) / ctas) * ((x.key_tiles + split - 1) / split + 512 / kKeys) * kKeys + items * 4, key = cost << 16 | split;
        if (key < best) best = key;
    }
#pragma unroll
    for (uint32_t step = 16; step; step /= 2) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, best, step);
        if (other < best) best = other;
    }
    x.split = x.key_tiles ? static_cast<uint32_t>(best & 0xffff) : 1;
    x.count = x.key_tiles ? pairs * x.split : 0;
    return x;
}

// Up to four MMAs of 16 k, the 128-row operand from tensor memory (8 columns a step), the narrow one kStep (of 16 bytes) further each time.
template <uint32_t kStep>
__device__ __forceinline__ void mma_block_from_tmem(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n.reg .pred e, p, q;\n.reg .b64 b0, b1, b2, b3;\n.reg .b32 l1, l2, l3, m1, m2, m3;\n"
        "elect.sync _|e, 0xffffffff;\nsetp.ne.b32 p, %4, 0;\nsetp.eq.u32 q, 0, 0;\n"
        "add.s32 l1, %1, 8;\nadd.s32 l2, %1, 16;\nadd.s32 l3, %1, 24;\nadd.s32 m1, %2, %6;\nadd.s32 m2, m1, %6;\nadd.s32 m3, m2, %6;\n"
        "mov.b64 b0, {%2, %5};\nmov.b64 b1, {m1, %5};\nmov.b64 b2, {m2, %5};\nmov.b64 b3, {m3, %5};\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b0, %3, p;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [l1], b1, %3, q;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [l2], b2, %3, q;\n"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [l3], b3, %3, q;\n}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(kHighSwizzled), "n"(kStep)
        : "memory");
}

// Two F32 operations in one instruction: x * scale + shift, and sums.
__device__ __forceinline__ void fma2(uint32_t& x0, uint32_t& x1, float scale, float shift) {
    asm("{\n.reg .b64 x, a, b;\nmov.b64 x, {%0, %1};\nmov.b64 a, {%2, %2};\nmov.b64 b, {%3, %3};\nfma.rn.ftz.f32x2 x, x, a, b;\nmov.b64 {%0, %1}, x;\n}"
        : "+r"(x0), "+r"(x1)
        : "r"(__float_as_uint(scale)), "r"(__float_as_uint(shift)));
}
__device__ __forceinline__ void add2(float& x0, float& x1, uint32_t y0, uint32_t y1) {
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%0, %1};\nmov.b64 y, {%2, %3};\nadd.rn.ftz.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}" : "+f"(x0), "+f"(x1) : "r"(y0), "r"(y1));
}

template <uint32_t kHeadDim>
__global__ void __launch_bounds__(PrefixShape<kHeadDim>::kThreads, 1)
prefix_attention_kernel(const __grid_constant__ CUtensorMap map_keys, const __grid_constant__ CUtensorMap map_values, const __grid_constant__ PrefixParams p) {
    using S = PrefixShape<kHeadDim>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* const query_smem = smem + S::kSlots * S::kSlot;
    PrefixState* const st = reinterpret_cast<PrefixState*>(query_smem + S::kQueryBytes);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = smem_u32(st->full), empty = smem_u32(st->empty), scores_full = smem_u32(st->scores_full), weights_full = smem_u32(st->weights_full);
    const uint32_t products = smem_u32(st->products), query_full = smem_u32(&st->query_full), query_empty = smem_u32(&st->query_empty), info_full = smem_u32(st->info_full);
    volatile uint32_t* abort_flag = st->abort;
    uint32_t* const status = p.a.status_word;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < S::kSlots; ++s) mbar_init(full + 8 * s, 1), mbar_init(empty + 8 * s, 1);
        for (uint32_t b = 0; b < S::kBuffers; ++b) mbar_init(scores_full + 8 * b, 1), mbar_init(weights_full + 8 * b, 4), mbar_init(products + 8 * b, 1);
        for (uint32_t i = 0; i < kInfoRing; ++i) mbar_init(info_full + 8 * i, 1);
        mbar_init(query_full, 4 * S::kStreams), mbar_init(query_empty, 1);
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_keys) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_values) : "memory");
        for (uint32_t i = 0; i < 1 + 12; ++i) st->abort[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&st->tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Everything above runs while the launch before this one drains; from here on its results are read.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Items items = items_of<S::kKeys>(p, gridDim.x);
    if (blockIdx.x == 0 && threadIdx.x == 0 && *p.prefix_tokens > static_cast<int32_t>(p.prefix_pages << p.a.page_shift)) atomicCAS(status, 0u, kStatusPage);
    // Does any row end within the prefix?
    bool ends_within = false;
    const int32_t room = static_cast<int32_t>(p.a.table_pages << p.a.page_shift);   // a length beyond the table counts as the table's
    for (uint32_t b = threadIdx.x; b < p.a.sequences; b += S::kThreads) {
        const int32_t from = p.a.token_starts[b], to = p.a.token_starts[b + 1];
        ends_within |= to > from && static_cast<int64_t>(min(p.a.lengths[b], room)) - to + from + 1 < static_cast<int64_t>(items.tokens);
    }
    ends_within = __syncthreads_or(ends_within);
    const uint32_t tmem = st->tmem, group = p.a.query_heads / p.a.kv_heads, all_queries = p.a.rows * group;   // (of a key-value head; below 2^26)

    if (warp == 0 || warp == 3) {
        // ---------------- pages: warp 0 the keys, warp 3 the values ----------------
        const uint32_t box_shift = p.a.page_shift < 6 ? p.a.page_shift : 6, boxes = S::kKeys >> box_shift, box_bytes = 128u << box_shift;
        const uint32_t beyond = (p.a.pages * p.a.kv_heads) << p.a.page_shift;   // a row behind the cache: TMA reads zeros there
        const CUtensorMap* const map = warp == 0 ? &map_keys : &map_values;
        const uint32_t first_slot = warp == 0 ? 0 : S::kKeySlots, end_slot = warp == 0 ? S::kKeySlots : S::kSlots;
        uint32_t slot = first_slot, phase = 1, count = 0;
        bool alive = true;
        for (uint32_t item = blockIdx.x; alive && item < items.count; item += gridDim.x) {
            uint32_t head, tile, first, last;
            items.locate(p, item, &head, &tile, &first, &last);
            auto page_of = [&](uint32_t t) {
                const uint32_t key = t * S::kKeys + ((lane % boxes) << box_shift);   // (the second half of a slot by the lanes behind)
                return t < last && lane < 2 * boxes && key < items.tokens ? __ldg(p.prefix_table + (key >> p.a.page_shift)) : INT32_MIN;
            };
            int32_t page = page_of(first);
            for (uint32_t t = first; alive && t < last; ++t, ++count) {
                const uint32_t key = t * S::kKeys + ((lane % boxes) << box_shift);
                const bool there = page >= 0 && static_cast<uint32_t>(page) < p.a.pages;
                if (!there && page != INT32_MIN) atomicCAS(status, 0u, kStatusPage);
                const uint32_t row = there ? ((static_cast<uint32_t>(page) * p.a.kv_heads + head) << p.a.page_shift) + (key & ((1u << p.a.page_shift) - 1)) : beyond;
                const uint32_t mask = __ballot_sync(0xffffffffu, there && lane < boxes);
                page = page_of(t + 1);
                if (warp == 0 && lane == 0) {   // (the ring is that long: a ring of keys, and the tiles whose scores are formed, ahead of the softmax)
                    st->info[count % kInfoRing] = mask;
                    mbar_arrive(info_full + 8 * (count % kInfoRing));
                }
                __syncwarp();
                for (uint32_t c = 0; c < S::kParts; ++c) {
                    if (!(alive = warp_look_suspended(empty + 8 * slot, phase, abort_flag, status, kStatusPrefixLoad))) break;
                    if (lane == 0) mbar_expect_tx(full + 8 * slot, S::kSlot);
                    __syncwarp();
                    if (lane < 2 * boxes) tma_load_2d(smem_u32(smem) + slot * S::kSlot + lane * box_bytes, map, c * 256 + (lane < boxes ? 0 : 128), row, full + 8 * slot);
                    __syncwarp();
                    if (++slot == end_slot) slot = first_slot, phase ^= 1;
                }
            }
        }
    } else if (warp == 1 || (warp == 2 && S::kStreams == 2)) {
        // ---------------- MMA issuer: S of a tile, then O of a tile before it. With two streams a warp for each: what one has to wait for, look at and say for a tile took
        // 1370 cycles for 64 keys, more than the products or the softmax. ----------------
        constexpr uint32_t idesc_any = (1u << 4) | (1u << 7) | (1u << 10) | ((kRowsM >> 4) << 24);   // F32 += BF16 x BF16
        constexpr uint32_t idesc = idesc_any | ((S::kKeys >> 3) << 17), idesc_values = idesc_any | ((128 >> 3) << 17) | (1u << 16);   // V is MN-major
        const uint32_t slots = low_word(smem_u32(smem), 16), slots_values = low_word(smem_u32(smem), S::kSlot / 2), queries = low_word(smem_u32(query_smem), 16);
        const bool forms = warp == 1, multiplies = warp == 2 || S::kStreams == 1;
        uint32_t key_slot = 0, key_phase = 0, slot = S::kKeySlots, phase = 0, scores = 0, done = 0, round = 0;
        bool alive = true;
        auto scores_of_tile = [&]() {
            const uint32_t buffer = scores % S::kBuffers;
            // S goes where the weights of kBuffers tiles before were: of this warp's own MMAs those that read them are ahead in the pipe
            if (S::kStreams == 2 && scores >= S::kBuffers && !warp_look_suspended(products + 8 * buffer, scores / S::kBuffers - 1 & 1, abort_flag, status, kStatusPrefixMma)) return false;
            for (uint32_t c = 0; c < S::kParts; ++c) {
                if (!warp_look_suspended(full + 8 * key_slot, key_phase, abort_flag, status, kStatusPrefixMma)) return false;
                tc_fence_after();
                const uint32_t d = tmem + S::kScoresAt + buffer * S::kKeys, a = queries + 2 * c * (kSlotBytes >> 4), b = slots + key_slot * (S::kSlot >> 4);
                mma_block<kHighSwizzled, 2>(d, a, b, idesc, c, 4);
                mma_block<kHighSwizzled, 2>(d, a + (kSlotBytes >> 4), b + (S::kSlot >> 5), idesc, 1, 4);
                commit(empty + 8 * key_slot);
                if (++key_slot == S::kKeySlots) key_slot = 0, key_phase ^= 1;
            }
            commit(scores_full + 8 * buffer);
            ++scores;
            return true;
        };
        auto product_of_tile = [&](bool follows) {
            const uint32_t buffer = done % S::kBuffers, d = tmem + S::kOutAt + (S::kStreams == 2 ? (done & 1) * kHeadDim : 0);
            if (!warp_look_suspended(weights_full + 8 * buffer, done / S::kBuffers & 1, abort_flag, status, kStatusPrefixProduct)) return false;
            for (uint32_t c = 0; c < S::kParts; ++c) {
                if (!warp_look_suspended(full + 8 * slot, phase, abort_flag, status, kStatusPrefixProduct)) return false;
                tc_fence_after();
                const uint32_t a = tmem + S::kScoresAt + buffer * S::kKeys, b = slots_values + slot * (S::kSlot >> 4);   // 16 keys: 8 columns of P, 16 rows of V
                mma_block_from_tmem<(16 * 128 >> 4)>(d + c * 128, a, b, idesc_values, follows);
                if (S::kKeys == 128) mma_block_from_tmem<(16 * 128 >> 4)>(d + c * 128, a + 32, b + 4 * (16 * 128 >> 4), idesc_values, 1);
                commit(empty + 8 * slot);
                if (++slot == S::kSlots) slot = S::kKeySlots, phase ^= 1;
            }
            commit(products + 8 * buffer);
            ++done;
            return true;
        };
        for (uint32_t item = blockIdx.x; alive && item < items.count; item += gridDim.x, ++round) {
            uint32_t head, tile, first, last;
            items.locate(p, item, &head, &tile, &first, &last);
            if (forms && !warp_look_suspended(query_full, round & 1, abort_flag, status, kStatusPrefixMma)) break;
            uint32_t formed = first;
            for (uint32_t t = first; alive && t < last; ++t) {
                for (; alive && forms && formed < last && (!multiplies || formed < t + S::kBuffers); ++formed) {
                    alive = scores_of_tile();
                    if (formed + 1 == last) commit(query_empty);
                }
                if (multiplies) alive = alive && product_of_tile(t >= first + S::kStreams);
            }
        }
    } else if (warp >= 4) {
        // ---------------- queries of an item, then the softmax: a query a thread ----------------
        const uint32_t stream = (warp - 4) / 4, thread = threadIdx.x & 127, lanes = ((warp & 3) * 32) << 16;
        const uint32_t box_shift = p.a.page_shift < 6 ? p.a.page_shift : 6, all_boxes = (1u << (S::kKeys >> box_shift)) - 1;
        const uint32_t out = tmem + S::kOutAt + stream * (S::kStreams == 2 ? kHeadDim : 0) + lanes;
        const float scale = p.a.scale_log2;
        uint32_t count = 0, round = 0;   // tiles and items of this CTA
        bool alive = true;
        for (uint32_t item = blockIdx.x; alive && item < items.count; item += gridDim.x, ++round) {
            uint32_t head, tile, first, last;
            items.locate(p, item, &head, &tile, &first, &last);
            // The item's queries in the 128-byte swizzle of the operand, once the products of the item before are through; past the last they are zero. (All of these warps: by
            // one alone they were there after 5.4 us.)
            if (!warp_look_suspended(query_empty, (round & 1) ^ 1, abort_flag, status, kStatusPrefixQuery)) break;
            {
                // a lane's piece of every (kWarps * 32 / kPieces)-th row; its token and the head among those that share the key-value head go along
                constexpr uint32_t kPieces = kHeadDim / 8, kWarps = 4 * S::kStreams, kStep = kWarps * 32 / kPieces;
                const uint32_t piece = lane % kPieces, row0 = ((warp - 4) * 32 + lane) / kPieces, query0 = tile * kRowsM + row0;
                uint32_t token = query0 / group, within = query0 - token * group;
                const uint32_t to = smem_u32(query_smem) + (piece >> 3) * kSlotBytes;
#pragma unroll 4
                for (uint32_t row = row0; row < kRowsM; row += kStep, within += kStep) {
                    while (within >= group) within -= group, ++token;
                    const bool live = token < p.a.rows;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                                 ::"r"(to + row * 128 + (((piece & 7) ^ (row & 7)) << 4)),
                                 "l"(p.a.query + (static_cast<uint64_t>(live ? token : 0) * p.a.query_heads + head * group + within) * kHeadDim + piece * 8), "r"(live ? 16 : 0)
                                 : "memory");
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(query_full);
            }
            // How many tokens of the prefix this row sees.
            uint32_t limit = items.tokens;
            if (ends_within) {
                const int32_t row = static_cast<int32_t>((tile * kRowsM + thread) / group);
                uint32_t low = 0, high = p.a.sequences;   // the last sequence that starts at or before the row
                while (high - low > 1) {
                    const uint32_t middle = (low + high) / 2;
                    if (p.a.token_starts[middle] <= row) low = middle;
                    else high = middle;
                }
                const int64_t seen = static_cast<int64_t>(min(p.a.lengths[low], room)) - p.a.token_starts[low + 1] + row + 1;
                limit = seen <= 0 ? 0 : seen < static_cast<int64_t>(limit) ? static_cast<uint32_t>(seen) : limit;
            }
            const uint32_t seen_by_all = __reduce_min_sync(0xffffffffu, limit);
            float reference = -INFINITY, sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            bool started = false;
            uint32_t first_key = 0;
            for (uint32_t t = first; t < last; ++t, ++count) {
                const uint32_t buffer = count % S::kBuffers;
                if (S::kStreams == 2 && (count & 1) != stream) continue;
                if (!warp_look_suspended(info_full + 8 * (count % kInfoRing), count / kInfoRing & 1, abort_flag, status, kStatusPrefixInfo) ||
                    !warp_look_suspended(scores_full + 8 * buffer, count / S::kBuffers & 1, abort_flag, status, kStatusPrefixScores)) {
                    alive = false;
                    break;
                }
                tc_fence_after();
                const uint32_t there = st->info[count % kInfoRing], key = t * S::kKeys, from = tmem + S::kScoresAt + buffer * S::kKeys + lanes;
                const bool masked = there != all_boxes || key + S::kKeys > seen_by_all;
                // Which of 32 keys from c on this row sees.
                auto seen = [&](uint32_t c) {
                    uint32_t bits = limit <= key + c ? 0 : limit - key - c >= 32 ? 0xffffffffu : (1u << (limit - key - c)) - 1;
                    if (box_shift >= 5) bits = there >> (c >> box_shift) & 1 ? bits : 0;
                    else bits &= (there >> (c >> 4) & 1 ? 0xffffu : 0) | (there >> ((c >> 4) + 1) & 1 ? 0xffff0000u : 0);
                    return bits;
                };
                uint32_t v[S::kKeys];
#pragma unroll
                for (uint32_t c = 0; c < S::kKeys; c += 32) tc_load32(from + c, reinterpret_cast<uint32_t(&)[32]>(v[c]));
                tc_wait_ld();
                if (masked) {
#pragma unroll
                    for (uint32_t c = 0; c < S::kKeys; c += 32) {
                        const uint32_t bits = seen(c);
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i) v[c + i] = bits >> i & 1 ? v[c + i] : __float_as_uint(scale < 0.0f ? INFINITY : -INFINITY);
                    }
                }
                // The largest score: of scale * S, the product with the largest S or, with a scale below zero, the smallest.
                float most;
                if (scale < 0.0f) {
                    float m[4] = {INFINITY, INFINITY, INFINITY, INFINITY};
#pragma unroll
                    for (uint32_t i = 0; i < S::kKeys; i += 2) m[i / 2 % 4] = fminf(fminf(m[i / 2 % 4], __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
                    most = fminf(fminf(m[0], m[1]), fminf(m[2], m[3]));
                } else {
                    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (uint32_t i = 0; i < S::kKeys; i += 2) m[i / 2 % 4] = fmaxf(fmaxf(m[i / 2 % 4], __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
                    most = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
                }
                const float top = fmaxf(reference, most * scale);
                const bool above = top > reference + kSlack || (!started && top > reference);
                if (__any_sync(0xffffffffu, above)) {
                    const float now = above ? top : reference, factor = now == reference ? 1.0f : exp2_fast(reference - now);
                    reference = now;
                    sum[0] *= factor, sum[1] *= factor, sum[2] *= factor, sum[3] *= factor;
                    if (started) {
                        // the stream's tile before has to be through
                        const uint32_t earlier = count - S::kStreams;
                        if (!warp_look_suspended(products + 8 * (earlier % S::kBuffers), earlier / S::kBuffers & 1, abort_flag, status, kStatusPrefixProduct)) {
                            alive = false;
                            break;
                        }
                        tc_fence_after();
#pragma unroll 1
                        for (uint32_t c = 0; c < kHeadDim; c += 16) {
                            uint32_t v[16];
                            load_columns<16>(out + c, v);
                            tc_wait_ld();
#pragma unroll
                            for (uint32_t i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * factor);
                            store_columns16(out + c, v);
                        }
                    }
                }
                if (!started) first_key = key;
                started = true;
                const float minus = reference == -INFINITY ? 0.0f : -reference;
#pragma unroll
                for (uint32_t c = 0; c < S::kKeys; c += 32) {
                    uint32_t packed[16];
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 2) fma2(v[c + i], v[c + i + 1], scale, minus);
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) v[c + i] = __float_as_uint(exp2_fast(__uint_as_float(v[c + i])));
                    if (masked) {
                        const uint32_t bits = seen(c);   // (again: with a scale of zero the exponential is not zero)
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i) v[c + i] = bits >> i & 1 ? v[c + i] : 0;
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i) {
                        const __nv_bfloat162 two = __floats2bfloat162_rn(__uint_as_float(v[c + 2 * i]), __uint_as_float(v[c + 2 * i + 1]));
                        packed[i] = *reinterpret_cast<const uint32_t*>(&two);
                        add2(sum[2 * (i % 2)], sum[2 * (i % 2) + 1], packed[i] << 16, packed[i] & 0xffff0000u);
                    }
                    store_columns16(from + c / 2, packed);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(weights_full + 8 * buffer);
            }
            if (!alive) break;
            // ---- the item's part ----
            const uint64_t part = static_cast<uint64_t>(item) * S::kStreams + stream;
            if (started) {
                const uint32_t final = count - 1 - (S::kStreams == 2 && ((count - 1) & 1) != stream ? 1 : 0);   // the stream's last tile
                if (!warp_look_suspended(products + 8 * (final % S::kBuffers), final / S::kBuffers & 1, abort_flag, status, kStatusPrefixProduct)) break;
                tc_fence_after();
                float4* const to = reinterpret_cast<float4*>(p.parts) + part * (kHeadDim / 4) * kRowsM + thread;
#pragma unroll 1
                for (uint32_t c = 0; c < kHeadDim; c += 32) {
                    uint32_t v[32];
                    tc_load32(out + c, v);
                    tc_wait_ld();
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 4) {
                        if (tile * kRowsM + thread < all_queries) to[(c + i) / 4 * kRowsM] = make_float4(__uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
                    }
                }
                tc_fence_before();
            }
            // (a part all of whose scores are NaN or -infinity has the reference -infinity too, but counts: its sums may be NaN)
            if (started && reference == -INFINITY && limit > first_key) reference = kNoNumber;
            reinterpret_cast<float2*>(p.parts + static_cast<uint64_t>(p.max_items) * S::kStreams * kRowsM * kHeadDim)[part * kRowsM + thread] = make_float2(reference, (sum[0] + sum[1]) + (sum[2] + sum[3]));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- a sequence's own tokens ----------------------------------------------------------------------
// These are few next to the prefix, and often very few: what counts is how many are under way at once. So small CTAs, several an SM, each a chunk of the tokens
// of a (sequence, key-value head), 64 at a time through shared memory and mma.sync (m16n8k16): a warp forms the scores of 16 of the 64 keys and then the
// outputs of a quarter of the dims. (The paged attention's kernel, one CTA an SM, took 4.4 us for every pair of some 40 tokens: 171 sequences of 8 heads 41 us.)
constexpr uint32_t kOwnThreads = 128, kOwnTile = 64;

template <uint32_t kHeadDim, uint32_t kM>
struct OwnShape {
    static constexpr uint32_t kQueries = 16 * kM, kRowBytes = kHeadDim * 2;
    static constexpr uint32_t kKeysAt = kQueries * kRowBytes, kValuesAt = kKeysAt + kOwnTile * kRowBytes, kWeightsAt = kValuesAt + kOwnTile * kRowBytes;
    static constexpr uint32_t kMostAt = kWeightsAt + kQueries * kOwnTile * 2, kSmem = kMostAt + 4 * kQueries * 4;
};
// 16 bytes `piece` of a row: pieces of eight rows that follow one another lie in different banks.
template <uint32_t kRowBytes>
__device__ __forceinline__ uint32_t own_at(uint32_t row, uint32_t piece) { return row * kRowBytes + ((piece ^ (row & 7)) << 4); }
__device__ __forceinline__ void ldmatrix4(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_turned(uint32_t (&v)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <uint32_t kHeadDim, uint32_t kM>
__global__ void __launch_bounds__(kOwnThreads) own_attention_kernel(const __nv_bfloat16* keys, const __nv_bfloat16* values, const __grid_constant__ PrefixParams p) {
    using S = OwnShape<kHeadDim, kM>;
    constexpr uint32_t kPieces = kHeadDim / 8, kDims = kHeadDim / 4;   // 16-byte pieces of a row, dims of a warp
    extern __shared__ __align__(128) uint8_t own_smem[];
    const uint32_t smem = smem_u32(own_smem), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* const wide = reinterpret_cast<float*>(own_smem + S::kMostAt);   // [warp][query]
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t chunk = blockIdx.x % p.chunks, pair = blockIdx.x / p.chunks, head = pair % p.a.kv_heads, b = pair / p.a.kv_heads;
    const int32_t first_row = p.a.token_starts[b], end_row = p.a.token_starts[b + 1];
    int32_t length = p.a.lengths[b];
    const uint32_t shared = shared_tokens(p);
    if (first_row < 0 || end_row > static_cast<int32_t>(p.a.rows) || end_row < first_row || end_row - first_row > static_cast<int32_t>(p.a.max_new)) {
        if (threadIdx.x == 0) atomicCAS(p.a.status_word, 0u, kStatusRows);
        return;
    }
    const int32_t room = static_cast<int32_t>(p.a.table_pages << p.a.page_shift);
    if (length > room) {
        length = room;
        if (threadIdx.x == 0) atomicCAS(p.a.status_word, 0u, kStatusPage);
    }
    const uint32_t tokens = static_cast<uint32_t>(end_row - first_row), group = p.a.query_heads / p.a.kv_heads, queries = tokens * group;
    if (!tokens) return;
    const int32_t own = length - static_cast<int32_t>(shared);   // below zero: the sequence ends in the prefix
    const uint32_t tiles = own > 0 ? (static_cast<uint32_t>(own) + kOwnTile - 1) / kOwnTile : 0, per = (tiles + p.chunks - 1) / p.chunks;
    const uint32_t tile0 = chunk * per, tile1 = tile0 + per < tiles ? tile0 + per : tiles;
    auto place_of = [&](uint32_t query) { return (static_cast<uint64_t>(first_row) + query / group) * p.a.query_heads + head * group + query % group; };
    if (tile0 >= tile1) {
        if (threadIdx.x < queries) p.own_stats[place_of(threadIdx.x) * p.chunks + chunk] = make_float2(-INFINITY, 0.0f);
        return;
    }
    for (uint32_t i = threadIdx.x; i < S::kQueries * kPieces; i += kOwnThreads) {
        const uint32_t query = i / kPieces, piece = i % kPieces;
        const bool live = query < queries;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                     ::"r"(smem + own_at<S::kRowBytes>(query, piece)), "l"(p.a.query + place_of(live ? query : 0) * kHeadDim + piece * 8), "r"(live ? 16 : 0)
                     : "memory");
    }
    // Of this thread's rows (of each 16: lane / 4 and 8 further): tokens seen, reference maximum, part of the denominator. And a quarter of the dims of the output.
    int32_t limit[kM][2];
    float reference[kM][2], sum[kM][2], out[kM][kDims / 8][4];
#pragma unroll
    for (uint32_t m = 0; m < kM; ++m) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t query = 16 * m + 8 * h + lane / 4;
            limit[m][h] = query < queries ? own - static_cast<int32_t>(tokens) + static_cast<int32_t>(query / group) + 1 : 0;
            reference[m][h] = -INFINITY, sum[m][h] = 0.0f;
        }
#pragma unroll
        for (uint32_t n = 0; n < kDims / 8; ++n) out[m][n][0] = out[m][n][1] = out[m][n][2] = out[m][n][3] = 0.0f;
    }
    const int32_t* const table = p.a.page_table + static_cast<uint64_t>(b) * p.a.table_pages + (shared >> p.a.page_shift);
    // A warp copies 16 of a tile's keys and values; a lane looks up the place of one of the 16.
    auto slot_of = [&](uint32_t tile) -> int64_t {
        const uint32_t key = tile * kOwnTile + warp * 16 + lane % 16;
        if (tile >= tile1 || key >= static_cast<uint32_t>(own)) return -1;
        const int32_t page = __ldg(table + (key >> p.a.page_shift));
        if (page < 0 || static_cast<uint32_t>(page) >= p.a.pages) {
            atomicCAS(p.a.status_word, 0u, kStatusPage);
            return -1;
        }
        return ((static_cast<int64_t>(page) * p.a.kv_heads + head) << p.a.page_shift) + (key & ((1u << p.a.page_shift) - 1));
    };
    int64_t slot = slot_of(tile0);
    for (uint32_t tile = tile0; tile < tile1; ++tile) {
        if (tile != tile0) __syncthreads();   // the tile before is no longer read
        auto copy = [&](const __nv_bfloat16* from, uint32_t to) {
#pragma unroll
            for (uint32_t i = 0; i < 16 * kPieces / 32; ++i) {
                const uint32_t at = i * 32 + lane, row = at / kPieces, piece = at % kPieces;
                const int64_t here = __shfl_sync(0xffffffffu, slot, row);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                             ::"r"(to + own_at<S::kRowBytes>(warp * 16 + row, piece)), "l"(from + (here < 0 ? 0 : here) * kHeadDim + piece * 8), "r"(here < 0 ? 0 : 16)
                             : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        copy(keys, smem + S::kKeysAt);
        copy(values, smem + S::kValuesAt);
        const uint32_t there = __ballot_sync(0xffffffffu, slot >= 0);   // (keys without a page count as not there)
        slot = slot_of(tile + 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (tile == tile0) __syncthreads();   // the queries; a warp's own keys it waits for itself
        else __syncwarp();
        // ---- scores of the warp's 16 keys ----
        float s[kM][2][4];
#pragma unroll
        for (uint32_t m = 0; m < kM; ++m) {
#pragma unroll
            for (uint32_t n = 0; n < 2; ++n) s[m][n][0] = s[m][n][1] = s[m][n][2] = s[m][n][3] = 0.0f;
        }
#pragma unroll 4
        for (uint32_t k = 0; k < kHeadDim / 16; ++k) {
            uint32_t key[4];
            ldmatrix4(key, smem + S::kKeysAt + own_at<S::kRowBytes>(warp * 16 + (lane & 7) + (lane >> 4) * 8, 2 * k + (lane >> 3 & 1)));
#pragma unroll
            for (uint32_t m = 0; m < kM; ++m) {
                uint32_t query[4];
                ldmatrix4(query, smem + own_at<S::kRowBytes>(16 * m + (lane & 15), 2 * k + (lane >> 4)));
                mma_16816(s[m][0], query, key[0], key[1]);
                mma_16816(s[m][1], query, key[2], key[3]);
            }
        }
        const int32_t key0 = static_cast<int32_t>(tile * kOwnTile + warp * 16 + 2 * (lane & 3));
#pragma unroll
        for (uint32_t m = 0; m < kM; ++m) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                float most = -INFINITY;
#pragma unroll
                for (uint32_t n = 0; n < 2; ++n) {
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        float& x = s[m][n][2 * h + e];
                        x = key0 + static_cast<int32_t>(8 * n + e) < limit[m][h] && (there >> (8 * n + 2 * (lane & 3) + e) & 1) ? x * p.a.scale_log2 : -INFINITY;
                        most = fmaxf(most, x);
                    }
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                if ((lane & 3) == 0) wide[warp * S::kQueries + 16 * m + 8 * h + lane / 4] = most;
            }
        }
        __syncthreads();
#pragma unroll
        for (uint32_t m = 0; m < kM; ++m) {
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
                const uint32_t query = 16 * m + 8 * h + lane / 4;
                float now = reference[m][h];
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) now = fmaxf(now, wide[w * S::kQueries + query]);
                const float factor = now == reference[m][h] ? 1.0f : exp2_fast(reference[m][h] - now), minus = now == -INFINITY ? 0.0f : now;
                reference[m][h] = now;
                sum[m][h] *= factor;
#pragma unroll
                for (uint32_t n = 0; n < kDims / 8; ++n) out[m][n][2 * h] *= factor, out[m][n][2 * h + 1] *= factor;
#pragma unroll
                for (uint32_t n = 0; n < 2; ++n) {
                    const __nv_bfloat162 two = __floats2bfloat162_rn(exp2_fast(s[m][n][2 * h] - minus), exp2_fast(s[m][n][2 * h + 1] - minus));
                    const uint32_t bits = *reinterpret_cast<const uint32_t*>(&two);
                    sum[m][h] += __uint_as_float(bits << 16) + __uint_as_float(bits & 0xffff0000u);
                    *reinterpret_cast<uint32_t*>(own_smem + S::kWeightsAt + own_at<kOwnTile * 2>(query, warp * 2 + n) + (lane & 3) * 4) = bits;
                }
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        // ---- outputs of the warp's dims ----
#pragma unroll
        for (uint32_t k = 0; k < kOwnTile / 16; ++k) {
            uint32_t weights[kM][4];
#pragma unroll
            for (uint32_t m = 0; m < kM; ++m) ldmatrix4(weights[m], smem + S::kWeightsAt + own_at<kOwnTile * 2>(16 * m + (lane & 15), 2 * k + (lane >> 4)));
#pragma unroll
            for (uint32_t n = 0; n < kDims / 8; n += 2) {
                uint32_t value[4];
                ldmatrix4_turned(value, smem + S::kValuesAt + own_at<S::kRowBytes>(16 * k + (lane & 15), (warp * kDims) / 8 + n + (lane >> 4)));
#pragma unroll
                for (uint32_t m = 0; m < kM; ++m) {
                    mma_16816(out[m][n], weights[m], value[0], value[1]);
                    mma_16816(out[m][n + 1], weights[m], value[2], value[3]);
                }
            }
        }
    }
    // ---- the chunk's part ----
#pragma unroll
    for (uint32_t m = 0; m < kM; ++m) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 1);
            sum[m][h] += __shfl_xor_sync(0xffffffffu, sum[m][h], 2);
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t m = 0; m < kM; ++m) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            if ((lane & 3) == 0) wide[warp * S::kQueries + 16 * m + 8 * h + lane / 4] = sum[m][h];
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t m = 0; m < kM; ++m) {
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t query = 16 * m + 8 * h + lane / 4;
            if (query >= queries) continue;
            const uint64_t part = place_of(query) * p.chunks + chunk;
            if (warp == 0 && (lane & 3) == 0) {
                // (a part all of whose scores are NaN or -infinity has the reference -infinity too, but counts: its sums may be NaN)
                const bool none = reference[m][h] == -INFINITY && limit[m][h] > static_cast<int32_t>(tile0 * kOwnTile);
                float all = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) all += wide[w * S::kQueries + query];
                p.own_stats[part] = make_float2(none ? kNoNumber : reference[m][h], all);
            }
#pragma unroll
            for (uint32_t n = 0; n < kDims / 8; ++n) {
                *reinterpret_cast<float2*>(p.own_parts + part * kHeadDim + warp * kDims + n * 8 + 2 * (lane & 3)) = make_float2(out[m][n][2 * h], out[m][n][2 * h + 1]);
            }
        }
    }
}

// Joins the parts of the prefix and of the rows' own tokens, in their order: a float4 a thread, and a warp (some warps) the weights of one of a CTA's queries.
constexpr uint32_t kMergeThreads = 256;
template <uint32_t kHeadDim>
constexpr uint32_t kMergeQueries = kMergeThreads / (kHeadDim / 4);
template <uint32_t kHeadDim>
__global__ void __launch_bounds__(kMergeThreads) prefix_merge_kernel(const __grid_constant__ PrefixParams p, uint32_t ctas) {
    using S = PrefixShape<kHeadDim>;
    constexpr uint32_t kQueries = kMergeQueries<kHeadDim>, kAhead = 8, kSlices = kRowsM / kQueries;
    constexpr uint32_t kMost = (kMaxSplit * S::kStreams + kMaxChunks + kAhead - 1) / kAhead * kAhead;
    __shared__ float2 stat[kQueries][kMost];   // reference maximum and denominator of a part; then, of those that count, the weight and the part's number
    __shared__ float total[kQueries];
    __shared__ uint32_t live[kQueries], count[kQueries];
    if (threadIdx.x < kQueries) live[threadIdx.x] = 0;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Items items = items_of<S::kKeys>(p, ctas);
    const uint32_t group = p.a.query_heads / p.a.kv_heads, all_queries = p.a.rows * group, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t slice = blockIdx.x % kSlices, tile = blockIdx.x / kSlices % p.tiles, head = blockIdx.x / kSlices / p.tiles;
    const uint32_t query0 = tile * kRowsM + slice * kQueries;
    if (query0 >= all_queries) return;
    const uint32_t shared_parts = items.key_tiles ? items.split * S::kStreams : 0, parts = shared_parts + p.chunks, padded = (parts + kAhead - 1) / kAhead * kAhead;
    // part n of the prefix: item (head, n / streams, tile), stream n % streams
    const uint64_t first_part = (static_cast<uint64_t>(head) * items.split * p.tiles + tile) * S::kStreams, next_item = static_cast<uint64_t>(p.tiles) * S::kStreams;
    auto part_of = [&](uint32_t n) { return first_part + n / S::kStreams * next_item + n % S::kStreams; };
    auto place_of = [&](uint32_t query) { return static_cast<uint64_t>(query / group) * p.a.query_heads + head * group + query % group; };
    __syncthreads();
    // The rows that belong to a sequence; meanwhile the parts' statistics.
    const float2* const stats = reinterpret_cast<const float2*>(p.parts + static_cast<uint64_t>(p.max_items) * S::kStreams * kRowsM * kHeadDim);
    for (uint32_t i = threadIdx.x; i < kQueries * padded; i += kMergeThreads) {
        const uint32_t n = i / kQueries, query = i % kQueries;
        float2 x = make_float2(-INFINITY, 0.0f);
        if (n < shared_parts) x = stats[part_of(n) * kRowsM + slice * kQueries + query];
        else if (n < parts && query0 + query < all_queries) x = p.own_stats[place_of(query0 + query) * p.chunks + n - shared_parts];
        stat[query][n] = x;
    }
    for (uint32_t b = threadIdx.x; b < p.a.sequences; b += kMergeThreads) {
        const int32_t from = p.a.token_starts[b], to = p.a.token_starts[b + 1];
        if (from < 0 || to > static_cast<int32_t>(p.a.rows) || to < from || to - from > static_cast<int32_t>(p.a.max_new)) continue;
        for (uint32_t i = 0; i < kQueries; ++i) {
            const int32_t row = static_cast<int32_t>((query0 + i) / group);
            if (from <= row && row < to) live[i] = 1;
        }
    }
    __syncthreads();
    // A query's weights 2^(reference - largest reference), and its denominator. Parts of which it sees nothing are passed over. All others count, with a
    // weight of zero too: zero times a NaN is one.
    if (warp < kQueries) {
        float most = -INFINITY, all = 0.0f;
        for (uint32_t n = lane; n < parts; n += 32) most = fmaxf(most, stat[warp][n].x);
#pragma unroll
        for (uint32_t step = 16; step; step /= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, step));
        uint32_t kept = 0;
        for (uint32_t first = 0; first < padded; first += 32) {
            const uint32_t n = first + lane;
            const float2 x = n < parts ? stat[warp][n] : make_float2(-INFINITY, 0.0f);
            const uint32_t counts = __ballot_sync(0xffffffffu, x.x != -INFINITY);
            if (x.x != -INFINITY) {
                const float w = exp2_fast(x.x - most);
                all = fmaf(w, x.y, all);
                stat[warp][kept + __popc(counts & ((1u << lane) - 1))] = make_float2(w, __uint_as_float(n));   // (at or before its own place, which all lanes have read)
            }
            kept += __popc(counts);
            __syncwarp();
        }
#pragma unroll
        for (uint32_t step = 16; step; step /= 2) all += __shfl_xor_sync(0xffffffffu, all, step);
        if (lane == 0) total[warp] = all, count[warp] = kept;
    }
    __syncthreads();
    const uint32_t i = threadIdx.x % kQueries, query = query0 + i, column = threadIdx.x / kQueries, row = slice * kQueries + i;
    if (query >= all_queries || !live[i]) return;
    const uint64_t place = place_of(query);
    const float4* const shared_from = reinterpret_cast<const float4*>(p.parts) + column * kRowsM + row;
    const float4* const own_from = reinterpret_cast<const float4*>(p.own_parts + place * p.chunks * kHeadDim) + column;
    const uint32_t kept = count[i];
    float4 sum = make_float4(0, 0, 0, 0);
    for (uint32_t first = 0; first < kept; first += kAhead) {
        float4 v[kAhead];
        float w[kAhead];
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            v[a] = make_float4(0, 0, 0, 0), w[a] = 0.0f;
            if (first + a < kept) {
                const float2 x = stat[i][first + a];
                const uint32_t n = __float_as_uint(x.y);
                w[a] = x.x;
                v[a] = n < shared_parts ? shared_from[part_of(n) * (kHeadDim / 4 * kRowsM)] : own_from[(n - shared_parts) * (kHeadDim / 4)];
            }
        }
#pragma unroll
        for (uint32_t a = 0; a < kAhead; ++a) {
            sum.x = fmaf(w[a], v[a].x, sum.x), sum.y = fmaf(w[a], v[a].y, sum.y), sum.z = fmaf(w[a], v[a].z, sum.z), sum.w = fmaf(w[a], v[a].w, sum.w);
        }
    }
    const float all = total[i], inverse = 1.0f / all;
    const __nv_bfloat162 a = __floats2bfloat162_rn(all == 0.0f ? 0.0f : sum.x * inverse, all == 0.0f ? 0.0f : sum.y * inverse);
    const __nv_bfloat162 c = __floats2bfloat162_rn(all == 0.0f ? 0.0f : sum.z * inverse, all == 0.0f ? 0.0f : sum.w * inverse);
    reinterpret_cast<uint2*>(p.a.output + place * kHeadDim)[column] = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
}

// What the plan's scratch holds, in bytes from its start.
struct Layout {
    uint64_t own_parts, own_stats, parts, bytes;
    uint32_t max_items, tiles, chunks;
};
Layout layout_of(uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t rows, uint32_t max_new, uint32_t sm_count) {
    auto aligned = [](uint64_t x) { return (x + 255) / 256 * 256; };
    const uint64_t outputs = static_cast<uint64_t>(rows) * query_heads, streams = head_dim == 128 ? 2 : 1;
    Layout l;
    l.tiles = static_cast<uint32_t>((static_cast<uint64_t>(rows) * (query_heads / kv_heads) + kRowsM - 1) / kRowsM);
    const uint64_t pairs = static_cast<uint64_t>(kv_heads) * l.tiles, most = kRounds * static_cast<uint64_t>(sm_count);   // (of queries and heads; below 2^30)
    l.max_items = static_cast<uint32_t>(pairs > most ? pairs : most);
    // The sequences' own tokens in as many chunks as give an SM about so many CTAs.
    constexpr uint64_t kOwnCtas = 8;
    const uint64_t sequences = (rows + max_new - 1) / max_new, chunks = kOwnCtas * static_cast<uint64_t>(sm_count) / (sequences * kv_heads);
    l.chunks = static_cast<uint32_t>(chunks < 1 ? 1 : chunks < kMaxChunks ? chunks : kMaxChunks);
    l.own_parts = kCounterBytes;
    l.own_stats = aligned(l.own_parts + outputs * l.chunks * head_dim * sizeof(float));
    l.parts = aligned(l.own_stats + outputs * l.chunks * sizeof(float2));
    l.bytes = l.parts + l.max_items * streams * kRowsM * (head_dim + 2) * sizeof(float);
    return l;
}

bool check_shared(int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_plan_v1* plan, const augur_cuda_nvfp4_sm100_shared_prefix_attention_args_v1* a,
                  bool full, augur_cuda_result_v1* failure) {
    Range ranges[kAttentionRanges + 2];
    size_t count;
    if (!attention_args_ok(d, s, plan, a, ranges, &count, failure)) return false;
    const uint64_t pages = a->prefix_pages_len_bytes / 4;
    if (!pages || a->prefix_pages_len_bytes % 4 != 0 || pages > (1u << kMaxTokensLog2) || pages * a->layer.page_tokens > (1u << kMaxTokensLog2) || a->prefix_tokens_len_bytes != 4) return false;
    ranges[count + 1] = ranges[count - 1];   // the scratch stays the last
    ranges[count - 1] = {a->prefix_pages, a->prefix_pages_len_bytes, 4}, ranges[count] = {a->prefix_tokens, 4, 4};
    count += 2;
    if (!all_disjoint(ranges, count)) return false;
    uint64_t need = 0;
    if (augur_cuda_nvfp4_sm100_shared_prefix_attention_scratch_extent_host_v1(a->query_heads, a->layer.kv_heads, a->layer.head_dim, a->batch.rows, a->max_new_tokens,
                                                                              plan->sm_count, &need).status != AUGUR_CUDA_STATUS_OK || plan->scratch_bytes < need) return false;
    return !full || inspect_device_ranges(d, ranges, count - 1, failure);
}

template <uint32_t kHeadDim, uint32_t kM>
void launch_own(cudaStream_t stream, const __nv_bfloat16* keys, const __nv_bfloat16* values, const PrefixParams& p) {
    launch_dependent(stream, own_attention_kernel<kHeadDim, kM>, p.a.sequences * p.a.kv_heads * p.chunks, kOwnThreads, OwnShape<kHeadDim, kM>::kSmem, keys, values, p);
}

template <uint32_t kHeadDim>
void launch_prefix(cudaStream_t stream, const CUtensorMap& map_keys, const CUtensorMap& map_values, const __nv_bfloat16* keys, const __nv_bfloat16* values, const PrefixParams& p,
                   uint32_t sm_count) {
    using S = PrefixShape<kHeadDim>;
    // The prefix behind the own tokens: its parts are the many, and still in L2 when they are joined. (The other way round the join of 64 sequences took 14 us, not 9.)
    const uint32_t queries = p.a.query_heads / p.a.kv_heads * p.a.max_new;
    (queries <= 16 ? launch_own<kHeadDim, 1> : queries <= 32 ? launch_own<kHeadDim, 2> : launch_own<kHeadDim, 4>)(stream, keys, values, p);
    launch_dependent(stream, prefix_attention_kernel<kHeadDim>, sm_count, S::kThreads, S::kSmem, map_keys, map_values, p);
    launch_dependent(stream, prefix_merge_kernel<kHeadDim>, p.a.kv_heads * p.tiles * (kRowsM / kMergeQueries<kHeadDim>), kMergeThreads, 0, p, sm_count);
    count_launch(3);
}

template <uint32_t kHeadDim>
cudaError_t configure() {
    constexpr cudaFuncAttribute kSmem = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = cudaFuncSetAttribute(prefix_attention_kernel<kHeadDim>, kSmem, PrefixShape<kHeadDim>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(own_attention_kernel<kHeadDim, 1>, kSmem, OwnShape<kHeadDim, 1>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(own_attention_kernel<kHeadDim, 2>, kSmem, OwnShape<kHeadDim, 2>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(own_attention_kernel<kHeadDim, 4>, kSmem, OwnShape<kHeadDim, 4>::kSmem);
    return e;
}

}  // namespace

cudaError_t shared_prefix_configure_device() {
    const cudaError_t e = configure<128>();
    return e == cudaSuccess ? configure<256>() : e;
}

}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_shared_prefix_attention_scratch_extent_host_v1(
    uint32_t query_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t rows, uint32_t max_new_tokens, uint32_t sm_count, uint64_t* out_bytes) {
    if (!out_bytes || !shape_ok(query_heads, kv_heads, head_dim, max_new_tokens) || !sm_count || sm_count > 4096 || !rows || rows > (1u << 20)) return invalid();
    *out_bytes = layout_of(query_heads, kv_heads, head_dim, rows, max_new_tokens, sm_count).bytes;
    return ok();
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
    const uint32_t head_dim = a->layer.head_dim, kv_heads = a->layer.kv_heads, box = a->layer.page_tokens < kUnit ? a->layer.page_tokens : kUnit;
    const Layout l = layout_of(a->query_heads, kv_heads, head_dim, a->batch.rows, a->max_new_tokens, plan->sm_count);
    PrefixParams p{};
    p.a = attention_params(plan, a);
    p.prefix_table = reinterpret_cast<const int32_t*>(a->prefix_pages);
    p.prefix_tokens = reinterpret_cast<const int32_t*>(a->prefix_tokens);
    p.prefix_pages = static_cast<uint32_t>(a->prefix_pages_len_bytes / 4);
    p.own_parts = reinterpret_cast<float*>(plan->scratch + l.own_parts);
    p.own_stats = reinterpret_cast<float2*>(plan->scratch + l.own_stats);
    p.parts = reinterpret_cast<float*>(plan->scratch + l.parts);
    p.max_items = l.max_items, p.tiles = l.tiles, p.chunks = l.chunks;
    const uint64_t cache_rows = static_cast<uint64_t>(a->layer.pages) * kv_heads * a->layer.page_tokens;
    CUtensorMap keys, values;
    if (!make_code_map(&keys, a->layer.keys, cache_rows, head_dim * 4, box) || !make_code_map(&values, a->layer.values, cache_rows, head_dim * 4, box)) {
        return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE);
    }
    const auto* const key_data = reinterpret_cast<const __nv_bfloat16*>(a->layer.keys);
    const auto* const value_data = reinterpret_cast<const __nv_bfloat16*>(a->layer.values);
    (head_dim == 256 ? launch_prefix<256> : launch_prefix<128>)(s->stream, keys, values, key_data, value_data, p, plan->sm_count);
    return submitted();
}
