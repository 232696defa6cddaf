// Writing and moving the pages of a key-value cache on sm_100a: rotary positions with the cache write of a step's tokens, and page copies.
#include <cstdlib>

#include "kv_cache.cuh"

namespace augur_sm100 {
namespace {

static_assert(sizeof(augur_cuda_nvfp4_sm100_kv_layer_v1) == 40 && sizeof(augur_cuda_nvfp4_sm100_kv_batch_v1) == 64, "cache ABI");
static_assert(sizeof(augur_cuda_nvfp4_sm100_kv_append_args_v1) == 312, "append ABI");
static_assert(sizeof(augur_cuda_nvfp4_sm100_kv_page_copy_args_v1) == 48, "page copy ABI");
static_assert(sizeof(augur_cuda_nvfp4_sm100_kv_e4m3_layer_v1) == 56 && sizeof(augur_cuda_nvfp4_sm100_kv_append_e4m3_args_v1) == 328 &&
                  sizeof(augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_args_v1) == 72,
              "E4M3 cache ABI");

// ---- rotary positions and the cache write ---------------------------------------------------------

struct AppendParams {
    const __nv_bfloat16 *query, *key, *value;
    uint64_t query_row_stride, query_head_stride, key_row_stride, key_head_stride, value_row_stride, value_head_stride;
    const int32_t *positions, *page_table, *lengths, *token_starts;
    const float *inv_freq, *query_norm, *key_norm;
    __nv_bfloat16* query_out;
    void *keys, *values;                 // BF16, or E4M3 codes with
    uint8_t* scales;
    uint32_t rows, sequences, table_pages, pages, query_heads, kv_heads, page_shift;
    uint32_t half;                       // rotary pairs
    uint32_t sections[3], interleaved;
    float epsilon;
};

// The scale byte of the eight elements x of each of kLanes lanes and their codes: the scale is the smallest power of two, of the ones allowed, with which
// the largest element that is a number is at most 448 = 1.75 * 2^8. Elements that are looked at one by one only where one of the head's is infinite or
// too large (a maximum passes over NaN, and the conversion keeps it).
template <uint32_t kLanes>
__device__ __forceinline__ uint2 quantise_head(float (&x)[8], unsigned mask, uint32_t* scale) {
    float most = 0.0f;
#pragma unroll
    for (uint32_t e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
#pragma unroll
    for (uint32_t step = kLanes / 2; step; step /= 2) most = fmaxf(most, __shfl_xor_sync(mask, most, step));
    constexpr float kLargest = 448.0f * (1ull << (kE4m3LargestScale - 127));
    if (most > kLargest) {
        most = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
            most = fmaxf(most, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f);
            if (fabsf(x[e]) > kLargest) x[e] = __uint_as_float(0x7fc00000u);   // (the conversion would clamp it)
        }
#pragma unroll
        for (uint32_t step = kLanes / 2; step; step /= 2) most = fmaxf(most, __shfl_xor_sync(mask, most, step));
    }
    const uint32_t bits = __float_as_uint(most), exact = (bits >> 23) + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    const uint32_t byte = exact < kE4m3LeastScale + 8 ? kE4m3LeastScale : exact > kE4m3LargestScale + 8 ? kE4m3LargestScale : exact - 8;
    const float inverse = __uint_as_float((254 - byte) << 23);
    uint32_t pair[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e) {
        uint16_t two;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(x[2 * e + 1] * inverse), "f"(x[2 * e] * inverse));
        pair[e] = two;
    }
    *scale = byte;
    return make_uint2(pair[0] | pair[1] << 16, pair[2] | pair[3] << 16);
}

constexpr uint32_t kAppendThreads = 256, kAppendCtas = 2368;   // two rounds of eight an SM

// head_dim / 8 neighbouring lanes turn one head, eight elements (one 16-byte access) each, for kRows rows one after the other; blockIdx.y deals out the
// heads. The sines and cosines of a row are formed once per CTA. What the rotation pairs lies rotary_dim / 16 lanes away: a shuffle.
// A step of few rows is a matter of latency: a row a CTA, every load under way before the row's sequence and angles are known (one CTA for all
// heads of a row, loads behind them: 8 rows of 24 + 2 x 4 heads of 256 5.9 us, now 3.5, which is the host's submit). With many rows the chain of lookups
// counts as often as there are rounds of CTAs: four rows at once (1024 rows of those heads with head norms 17.5 -> 11.3 us, 640 rows 11.1 -> 8.3; 480 rows of 32 + 2 x 8
// heads of 128, which are 1440 CTAs, 5.4 one by one and 6.2 by fours).
// E4M3: a head's scale wants its largest magnitude, one more reduction over the lanes that hold it, of the F32 elements (the key is never rounded to BF16).
template <uint32_t kHeadDim, uint32_t kRows, bool kE4m3>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ AppendParams p) {
    constexpr uint32_t kLanes = kHeadDim / 8, kGroups = kAppendThreads / kLanes;
    __shared__ __align__(16) float cosine[kE4m3 ? 2 * kRows : kRows][kHeadDim / 2], sine[kE4m3 ? 2 * kRows : kRows][kHeadDim / 2];   // (from kRows on the keys')
    __shared__ int32_t sequence_at[kRows], slot_page[kRows], slot_offset[kRows];
    const uint32_t row0 = blockIdx.x * kRows, heads = p.query_heads + 2 * p.kv_heads;
    const uint32_t h = blockIdx.y * kGroups + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    if (threadIdx.x < kRows) sequence_at[threadIdx.x] = -1;
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool is_query = h < p.query_heads, is_value = h >= p.query_heads + p.kv_heads, live = h < heads;
    const uint32_t head = is_query ? h : is_value ? h - p.query_heads - p.kv_heads : h - p.query_heads;
    const __nv_bfloat16* const from = is_query ? p.query + head * p.query_head_stride : is_value ? p.value + head * p.value_head_stride : p.key + head * p.key_head_stride;
    const uint64_t row_stride = is_query ? p.query_row_stride : is_value ? p.value_row_stride : p.key_row_stride;
    const float* const norm = is_query ? p.query_norm : is_value ? nullptr : p.key_norm;
    uint4 raw[kRows];
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
        raw[r] = make_uint4(0, 0, 0, 0);
        if (live && row0 + r < p.rows) raw[r] = __ldg(reinterpret_cast<const uint4*>(from + (row0 + r) * row_stride) + lane);
    }
    float weight[8];
    if (live && norm) {
        if (reinterpret_cast<uint64_t>(norm) % 16 == 0) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(norm) + 2 * lane), b = __ldg(reinterpret_cast<const float4*>(norm) + 2 * lane + 1);
            weight[0] = a.x, weight[1] = a.y, weight[2] = a.z, weight[3] = a.w, weight[4] = b.x, weight[5] = b.y, weight[6] = b.z, weight[7] = b.w;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; ++e) weight[e] = __ldg(norm + 8 * lane + e);
        }
    }
    for (uint32_t b = threadIdx.x; b < p.sequences; b += kAppendThreads) {
        const int32_t first = __ldg(p.token_starts + b), end = __ldg(p.token_starts + b + 1), length = __ldg(p.lengths + b);
#pragma unroll
        for (uint32_t r = 0; r < kRows; ++r) {
            const int32_t row = static_cast<int32_t>(row0 + r);
            if (row < first || row >= end || row0 + r >= p.rows) continue;
            const int64_t position = static_cast<int64_t>(length) - end + row;   // in the cache
            const int64_t page = position >> p.page_shift;
            int32_t at = -1;
            if (position >= 0 && page < p.table_pages) at = __ldg(p.page_table + static_cast<uint64_t>(b) * p.table_pages + page);
            sequence_at[r] = static_cast<int32_t>(b);
            slot_page[r] = at >= 0 && static_cast<uint32_t>(at) < p.pages ? at : -1;
            slot_offset[r] = static_cast<int32_t>(position & ((int64_t(1) << p.page_shift) - 1));
        }
    }
    // (from the last threads on: the first ones are busy with few sequences)
    for (uint32_t j = kAppendThreads - 1 - threadIdx.x; j < kRows * p.half; j += kAppendThreads) {
        const uint32_t r = j / p.half, i = j - r * p.half;
        if (row0 + r >= p.rows) break;
        uint32_t axis;
        if (p.interleaved) {
            axis = i % 3;
            if (i >= 3 * p.sections[axis]) axis = 0;
        } else {
            axis = (i >= p.sections[0] ? 1u : 0u) + (i >= p.sections[0] + p.sections[1] ? 1u : 0u);
        }
        // In turns, in 64 bits: a position of 2^20 leaves 2^-33 of a turn, where the F32 product would have lost 2^-7.
        const double turns =
            static_cast<double>(__ldg(p.positions + static_cast<uint64_t>(axis) * p.rows + row0 + r)) * static_cast<double>(__ldg(p.inv_freq + i)) * 0.15915494309189535;
        const float part_turn = static_cast<float>(turns - rint(turns));
        sincospif(2.0f * part_turn, &sine[r][i], &cosine[r][i]);
        if constexpr (kE4m3) {
            // Nothing rounds a key between here and its code: what the angle has lost in F32 (up to 2^-26 of a turn, more than the function's own error) is
            // brought back to first order; the queries stay those of a write to BF16.
            // (67 million elements of keys, positions to 2^20: 243 codes other than a computation in 64 bits gives, with it 221.)
            const float rest = static_cast<float>(turns - rint(turns) - part_turn) * 6.2831853f;
            sine[kRows + r][i] = fmaf(cosine[r][i], rest, sine[r][i]), cosine[kRows + r][i] = fmaf(-sine[r][i], rest, cosine[r][i]);
        }
    }
    __syncthreads();
    if (!live) return;   // (whole groups; nothing is waited for below)
    const uint32_t half_lanes = p.half / 8;
    const bool turns = lane < 2 * half_lanes, upper = lane >= half_lanes;
    const uint32_t partner = !turns ? lane : upper ? lane - half_lanes : lane + half_lanes;
    const uint32_t pair = (turns ? 8 * (upper ? lane - half_lanes : lane) : 0) + (kE4m3 && !is_query ? kRows * (kHeadDim / 2) : 0);
    const unsigned mask = kLanes == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);   // the lanes of a head stay together
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
        if (row0 + r >= p.rows || sequence_at[r] < 0 || (!is_query && slot_page[r] < 0)) continue;
        const uint64_t slot = is_query ? 0 : ((static_cast<uint64_t>(slot_page[r]) * p.kv_heads + head) << p.page_shift) + slot_offset[r];
        __nv_bfloat16* to = nullptr;
        if (is_query) to = p.query_out + (static_cast<uint64_t>(row0 + r) * p.query_heads + head) * kHeadDim;
        else if (!kE4m3) to = static_cast<__nv_bfloat16*>(is_value ? p.values : p.keys) + slot * kHeadDim;
        uint4 result = raw[r];
        float x[8];
        const uint32_t word[4] = {raw[r].x, raw[r].y, raw[r].z, raw[r].w};
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(word[e] << 16);
            x[2 * e + 1] = __uint_as_float(word[e] & 0xffff0000u);
        }
        if (!is_value) {
            if (norm) {
                float sum = 0.0f;
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
                for (uint32_t step = kLanes / 2; step; step /= 2) sum += __shfl_xor_sync(mask, sum, step);
                const float scale = __frsqrt_rn(sum * (1.0f / kHeadDim) + p.epsilon);
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) x[e] = x[e] * scale * weight[e];
            }
#pragma unroll
            for (uint32_t e = 0; e < 8; e += 4) {
                const float4 c = *reinterpret_cast<const float4*>(cosine[r] + pair + e), n = *reinterpret_cast<const float4*>(sine[r] + pair + e);
                const float cosines[4] = {c.x, c.y, c.z, c.w}, sines[4] = {n.x, n.y, n.z, n.w};
                float other[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) other[i] = __shfl_sync(mask, x[e + i], partner, kLanes);
                if (turns) {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) x[e + i] = fmaf(x[e + i], cosines[i], (upper ? other[i] : -other[i]) * sines[i]);
                }
            }
            uint32_t packed[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
                packed[e] = *reinterpret_cast<const uint32_t*>(&two);
            }
            result = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        }
        if (kE4m3 && !is_query) {
            uint32_t scale;
            const uint2 codes = quantise_head<kLanes>(x, mask, &scale);
            *(reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_value ? p.values : p.keys) + slot * kHeadDim) + lane) = codes;
            if (lane == 0) p.scales[2 * slot + (is_value ? 1 : 0)] = static_cast<uint8_t>(scale);
        } else {
            *(reinterpret_cast<uint4*>(to) + lane) = result;
        }
    }
}

template <class Args>
bool check_append(int32_t d, augur_cuda_stream_t s, const Args* a, bool full, augur_cuda_result_v1* failure) {
    *failure = invalid();
    if (!header_ok(d, s, a)) {
        if (a && s && d >= 0 && s->ordinal == d && a->abi_version != AUGUR_CUDA_ABI_VERSION_V1) *failure = make_result(AUGUR_CUDA_STATUS_ABI_VERSION_MISMATCH);
        return false;
    }
    if (!kv_layer_ok(a->layer) || !kv_batch_ok(a->batch) || a->reserved != 0 || a->interleaved > 1) return false;
    const uint32_t head_dim = a->layer.head_dim, kv_heads = a->layer.kv_heads, rows = a->batch.rows;
    if (!a->query_heads || a->query_heads > 1024 || a->rotary_dim > head_dim || a->rotary_dim % 16 != 0 || a->rotary_dim == 0) return false;
    if (!(std::isfinite(a->epsilon) && a->epsilon >= 0.0f)) return false;
    const uint64_t pairs = static_cast<uint64_t>(a->sections[0]) + a->sections[1] + a->sections[2];
    if (pairs != a->rotary_dim / 2) return false;
    const uint64_t strides[6] = {a->query_row_stride, a->query_head_stride, a->key_row_stride, a->key_head_stride, a->value_row_stride, a->value_head_stride};
    for (const uint64_t stride : strides) {
        if (stride % 8 != 0 || stride < head_dim) return false;
    }
    if (a->query_len_bytes != 2 * strided_elements(rows, a->query_heads, head_dim, strides[0], strides[1])) return false;
    if (a->key_len_bytes != 2 * strided_elements(rows, kv_heads, head_dim, strides[2], strides[3])) return false;
    if (a->value_len_bytes != 2 * strided_elements(rows, kv_heads, head_dim, strides[4], strides[5])) return false;
    if (a->positions_len_bytes != static_cast<uint64_t>(rows) * 12 || a->inv_freq_len_bytes != a->rotary_dim * UINT64_C(2)) return false;
    if (a->query_out_len_bytes != static_cast<uint64_t>(rows) * a->query_heads * head_dim * 2) return false;
    if (a->norm_len_bytes != (a->query_norm_f32 || a->key_norm_f32 ? head_dim * UINT64_C(4) : 0)) return false;
    // What is written is disjoint from everything; what is read may share memory (q, k and v of one projection, one norm weight for both).
    Range written[1 + kKvRanges] = {{a->query_out, a->query_out_len_bytes, 16}};
    const size_t outputs = 1 + kv_ranges(a->layer, written + 1);
    Range read[10] = {{a->query, a->query_len_bytes, 16}, {a->key, a->key_len_bytes, 16}, {a->value, a->value_len_bytes, 16},
                      {a->positions, a->positions_len_bytes, 4}, {a->inv_freq_f32, a->inv_freq_len_bytes, 4},
                      {a->batch.page_table, a->batch.page_table_len_bytes, 4}, {a->batch.lengths, a->batch.lengths_len_bytes, 4},
                      {a->batch.token_starts, a->batch.token_starts_len_bytes, 4}, {}, {}};
    size_t count = 8;
    if (a->query_norm_f32) read[count++] = {a->query_norm_f32, a->norm_len_bytes, 4};
    if (a->key_norm_f32) read[count++] = {a->key_norm_f32, a->norm_len_bytes, 4};
    if (!all_disjoint(written, outputs)) return false;
    for (size_t i = 0; i < count; ++i) {
        for (size_t j = 0; j < outputs; ++j) {
            if (!disjoint(read[i], written[j])) return false;
        }
    }
    return !full || (inspect_device_ranges(d, written, outputs, failure) && inspect_device_ranges(d, read, count, failure));
}

uint8_t* scales_of(const augur_cuda_nvfp4_sm100_kv_layer_v1&) { return nullptr; }
uint8_t* scales_of(const augur_cuda_nvfp4_sm100_kv_e4m3_layer_v1& l) { return reinterpret_cast<uint8_t*>(l.scales); }

template <bool kE4m3, class Args>
augur_cuda_result_v1 submit_append(int32_t d, augur_cuda_stream_t s, const Args* a) {
    augur_cuda_result_v1 failure;
    if (!check_append(d, s, a, false, &failure)) return failure;
    if (consume_injected_fault()) return make_result(AUGUR_CUDA_STATUS_DIAGNOSTIC_FAULT_INJECTED);
    const cudaError_t e = cudaSetDevice(d);
    if (e != cudaSuccess) return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE, e);
    AppendParams p{};
    p.query = reinterpret_cast<const __nv_bfloat16*>(a->query);
    p.key = reinterpret_cast<const __nv_bfloat16*>(a->key);
    p.value = reinterpret_cast<const __nv_bfloat16*>(a->value);
    p.query_row_stride = a->query_row_stride, p.query_head_stride = a->query_head_stride;
    p.key_row_stride = a->key_row_stride, p.key_head_stride = a->key_head_stride;
    p.value_row_stride = a->value_row_stride, p.value_head_stride = a->value_head_stride;
    p.positions = reinterpret_cast<const int32_t*>(a->positions);
    p.page_table = reinterpret_cast<const int32_t*>(a->batch.page_table);
    p.lengths = reinterpret_cast<const int32_t*>(a->batch.lengths);
    p.token_starts = reinterpret_cast<const int32_t*>(a->batch.token_starts);
    p.inv_freq = reinterpret_cast<const float*>(a->inv_freq_f32);
    p.query_norm = reinterpret_cast<const float*>(a->query_norm_f32);
    p.key_norm = reinterpret_cast<const float*>(a->key_norm_f32);
    p.query_out = reinterpret_cast<__nv_bfloat16*>(a->query_out);
    p.keys = reinterpret_cast<void*>(a->layer.keys);
    p.values = reinterpret_cast<void*>(a->layer.values);
    p.scales = scales_of(a->layer);
    p.rows = a->batch.rows, p.sequences = a->batch.sequences, p.table_pages = a->batch.table_pages, p.pages = a->layer.pages;
    p.query_heads = a->query_heads, p.kv_heads = a->layer.kv_heads, p.page_shift = static_cast<uint32_t>(__builtin_ctz(a->layer.page_tokens));
    p.half = a->rotary_dim / 2;
    for (uint32_t i = 0; i < 3; ++i) p.sections[i] = a->sections[i];
    p.interleaved = a->interleaved, p.epsilon = a->epsilon;
    const uint32_t groups = kAppendThreads / (a->layer.head_dim / 8), heads = a->query_heads + 2 * a->layer.kv_heads, slices = (heads + groups - 1) / groups;
    const bool many = static_cast<uint64_t>(p.rows) * slices > kAppendCtas;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.stream = s->stream, config.attrs = &attribute, config.numAttrs = 1;
    config.gridDim = dim3(many ? (p.rows + 3) / 4 : p.rows, slices), config.blockDim = dim3(kAppendThreads);
    if (a->layer.head_dim == 256) cudaLaunchKernelEx(&config, many ? kv_append_kernel<256, 4, kE4m3> : kv_append_kernel<256, 1, kE4m3>, p);
    else cudaLaunchKernelEx(&config, many ? kv_append_kernel<128, 4, kE4m3> : kv_append_kernel<128, 1, kE4m3>, p);
    count_launch();
    return submitted();
}

// ---- page copies ---------------------------------------------------------------------------------

// The page numbers travel as launch parameters: nothing to copy ahead, nothing to keep. Few pairs (a fork) in a short list: a launch with 8 KB of
// parameters costs the host 2 us more than one with 64 bytes.
constexpr uint32_t kPairsPerLaunch = 1000, kFewPairs = 8;
constexpr uint32_t kCopyThreads = 256, kCopyPiece = kCopyThreads * 16 * 4;
template <uint32_t kPairs>
struct PagePairs {
    uint32_t source[kPairs], destination[kPairs];
};

// What the copies move: a page of a layer takes `pieces` CTAs for its keys and as many for its values, and (an E4M3 cache) `scale_pieces` for its scales.
struct CopyParams {
    uint8_t *keys, *values, *scales;
    uint64_t page_bytes, scale_page_bytes;
    uint32_t pages, layers, pieces, scale_pieces;
};

template <uint32_t kPairs>
__global__ void __launch_bounds__(kCopyThreads) kv_page_copy_kernel(const __grid_constant__ PagePairs<kPairs> pairs, const __grid_constant__ CopyParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t all = 2 * p.pieces + p.scale_pieces;
    uint32_t at = blockIdx.x, piece = at % all;
    at /= all;
    const uint32_t layer = at % p.layers, pair = at / p.layers;
    uint8_t* tensor = p.scales;
    uint64_t page_bytes = p.scale_page_bytes;
    if (piece < 2 * p.pieces) {
        tensor = piece < p.pieces ? p.keys : p.values;
        page_bytes = p.page_bytes;
        if (piece >= p.pieces) piece -= p.pieces;
    } else {
        piece -= 2 * p.pieces;
    }
    uint8_t* base = tensor + static_cast<uint64_t>(layer) * p.pages * page_bytes;
    const uint64_t first = static_cast<uint64_t>(piece) * kCopyPiece;
    const uint8_t* from = base + pairs.source[pair] * page_bytes + first;
    uint8_t* to = base + pairs.destination[pair] * page_bytes + first;
    const uint64_t bytes = page_bytes - first < kCopyPiece ? page_bytes - first : kCopyPiece;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    uint4 v[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t offset = (i * kCopyThreads + threadIdx.x) * 16;
        if (offset < bytes) v[i] = *reinterpret_cast<const uint4*>(from + offset);
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t offset = (i * kCopyThreads + threadIdx.x) * 16;
        if (offset < bytes) *reinterpret_cast<uint4*>(to + offset) = v[i];
    }
}

uint64_t scales_len_of(const augur_cuda_nvfp4_sm100_kv_page_copy_args_v1&) { return 0; }
uint64_t scales_len_of(const augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_args_v1& a) { return a.scales_len_bytes; }
uint64_t scale_page_of(const augur_cuda_nvfp4_sm100_kv_page_copy_args_v1&) { return 0; }
uint64_t scale_page_of(const augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_args_v1& a) { return a.scale_page_bytes; }
uint64_t scales_at(const augur_cuda_nvfp4_sm100_kv_page_copy_args_v1&) { return 0; }
uint64_t scales_at(const augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_args_v1& a) { return a.scales; }

template <bool kScales, class Args>
bool check_page_copy(int32_t d, augur_cuda_stream_t s, const Args* a, bool full, augur_cuda_result_v1* failure) {
    *failure = invalid();
    if (!header_ok(d, s, a)) {
        if (a && s && d >= 0 && s->ordinal == d && a->abi_version != AUGUR_CUDA_ABI_VERSION_V1) *failure = make_result(AUGUR_CUDA_STATUS_ABI_VERSION_MISMATCH);
        return false;
    }
    if (!a->layers || a->layers > 1024 || !a->pages || a->pages > (1u << 27)) return false;
    auto tensor_ok = [&](uint64_t bytes, uint64_t page) {
        return page && page % 16 == 0 && page <= (1u << 30) && bytes / a->layers / a->pages == page && bytes == page * a->pages * a->layers;
    };
    if (!tensor_ok(a->len_bytes, a->page_bytes) || (kScales && !tensor_ok(scales_len_of(*a), scale_page_of(*a)))) return false;
    const Range r[3] = {{a->keys, a->len_bytes, 16}, {a->values, a->len_bytes, 16}, {scales_at(*a), scales_len_of(*a), 16}};
    if (!all_disjoint(r, kScales ? 3 : 2)) return false;
    return !full || inspect_device_ranges(d, r, kScales ? 3 : 2, failure);
}

template <uint32_t kPairs>
void launch_copies(cudaStream_t stream, uint32_t grid, const uint32_t* sources, const uint32_t* destinations, uint32_t count, const CopyParams& p) {
    PagePairs<kPairs> pairs{};
    for (uint32_t i = 0; i < count; ++i) pairs.source[i] = sources[i], pairs.destination[i] = destinations[i];
    launch_dependent(stream, kv_page_copy_kernel<kPairs>, grid, kCopyThreads, 0, pairs, p);
    count_launch();
}

// Destinations distinct, none of them a source, all inside the cache.
bool pairs_ok(uint32_t pages, const uint32_t* sources, const uint32_t* destinations, uint32_t count, bool* out_of_memory) {
    *out_of_memory = false;
    if (!sources || !destinations || count > pages) return false;
    for (uint32_t i = 0; i < count; ++i) {
        if (sources[i] >= pages || destinations[i] >= pages) return false;
    }
    if (count == 1) return sources[0] != destinations[0];
    uint8_t* taken = static_cast<uint8_t*>(std::calloc((pages + 7) / 8, 1));
    if (!taken) {
        *out_of_memory = true;
        return false;
    }
    bool fine = true;
    for (uint32_t i = 0; i < count && fine; ++i) {
        const uint32_t page = destinations[i];
        fine = (taken[page >> 3] >> (page & 7) & 1) == 0;
        taken[page >> 3] |= static_cast<uint8_t>(1u << (page & 7));
    }
    for (uint32_t i = 0; i < count && fine; ++i) fine = (taken[sources[i] >> 3] >> (sources[i] & 7) & 1) == 0;
    std::free(taken);
    return fine;
}

template <bool kScales, class Args>
augur_cuda_result_v1 submit_page_copy(int32_t d, augur_cuda_stream_t s, const Args* a, const uint32_t* sources, const uint32_t* destinations, uint32_t count) {
    augur_cuda_result_v1 failure;
    if (!check_page_copy<kScales>(d, s, a, false, &failure)) return failure;
    bool out_of_memory = false;
    if (count && !pairs_ok(a->pages, sources, destinations, count, &out_of_memory)) return out_of_memory ? make_result(AUGUR_CUDA_STATUS_OUT_OF_MEMORY) : invalid();
    if (consume_injected_fault()) return make_result(AUGUR_CUDA_STATUS_DIAGNOSTIC_FAULT_INJECTED);
    if (!count) return ok();
    const cudaError_t e = cudaSetDevice(d);
    if (e != cudaSuccess) return make_result(AUGUR_CUDA_STATUS_RUNTIME_FAILURE, e);
    CopyParams p{reinterpret_cast<uint8_t*>(a->keys), reinterpret_cast<uint8_t*>(a->values), reinterpret_cast<uint8_t*>(scales_at(*a)),
                 a->page_bytes, scale_page_of(*a), a->pages, a->layers, static_cast<uint32_t>((a->page_bytes + kCopyPiece - 1) / kCopyPiece),
                 static_cast<uint32_t>((scale_page_of(*a) + kCopyPiece - 1) / kCopyPiece)};
    const uint64_t per_pair = static_cast<uint64_t>(2 * p.pieces + p.scale_pieces) * a->layers;        // below 2^28
    const uint32_t most = static_cast<uint32_t>(per_pair * kPairsPerLaunch < INT32_MAX ? kPairsPerLaunch : INT32_MAX / per_pair);
    for (uint32_t at = 0; at < count;) {
        const uint32_t take = count - at < most ? count - at : most, grid = static_cast<uint32_t>(per_pair * take);
        if (take <= kFewPairs) {
            launch_copies<kFewPairs>(s->stream, grid, sources + at, destinations + at, take, p);
        } else {
            launch_copies<kPairsPerLaunch>(s->stream, grid, sources + at, destinations + at, take, p);
        }
        at += take;
    }
    return submitted();
}

}  // namespace
}  // namespace augur_sm100

using namespace augur_sm100;

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_append_preflight_v1(int32_t d, augur_cuda_stream_t s,
                                                                                            const augur_cuda_nvfp4_sm100_kv_append_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_append(d, s, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_append_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_kv_append_args_v1* a) {
    return submit_append<false>(d, s, a);
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_append_e4m3_preflight_v1(int32_t d, augur_cuda_stream_t s,
                                                                                                 const augur_cuda_nvfp4_sm100_kv_append_e4m3_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_append(d, s, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_append_e4m3_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_kv_append_e4m3_args_v1* a) {
    return submit_append<true>(d, s, a);
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_page_copy_preflight_v1(
    int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_kv_page_copy_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_page_copy<false>(d, s, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_page_copy_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_kv_page_copy_args_v1* a, const uint32_t* sources, const uint32_t* destinations,
    uint32_t count) {
    return submit_page_copy<false>(d, s, a, sources, destinations, count);
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_preflight_v1(
    int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_args_v1* a) {
    augur_cuda_result_v1 failure;
    return check_page_copy<true>(d, s, a, true, &failure) ? ok() : failure;
}

extern "C" augur_cuda_result_v1 AUGUR_CUDA_CALL augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_prevalidated_submit_v1(
    int32_t d, augur_cuda_stream_t s, const augur_cuda_nvfp4_sm100_kv_page_copy_e4m3_args_v1* a, const uint32_t* sources, const uint32_t* destinations,
    uint32_t count) {
    return submit_page_copy<true>(d, s, a, sources, destinations, count);
}
