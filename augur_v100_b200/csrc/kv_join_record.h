// What the join of the paged attention knows of a pair that several spans share, and the check that keeps it inside its tensors. Plain C++ outside
// nvcc, where a test compares the check with the rule over records of any bits.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define AUGUR_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define AUGUR_HOST_DEVICE inline
#endif

namespace augur_sm100 {

// tokens 0: of no pair. Records are by pair or, where there are more pairs than spans, by the span that holds the pair's first part.
struct JoinRecord {
    uint32_t row, tokens, head, first, last;   // first token row, new tokens, key-value head, first and last span
    uint32_t reserved[3];
};

// A launch that gave up leaves in a record's place whatever was there: a record of an earlier launch, or another operator's partial sums. So nothing may
// wrap round: sums and products in 64 bits.
AUGUR_HOST_DEVICE bool join_record_ok(const JoinRecord& r, uint32_t group, uint32_t columns, uint32_t rows, uint32_t kv_heads, uint32_t spans) {
    return static_cast<uint64_t>(r.tokens) * group <= columns && static_cast<uint64_t>(r.row) + r.tokens <= rows && r.head < kv_heads && r.first <= r.last && r.last < spans;
}

}  // namespace augur_sm100
