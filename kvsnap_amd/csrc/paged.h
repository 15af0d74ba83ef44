// Device helpers of the operators over a paged KV cache (include/kvsnap_attention.h): value types, divisions by
// sizes known at launch, and finding the sequence that a row belongs to.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/kvsnap_attention.h"

#include <cstdint>
#include <cstring>

namespace kvsnap {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

template <typename To, typename From>
__device__ __forceinline__ To bits(From x) {
    static_assert(sizeof(To) == sizeof(From), "a view of the same bits");
    return __builtin_bit_cast(To, x);
}

// n / d for 0 <= n < 2^32 by a multiplication and shifts (the round-up method of Granlund and Montgomery, "Division
// by Invariant Integers using Multiplication"): a 32-bit division is some 25 instructions here.
struct Divider {
    uint32_t d, multiplier, shift;

    static Divider of(uint32_t d) {
        uint32_t s = 0;
        while (s < 32 && (uint64_t(1) << s) < d) ++s;
        const uint64_t m = ((uint64_t(1) << 32) * ((uint64_t(1) << s) - d)) / d + 1;
        return Divider{d, static_cast<uint32_t>(m), s};
    }
    __device__ __forceinline__ uint32_t divide(uint32_t n) const {
        if (shift == 0) return n;
        const uint32_t t = __umulhi(multiplier, n);
        return (t + ((n - t) >> 1)) >> (shift - 1);
    }
};

// The value of an e8m0 byte: 2^(e - 127), NaN for 255.
__device__ __forceinline__ float power_of(uint32_t e) {
    return bits<float>(e == 255 ? 0x7fc00000u : e == 0 ? 0x00400000u : e << 23);
}

// Rows of sequence s, clamped to the `tokens` rows that there are: tables live in device memory, and a wrong one
// must not send an access out of its tensor.
struct Rows {
    int first, count;
};

__device__ __forceinline__ Rows rows_of(const kvsnap_sequences& q, int s, int tokens) {
    if (!q.query_starts) return Rows{s, s < tokens ? 1 : 0};
    const int first = min(max(q.query_starts[s], 0), tokens), end = min(max(q.query_starts[s + 1], 0), tokens);
    return Rows{first, max(end - first, 0)};
}

// Tokens of sequence s, at most 2^30 (no table names more) so that no position near them overflows, and those of them
// that its table row can name.
__device__ __forceinline__ int length_of(const kvsnap_sequences& q, int s) { return min(max(q.lengths[s], 0), 1 << 30); }
__device__ __forceinline__ int named_of(const kvsnap_sequences& q, int length, int block_size) {
    const int64_t named = int64_t(q.table_width) * block_size;
    return length < named ? length : static_cast<int>(named);
}

// The last sequence s with share(s) <= want, where share rises with s: each step of the search reads 64 entries
// with the wave's 64 lanes, so 64 sequences take one load's latency and 4096 two.  Wave-uniform `want`.
template <typename Share>
__device__ __forceinline__ int find_sequence(int n_seqs, int64_t want, Share share) {
    const int lane = __lane_id();
    int low = 0, high = n_seqs;
    while (high - low > 1) {
        const int step = (high - low + 63) >> 6;
        const int at = low + lane * step;
        const uint64_t below = __ballot(at < high && share(at) <= want);
        const int passed = __popcll(below);
        const int next = low + (passed > 0 ? passed - 1 : 0) * step;
        high = min(high, next + step);
        low = next;
        if (step == 1) break;
    }
    return __builtin_amdgcn_readfirstlane(low);
}

}  // namespace kvsnap
