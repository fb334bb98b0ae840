// Device helpers shared by the serving kernels (kv_append.hip, prefix_attention.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace es
{

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float    float2_t __attribute__((ext_vector_type(2)));
typedef float    float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

// The sequence that owns `token`: the largest s < n with offsets[s] <= token (sequences
// without tokens share an offset; the last of them that starts there is the owner).  -1 where
// the token lies before the first or behind the last sequence.  The 64 lanes of a wavefront
// probe 64 places at once, so 4096 sequences take two dependent loads.  `token` is the same
// in all lanes, which all take part.  *first and *end receive the owner's offsets.
__device__ inline int find_sequence(const int* __restrict__ offsets, int n, int token, int* first,
                                    int* end)
{
    int const lane = int(threadIdx.x) & 63;
    int       lo = 0, len = n;
    while (len > 1) {
        int const      stride = (len + 63) >> 6;
        int const      at = lane * stride;
        bool const     below = at < len && offsets[lo + at] <= token;
        uint64_t const m = __ballot(below);
        int const      c = __popcll(m);
        if (c == 0) return -1;
        lo += (c - 1) * stride;
        len = min(stride, len - (c - 1) * stride);
    }
    *first = offsets[lo];
    *end = offsets[lo + 1];
    return (*first <= token && token < *end) ? lo : -1;
}

}  // namespace es
