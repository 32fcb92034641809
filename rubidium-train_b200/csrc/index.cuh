// index.cuh — index arithmetic that has to hold up to the ends of 32 bits, apart from the
// kernels so that a host compiler can check it.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define RBK_HD __host__ __device__ __forceinline__
#else
#define RBK_HD inline
#endif

namespace rbk {

// tk + sub, or the last of `tokens` (> 0) where that is at or behind the end: tk <= tokens, sub 0 or 1.
// tokens may be 2^31 - 1, so tk + sub may not fit an int, but fits 32 bits without a sign.
RBK_HD constexpr int token_at(int tk, int sub, int tokens) {
    const uint32_t at = (uint32_t)tk + (uint32_t)sub, last = (uint32_t)tokens - 1u;
    return (int)(at < last ? at : last);
}

}  // namespace rbk
