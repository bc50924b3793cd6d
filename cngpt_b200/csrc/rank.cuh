// rank.cuh - the ranking of one row's logits that sampling and top-k share.
#pragma once

#include <cstdint>

namespace cg {

// Order-preserving bits of a logit: a < b exactly if key(a) < key(b), -0 and 0
// have one key, NaN has the lowest (0, below -inf's).
__device__ __forceinline__ uint32_t rank_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

__device__ __forceinline__ float rank_value(uint32_t k) {
    if (k == 0u) return __uint_as_float(0x7FFFFFFFu);
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

constexpr uint32_t RANK_NEG_INF = 0x007FFFFFu;  // rank_key(-inf): keys above it can be drawn

}  // namespace cg
