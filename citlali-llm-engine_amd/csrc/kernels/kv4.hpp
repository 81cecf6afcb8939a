// kv4.hpp -- layout of the paged cache of 4-bit keys and values (see
// citlali_hip_kv4_cache in citlali_hip.h) and the codes' arithmetic.
#pragma once

#include "device_common.hpp"
#include "launch.hpp"

namespace citlali::hip {

constexpr int kKv4Group = 32;            // dims of a token that share (d, m)
constexpr float kKv4Limit = 61440.f;     // 15 d + m stays finite in fp16 below this
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));

// Byte offsets in one kv head's part of a page of P tokens.
template <int HD>
struct Kv4Layout {
    static constexpr int kCodes = HD / 2;                // bytes of a token's K (or V) codes
    static constexpr int kParams = HD / kKv4Group * 4;   // bytes of its (d, m)
    static constexpr int kToken = 2 * (kCodes + kParams);
    __device__ static int k_params(int P) { return P * kCodes; }
    __device__ static int v_codes(int P) { return P * (kCodes + kParams); }
    __device__ static int v_params(int P) { return P * (2 * kCodes + kParams); }
};

// One kv head's part of a page.
template <int HD>
__device__ __forceinline__ uint8_t* kv4_head(const Kv4View& c, int page, int kv_head) {
    return c.pages + (((size_t)page * c.kv_heads + kv_head) << c.page_shift) * Kv4Layout<HD>::kToken;
}

// The fp16 values of 8 codes.  A K word holds dims 0 2 4 6 in its low half
// and 1 3 5 7 in its high half, so every pair (nibble i, nibble i + 4) is two
// neighbouring dims; OR-ed into the mantissa of 1024 (or, a nibble higher, as
// 16 q) a pair becomes fp16 in one instruction, 1024 comes off exactly, and one
// packed fma rounds d q + m once.  d and m: the pair's scales, one per half.
__device__ __forceinline__ f16x2 kv4_low(uint32_t w) {   // nibbles 0 and 4
    return __builtin_bit_cast(f16x2, (w & 0x000F000Fu) | 0x64006400u) - f16x2{(_Float16)1024.f, (_Float16)1024.f};
}
__device__ __forceinline__ f16x2 kv4_high(uint32_t w) {   // nibbles 1 and 5
    const f16x2 h = __builtin_bit_cast(f16x2, (w & 0x00F000F0u) | 0x64006400u);
    return __builtin_elementwise_fma(h, f16x2{(_Float16)0.0625f, (_Float16)0.0625f},
                                     f16x2{(_Float16)-64.f, (_Float16)-64.f});
}
__device__ __forceinline__ void kv4_pairs(uint32_t w, f16x2 d, f16x2 m, f16x2 (&out)[4]) {
    out[0] = __builtin_elementwise_fma(kv4_low(w), d, m);
    out[1] = __builtin_elementwise_fma(kv4_high(w), d, m);
    out[2] = __builtin_elementwise_fma(kv4_low(w >> 8), d, m);
    out[3] = __builtin_elementwise_fma(kv4_high(w >> 8), d, m);
}

}  // namespace citlali::hip
