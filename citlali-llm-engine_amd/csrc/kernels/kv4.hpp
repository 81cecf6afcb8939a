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
// The mask lies in an SGPR and 1024 in a VGPR (an operand may not be a literal
// there); from C++ the compiler makes two instructions of it.
__device__ __forceinline__ uint32_t kv4_and_or(uint32_t w, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(bits));
    return r;
}
__device__ __forceinline__ void kv4_pairs(uint32_t w, f16x2 d, f16x2 m, f16x2 (&out)[4]) {
    constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u, k1024 = 0x64006400u;
    const f16x2 off{(_Float16)1024.f, (_Float16)1024.f};
    const f16x2 sixteenth{(_Float16)0.0625f, (_Float16)0.0625f}, off16{(_Float16)-64.f, (_Float16)-64.f};
    const uint32_t v = w >> 8;
    out[0] = as_h2(kv4_and_or(w, kLow, k1024)) - off;
    out[1] = __builtin_elementwise_fma(as_h2(kv4_and_or(w, kHigh, k1024)), sixteenth, off16);
    out[2] = as_h2(kv4_and_or(v, kLow, k1024)) - off;
    out[3] = __builtin_elementwise_fma(as_h2(kv4_and_or(v, kHigh, k1024)), sixteenth, off16);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = __builtin_elementwise_fma(out[i], d, m);
}

}  // namespace citlali::hip
