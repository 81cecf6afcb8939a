// logprobs.hip -- log probability and rank of a given token, entropy and the
// most likely tokens of each row of logits.
#include "device_common.hpp"
#include "launch.hpp"

#include <math.h>

namespace citlali::hip {
namespace {

constexpr int kBlk = 256;

// Order of the tokens of a row: larger logit first, then the lower id, as one
// unsigned key; 0 (a NaN) is before nothing.  -0.0 counts as +0.0.
__device__ __forceinline__ uint64_t logit_key(float x, int id) {
    if (x != x) return 0ull;
    uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((uint64_t)u << 32) | (uint32_t)~(uint32_t)id;
}
__device__ __forceinline__ float key_logit(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

template <bool kHalf>
__device__ __forceinline__ float logit(const void* row, int i) {
    if constexpr (kHalf)
        return h2f(static_cast<const uint16_t*>(row)[i]);
    else
        return static_cast<const float*>(row)[i];
}

template <typename T, typename F>
__device__ T block_fold(T v, T* red, F f) {
    for (int o = 1; o < kWave; o <<= 1) v = f(v, (T)__shfl_xor(v, o, kWave));
    __syncthreads();
    if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
    __syncthreads();
    T r = red[0];
    for (int w = 1; w < kBlk / kWave; ++w) r = f(r, red[w]);
    return r;
}

// One workgroup per row, one pass over it for each thing asked for.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void logprobs_rows_kernel(Logprobs a) {
    __shared__ float redf[kBlk / kWave];
    __shared__ int redi[kBlk / kWave];
    __shared__ unsigned long long redk[kBlk / kWave];
    const int r = blockIdx.x;
    const void* row = static_cast<const char*>(a.logits) + (size_t)r * a.row_stride * (kHalf ? 2 : 4);
    float m = -INFINITY;
    int nan = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kBlk) {
        const float x = logit<kHalf>(row, i);
        nan |= x != x;
        m = fmaxf(m, x);
    }
    m = block_fold(m, redf, [](float p, float q) { return fmaxf(p, q); });
    nan = block_fold(nan, redi, [](int p, int q) { return p | q; });
    if (nan || m == INFINITY) m = NAN;
    float s = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < a.vocab; i += kBlk) {
        const float y = logit<kHalf>(row, i) - m;
        if (y == -INFINITY) continue;
        const float e = expf(y);
        s += e;
        t += e * y;
    }
    auto add = [](float p, float q) { return p + q; };
    s = block_fold(s, redf, add);
    t = block_fold(t, redf, add);
    const float lse = m == -INFINITY ? NAN : logf(s);
    if (a.entropies && threadIdx.x == 0) a.entropies[r] = lse - t / s;
    const int token = a.tokens ? a.tokens[r] : -1;
    if (a.tokens) {
        const bool given = token >= 0 && token < a.vocab;
        const float x = given ? logit<kHalf>(row, token) : 0.f;
        const uint64_t mine = given ? logit_key(x, token) : 0ull;
        int before = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kBlk) before += logit_key(logit<kHalf>(row, i), i) > mine;
        before = block_fold(before, redi, [](int p, int q) { return p + q; });
        if (threadIdx.x == 0) {
            if (a.logprobs) a.logprobs[r] = given ? x - m - lse : 0.f;
            if (a.ranks) a.ranks[r] = given ? before : -1;
        }
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < a.top_k; ++j) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kBlk) {
            const unsigned long long k = logit_key(logit<kHalf>(row, i), i);
            if (k < last && k > best) best = k;
        }
        last = block_fold(best, redk, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; });
        if (threadIdx.x == 0) {
            a.top_ids[(size_t)r * a.top_k + j] = last ? (int32_t)~(uint32_t)last : -1;
            a.top_logprobs[(size_t)r * a.top_k + j] = last ? key_logit(last) - m - lse : -INFINITY;
        }
    }
}

}  // namespace

size_t logprobs_workspace(int, int, int) { return 0; }

hipError_t launch_token_logprobs(const Logprobs& a, hipStream_t s) {
    if (a.half)
        launch_kernel(logprobs_rows_kernel<true>, dim3(a.rows), dim3(kBlk), 0, s, a);
    else
        launch_kernel(logprobs_rows_kernel<false>, dim3(a.rows), dim3(kBlk), 0, s, a);
    return hipGetLastError();
}

}  // namespace citlali::hip
