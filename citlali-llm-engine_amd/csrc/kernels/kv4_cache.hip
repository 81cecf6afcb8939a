// kv4_cache.hip -- the paged cache of 4-bit keys and values: appending tokens
// (head norms, rotation and quantisation in one pass), reading slots back, and
// the rotation's table.
#include "kv4.hpp"

#include <math.h>

namespace citlali::hip {
namespace {

constexpr int kBlk = 256;

__global__ void rope_table_kernel(float2* __restrict__ table, size_t n, int half, double log_theta) {
    const size_t i = (size_t)blockIdx.x * kBlk + threadIdx.x;
    if (i >= n) return;
    const int pair = (int)(i % half);
    double sn, cs;
    sincos((double)(i / half) * exp(log_theta * ((double)-pair / half)), &sn, &cs);
    table[i] = make_float2((float)cs, (float)sn);
}

template <typename T>
__device__ __forceinline__ T add_lanes(T v, int lanes) {   // over aligned groups of `lanes` lanes
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o, kWave);
    return v;
}
__device__ __forceinline__ _Float16 half_at(u32x4 v, int i) {
    return __builtin_bit_cast(_Float16, (uint16_t)(v[i / 2] >> (16 * (i & 1))));
}

// The eight normed and rotated values of a lane in T.  Lane l of the LR that
// share a head row holds dims 8 l .. 8 l + 7; its rotation partner, LR / 2
// lanes away, holds the dims head_dim / 2 away.
template <typename T, int HD>
__device__ __forceinline__ void norm_rotate(u32x4 raw, const uint16_t* w, float eps, const float* rope_row, int l,
                                            T (&y)[8]) {
    constexpr int LR = HD / 8;
    u32x4 other;
#pragma unroll
    for (int i = 0; i < 4; ++i) other[i] = __shfl_xor(raw[i], LR / 2, kWave);
    T x[8], p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = (T)(float)half_at(raw, i);
        p[i] = (T)(float)half_at(other, i);
    }
    if (w != nullptr) {
        T s = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += x[i] * x[i];
        s = add_lanes(s, LR);
        const T inv = (T)1 / sqrt(s / (T)HD + (T)eps);
        const u32x4 wx = *reinterpret_cast<const u32x4*>(w + 8 * l);
        const u32x4 wp = *reinterpret_cast<const u32x4*>(w + 8 * (l ^ (LR / 2)));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = x[i] * inv * (T)(float)half_at(wx, i);
            p[i] = p[i] * inv * (T)(float)half_at(wp, i);
        }
    }
    const float2* cs = reinterpret_cast<const float2*>(rope_row) + 8 * (l & (LR / 2 - 1));
    const bool upper = l >= LR / 2;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 t = cs[i];
        y[i] = upper ? p[i] * (T)t.y + x[i] * (T)t.x : x[i] * (T)t.x - p[i] * (T)t.y;
    }
}

// Codes of a lane's eight values; d and m (fp16 bits) are those of the four
// lanes that share a group.
__device__ __forceinline__ void quantise(const float (&in)[8], uint32_t (&code)[8], uint32_t& d16, uint32_t& m16) {
#pragma clang fp contract(off)   // the codes are the formula's, with its division by d
    float y[8], lo = INFINITY, hi = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        bad |= in[i] != in[i];
        y[i] = fminf(fmaxf(in[i], -kKv4Limit), kKv4Limit);
        lo = fminf(lo, y[i]);
        hi = fmaxf(hi, y[i]);
    }
    if (bad) lo = -INFINITY;   // stays the least of the four lanes
    lo = fminf(lo, dpp<kDppXor1>(lo));
    lo = fminf(lo, dpp<kDppXor2>(lo));
    hi = fmaxf(hi, dpp<kDppXor1>(hi));
    hi = fmaxf(hi, dpp<kDppXor2>(hi));
    bad = lo == -INFINITY;
    m16 = bad ? 0x7e00u : f2h_rne(lo);
    const float m = h2f((uint16_t)m16);
    float step = (hi - m) * (1.f / 15.f);
    asm("" : "+v"(step));   // rounded to fp32 before fp16: no v_fma_mixlo_f16
    d16 = bad ? 0u : f2h_rne(step);
    const float d = h2f((uint16_t)d16);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = d > 0.f ? rintf((y[i] - m) / d) : 0.f;
        code[i] = bad ? 0u : (uint32_t)fminf(fmaxf(c, 0.f), 15.f);
    }
}

// One wave takes one head (query, key or value) of 512 / HD consecutive
// tokens, 16 bytes a lane.
template <int HD>
__global__ __launch_bounds__(kBlk) void kv4_append_kernel(Kv4View c, Kv4Append a) {
    constexpr int LR = HD / 8, kRows = kWave / LR;
    using L = Kv4Layout<HD>;
    const int lane = threadIdx.x & (kWave - 1), l = lane % LR;
    const int slots_per_token = a.heads + 2 * c.kv_heads;
    const long long unit = (long long)blockIdx.x * (kBlk / kWave) + threadIdx.x / kWave;
    const int head = (int)(unit % slots_per_token);
    const long long t = unit / slots_per_token * kRows + lane / LR;
    // rows past the last token, and tokens without a position, take part in
    // the lane moves with row 0 and write nothing
    const bool real = t < a.tokens;
    const long long row = real ? t : 0;
    const int pos = a.positions[row];
    const bool known = real && pos >= 0 && pos < a.rope_positions;
    const float* rope_row = a.rope + (size_t)(known ? pos : 0) * HD;

    if (head < a.heads) {
        const u32x4 raw = *reinterpret_cast<const u32x4*>(a.q + row * a.q_stride + (size_t)head * HD + 8 * l);
        float y[8];
        norm_rotate<float, HD>(raw, a.q_norm, a.eps, rope_row, l, y);
        if (known) {
            u32x4 o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = f2h_rne(y[2 * i]) | ((uint32_t)f2h_rne(y[2 * i + 1]) << 16);
            *reinterpret_cast<u32x4*>(a.q_out + row * a.q_out_stride + (size_t)head * HD + 8 * l) = o;
        }
        return;
    }
    const bool is_k = head < a.heads + c.kv_heads;
    const int kvh = head - a.heads - (is_k ? 0 : c.kv_heads);
    const u32x4 raw =
        *reinterpret_cast<const u32x4*>((is_k ? a.k : a.v) + row * a.kv_stride + (size_t)kvh * HD + 8 * l);
    const int slot = a.slots[row];
    const int P = 1 << c.page_shift;
    const bool kept = known && slot >= 0 && (slot >> c.page_shift) < c.num_pages;
    uint8_t* base = kv4_head<HD>(c, kept ? slot >> c.page_shift : 0, kvh);
    const int o = slot & (P - 1);
    float y[8];
    uint32_t code[8], d16, m16;
    if (is_k) {
        double z[8];
        norm_rotate<double, HD>(raw, a.k_norm, a.eps, rope_row, l, z);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (float)z[i];
        quantise(y, code, d16, m16);
        if (!kept) return;
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= (code[2 * i] | (code[2 * i + 1] << 16)) << (4 * i);
        *reinterpret_cast<uint32_t*>(base + o * L::kCodes + 4 * l) = w;
        if ((l & 3) == 0)
            *reinterpret_cast<uint32_t*>(base + L::k_params(P) + o * L::kParams + l) = d16 | (m16 << 16);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (float)half_at(raw, i);
    quantise(y, code, d16, m16);
    if (!kept) return;
    uint16_t* vc = reinterpret_cast<uint16_t*>(base + L::v_codes(P)) + (o >> 2) * HD + (o & 3);
#pragma unroll
    for (int e = 0; e < 2; ++e)
        vc[(2 * l + e) * 4] =
            (uint16_t)(code[4 * e] | (code[4 * e + 1] << 4) | (code[4 * e + 2] << 8) | (code[4 * e + 3] << 12));
    if ((l & 3) == 0) {
        uint16_t* vp = reinterpret_cast<uint16_t*>(base + L::v_params(P)) +
                       ((o >> 2) * (HD / kKv4Group) + (l >> 2)) * 8 + (o & 3);
        vp[0] = (uint16_t)d16;
        vp[4] = (uint16_t)m16;
    }
}

// Lanes as in the append: one wave reads the K or V values of one head in
// 512 / HD slots.
template <int HD>
__global__ __launch_bounds__(kBlk) void kv4_read_kernel(Kv4View c, const int32_t* __restrict__ slots, int count,
                                                        uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
    constexpr int LR = HD / 8, kRows = kWave / LR;
    using L = Kv4Layout<HD>;
    const int lane = threadIdx.x & (kWave - 1), l = lane % LR;
    const long long unit = (long long)blockIdx.x * (kBlk / kWave) + threadIdx.x / kWave;
    const int head = (int)(unit % (2 * c.kv_heads));
    const long long t = unit / (2 * c.kv_heads) * kRows + lane / LR;
    if (t >= count) return;
    const bool is_k = head < c.kv_heads;
    const int kvh = is_k ? head : head - c.kv_heads;
    const int slot = slots[t];
    const int P = 1 << c.page_shift, o = slot & (P - 1);
    u32x4 out{0u, 0u, 0u, 0u};
    if (slot >= 0 && (slot >> c.page_shift) < c.num_pages) {
        const uint8_t* base = kv4_head<HD>(c, slot >> c.page_shift, kvh);
        f16x2 v[4];
        if (is_k) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(base + o * L::kCodes + 4 * l);
            const f16x2 dm = as_h2(
                *reinterpret_cast<const uint32_t*>(base + L::k_params(P) + o * L::kParams + (l & ~3)));
            kv4_pairs(w, f16x2{dm.x, dm.x}, f16x2{dm.y, dm.y}, v);
        } else {
            const uint16_t* vc = reinterpret_cast<const uint16_t*>(base + L::v_codes(P)) + (o >> 2) * HD + (o & 3);
            const _Float16* vp = reinterpret_cast<const _Float16*>(base + L::v_params(P)) +
                                 ((o >> 2) * (HD / kKv4Group) + (l >> 2)) * 8 + (o & 3);
            const _Float16 d = vp[0], m = vp[4];
            const uint32_t lo = vc[8 * l], hi = vc[8 * l + 4];
            f16x2 s[4];   // pair i: dims i and i + 4 of the lane
            kv4_pairs(lo | (hi << 16), f16x2{d, d}, f16x2{m, m}, s);
            v[0] = f16x2{s[0].x, s[1].x};
            v[1] = f16x2{s[2].x, s[3].x};
            v[2] = f16x2{s[0].y, s[1].y};
            v[3] = f16x2{s[2].y, s[3].y};
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = __builtin_bit_cast(uint32_t, v[i]);
    }
    *reinterpret_cast<u32x4*>((is_k ? k_out : v_out) + ((size_t)t * c.kv_heads + kvh) * HD + 8 * l) = out;
}

}  // namespace

bool kv4_shape_ok(int page_size, int head_dim) {
    return (head_dim == 64 || head_dim == 128) && page_size >= 16 && page_size <= 256 &&
           (page_size & (page_size - 1)) == 0;
}

hipError_t launch_rope_table(float* table, int positions, int head_dim, float theta, hipStream_t s) {
    const int half = head_dim / 2;
    const size_t n = (size_t)positions * half;
    launch_kernel(rope_table_kernel, dim3((unsigned)((n + kBlk - 1) / kBlk)), dim3(kBlk), 0, s,
                  reinterpret_cast<float2*>(table), n, half, log((double)theta));
    return hipGetLastError();
}

namespace {
unsigned blocks_for(long long rows, int head_dim, long long heads) {
    const long long per_wave = 512 / head_dim;
    const long long waves = (rows + per_wave - 1) / per_wave * heads;
    return (unsigned)((waves + kBlk / kWave - 1) / (kBlk / kWave));
}
}  // namespace

hipError_t launch_kv4_append(const Kv4View& c, const Kv4Append& a, hipStream_t s) {
    const dim3 grid(blocks_for(a.tokens, c.head_dim, a.heads + 2 * c.kv_heads));
    if (c.head_dim == 128)
        launch_kernel(kv4_append_kernel<128>, grid, dim3(kBlk), 0, s, c, a);
    else
        launch_kernel(kv4_append_kernel<64>, grid, dim3(kBlk), 0, s, c, a);
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4View& c, const int32_t* slots, int count, uint16_t* k_out, uint16_t* v_out,
                           hipStream_t s) {
    const dim3 grid(blocks_for(count, c.head_dim, 2 * c.kv_heads));
    if (c.head_dim == 128)
        launch_kernel(kv4_read_kernel<128>, grid, dim3(kBlk), 0, s, c, slots, count, k_out, v_out);
    else
        launch_kernel(kv4_read_kernel<64>, grid, dim3(kBlk), 0, s, c, slots, count, k_out, v_out);
    return hipGetLastError();
}

}  // namespace citlali::hip
