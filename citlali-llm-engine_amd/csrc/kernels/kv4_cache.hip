// kv4_cache.hip -- the paged cache of 4-bit keys and values: appending tokens
// (head norms, rotation and quantisation in one pass), reading slots back, moving
// those that stay up within their sequences, and the rotation's table.
#include "kv4.hpp"

#include <math.h>

#include <algorithm>

namespace citlali::hip {
namespace {

constexpr int kBlk = 256;
constexpr long long kEnoughWaves = 4096;

__global__ void rope_table_kernel(float2* __restrict__ table, size_t n, int half, double log_theta) {
    const size_t i = (size_t)blockIdx.x * kBlk + threadIdx.x;
    if (i >= n) return;
    const int pair = (int)(i % half);
    double sn, cs;
    sincos((double)(i / half) * exp(log_theta * ((double)-pair / half)), &sn, &cs);
    table[i] = make_float2((float)cs, (float)sn);
}

__device__ __forceinline__ _Float16 half_at(u32x4 v, int i) {
    return __builtin_bit_cast(_Float16, (uint16_t)(v[i / 2] >> (16 * (i & 1))));
}

// Sum over the LR lanes that share a head row (LR = 8 or 16).
template <int LR>
__device__ __forceinline__ float row_sum(float v) {
    return lane_group_sum<LR>(v);
}
template <int Ctrl>
__device__ __forceinline__ double dpp64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, Ctrl, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), Ctrl, 0xF, 0xF, false);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
template <int LR>
__device__ __forceinline__ double row_sum(double v) {
    v += dpp64<kDppXor1>(v);
    v += dpp64<kDppXor2>(v);
    v += dpp64<kDppHalfMirror>(v);
    if constexpr (LR == 16) v += dpp64<kDppMirror>(v);
    return v;
}
// The value LR / 2 lanes away in the row.
template <int LR>
__device__ __forceinline__ uint32_t partner(uint32_t v) {
    if constexpr (LR == 16)
        return __builtin_amdgcn_update_dpp(0, (int)v, DppRor<8>::value, 0xF, 0xF, false);
    else
        return __shfl_xor((int)v, LR / 2, kWave);
}

// x^-1/2 of a positive number, 0 of infinity: the hardware's estimate, in 64 bits
// one Newton step further (its error, about 2^-29, squared), which a 0 does without
// (its x r would be a NaN).
__device__ __forceinline__ float inv_root(float x) { return __builtin_amdgcn_rsqf(x); }
__device__ __forceinline__ double inv_root(double x) {
    const double r = __builtin_amdgcn_rsq(x);
    return r == 0.0 ? 0.0 : fma(0.5 * r, fma(-x * r, r, 1.0), r);
}

// Norm and rotation of a lane's eight values, in T.  Lane l of the LR that share
// a head row holds dims 8 l .. 8 l + 7; its rotation partner, LR / 2 lanes away,
// holds the dims head_dim / 2 away.  y = inv (x a + p b), inv the norm's factor,
// a = w_x cos and b = -+ w_p sin once for all heads (wx, wp: the norm's weights of
// both lanes, ones without a norm; cs: cosines and sines of the eight pairs).
// In 64 bits a, b and x a are exact.
template <typename T, int HD>
struct Rotation {
    static constexpr int LR = HD / 8;
    T a[8], b[8];
    __device__ Rotation(const float2 (&cs)[8], u32x4 wx, u32x4 wp, int l) {
        const uint32_t flip = l < LR / 2 ? 0x80000000u : 0u;   // the lower half of the pairs takes - sin
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = (T)(float)half_at(wx, i) * (T)cs[i].x;
            b[i] = (T)(float)half_at(wp, i) * (T)__uint_as_float(__float_as_uint(cs[i].y) ^ flip);
        }
    }
    __device__ void operator()(u32x4 raw, bool norm, float eps, float (&y)[8]) const {
        u32x4 other;
#pragma unroll
        for (int i = 0; i < 4; ++i) other[i] = partner<LR>(raw[i]);
        T inv = 1;
        if (norm) {
            T s = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const T x = (T)(float)half_at(raw, i);
                s += x * x;
            }
            inv = inv_root(row_sum<LR>(s) * (T)(1.0 / HD) + (T)eps);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = (float)(inv * ((T)(float)half_at(raw, i) * a[i] + (T)(float)half_at(other, i) * b[i]));
    }
};

// Codes of a lane's eight values, four to a number: lo has those of values 0
// .. 3 (or, kEven, of 0 2 4 6) from the low bits on, hi the others.  d and m
// (fp16 bits) are those of the four lanes that share a group.
// (y - m) / d rounded as fp32 division rounds it, from d's reciprocal: that is
// correctly rounded after one Newton step for every fp16 d, and then one step
// on the quotient is exact.
template <bool kEven>
__device__ __forceinline__ void quantise(const float (&y)[8], uint32_t& lo, uint32_t& hi, uint32_t& d16,
                                         uint32_t& m16) {
    // a NaN stays through these two
    auto min3 = [](float a, float b, float c) {
        float r;
        asm("v_minimum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
        return r;
    };
    auto max3 = [](float a, float b, float c) {
        float r;
        asm("v_maximum3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
        return r;
    };
    float least = min3(min3(y[0], y[1], y[2]), min3(y[3], y[4], y[5]), min3(y[6], y[7], y[7]));
    float most = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), max3(y[6], y[7], y[7]));
    const float l1 = dpp<kDppXor1>(least), m1 = dpp<kDppXor1>(most);
    least = min3(least, l1, l1);
    most = max3(most, m1, m1);
    const float l2 = dpp<kDppXor2>(least), m2 = dpp<kDppXor2>(most);
    least = min3(least, l2, l2);
    most = max3(most, m2, m2);
    const bool bad = least != least;
    least = __builtin_amdgcn_fmed3f(least, -kKv4Limit, kKv4Limit);
    most = __builtin_amdgcn_fmed3f(most, -kKv4Limit, kKv4Limit);
    m16 = f2h_rne(least);
    const float m = bad ? 0.f : h2f((uint16_t)m16);
    float step = (most - m) * (1.f / 15.f);
    asm("" : "+v"(step));   // rounded to fp32 before fp16: no v_fma_mixlo_f16
    d16 = bad ? 0u : f2h_rne(step);
    m16 = bad ? 0x7e00u : m16;
    const float d = h2f((uint16_t)d16), top = 15.f * d;
    float r = __builtin_amdgcn_rcpf(d);
    r = d > 0.f ? fmaf(fmaf(-d, r, 1.f), r, r) : 0.f;
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = __builtin_amdgcn_fmed3f(y[i] - m, 0.f, top);   // codes 0 .. 15; saturation as well
        const float q = x * r;
        c[i] = rintf(fmaf(fmaf(-q, d, x), r, q));
    }
    auto four = [](float c0, float c1, float c2, float c3) {   // whole numbers below 2^16
        return (uint32_t)fmaf(fmaf(fmaf(c3, 16.f, c2), 16.f, c1), 16.f, c0);
    };
    lo = kEven ? four(c[0], c[2], c[4], c[6]) : four(c[0], c[1], c[2], c[3]);
    hi = kEven ? four(c[1], c[3], c[5], c[7]) : four(c[4], c[5], c[6], c[7]);
    lo = bad ? 0u : lo;
    hi = bad ? 0u : hi;
}

// One wave takes `per` heads (all query, key or value heads) of 512 / HD
// consecutive tokens, 16 bytes a lane and head, the next head's on their way:
// the rotation's 64 bytes a lane, four times a head's, are read once for all.
// Bound by HBM: 8192 tokens of 32/8 heads move 182 MB in 43.7 us (4.2 TB/s; a
// copy of as many bytes takes 36), with the streams read and written
// nontemporal (4 us more without); few tokens (250: 4.8 us, one: 3.6) by the
// chain position -> table -> head.
template <int HD>
__global__ __launch_bounds__(kBlk) void kv4_append_kernel(Kv4View c, Kv4Append a, int per) {
    constexpr int LR = HD / 8, kRows = kWave / LR;
    using L = Kv4Layout<HD>;
    const int lane = threadIdx.x & (kWave - 1), l = lane % LR;
    const int q_units = (a.heads + per - 1) / per, kv_units = (c.kv_heads + per - 1) / per;
    const int units = q_units + 2 * kv_units;
    const uint32_t at = blockIdx.x * (kBlk / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const long long group = at / (uint32_t)units;
    if (group * kRows >= a.tokens) return;   // uniform
    int unit = (int)(at % (uint32_t)units);
    const bool is_q = unit < q_units, is_v = unit >= q_units + kv_units;
    unit -= is_q ? 0 : is_v ? q_units + kv_units : q_units;
    const int h0 = unit * per, h1 = min(is_q ? a.heads : c.kv_heads, h0 + per);
    // rows past the last token, and tokens without a position, take part in
    // the lane moves with row 0 and write nothing
    const long long t = group * kRows + lane / LR;
    const bool real = t < a.tokens;
    const long long row = real ? t : 0;
    const uint16_t* src = (is_q ? a.q + row * a.q_stride : (is_v ? a.v : a.k) + row * a.kv_stride) + 8 * l;
    const int pos = a.positions[row], slot = a.slots[row];
    const bool known = real && pos >= 0 && pos < a.rope_positions;
    const int P = 1 << c.page_shift, o = slot & (P - 1);
    const bool kept = known && slot >= 0 && (slot >> c.page_shift) < c.num_pages;

    float2 cs[8];
    const uint32_t ones = 0x3c003c00u;
    u32x4 wx{ones, ones, ones, ones}, wp = wx;
    const uint16_t* w = is_q ? a.q_norm : a.k_norm;
    if (!is_v) {
        const float2* rope =
            reinterpret_cast<const float2*>(a.rope + (size_t)(known ? pos : 0) * HD) + 8 * (l & (LR / 2 - 1));
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = rope[i];
        if (w != nullptr) {
            wx = *reinterpret_cast<const u32x4*>(w + 8 * l);
            wp = *reinterpret_cast<const u32x4*>(w + 8 * (l ^ (LR / 2)));
        }
    }
    // values of neighbouring slots (an even one and the next) in neighbouring
    // rows go out as words of two tokens
    bool pairs = false;
    if (is_v) {
        const int next = __shfl_xor(slot, LR, kWave);
        const bool even = ((lane / LR) & 1) == 0;
        const bool good = kept && (even ? (slot & 1) == 0 && next == slot + 1 : (slot & 1) == 1 && next == slot - 1);
        pairs = LR == 16 && __builtin_amdgcn_ballot_w64(!good) == 0;
    }

    u32x4 next = *reinterpret_cast<const u32x4*>(src + (size_t)h0 * HD);
    auto head = [&](int h) {   // head h; the next one's are on their way
        const u32x4 raw = next;
        const uint16_t* ahead = src + (size_t)min(h + 1, h1 - 1) * HD;
        next = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(ahead));
        return raw;
    };
    float y[8];
    if (is_q) {
        const Rotation<float, HD> rotate(cs, wx, wp, l);
#pragma unroll 1
        for (int h = h0; h < h1; ++h) {
            rotate(head(h), w != nullptr, a.eps, y);
            if (!known) continue;
            u32x4 out;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                out[i] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)y[2 * i], (_Float16)y[2 * i + 1]});
            uint16_t* to = a.q_out + row * a.q_out_stride + (size_t)h * HD + 8 * l;
            __builtin_nontemporal_store(out, reinterpret_cast<u32x4*>(to));
        }
        return;
    }
    uint32_t lo, hi, d16, m16;
    uint8_t* const page = kv4_head<HD>(c, kept ? slot >> c.page_shift : 0, 0);
    const size_t head_bytes = (size_t)L::kToken << c.page_shift;
    if (!is_v) {
        const Rotation<double, HD> rotate(cs, wx, wp, l);
#pragma unroll 1
        for (int h = h0; h < h1; ++h) {
            rotate(head(h), w != nullptr, a.eps, y);
            quantise<true>(y, lo, hi, d16, m16);
            if (!kept) continue;
            uint8_t* base = page + h * head_bytes;
            *reinterpret_cast<uint32_t*>(base + o * L::kCodes + 4 * l) = lo | (hi << 16);
            if ((l & 3) == 0)
                *reinterpret_cast<uint32_t*>(base + L::k_params(P) + o * L::kParams + l) = d16 | (m16 << 16);
        }
        return;
    }
#pragma unroll 1
    for (int h = h0; h < h1; ++h) {
        const u32x4 raw = head(h);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (float)half_at(raw, i);
        quantise<false>(y, lo, hi, d16, m16);   // dims 8 l .. and 8 l + 4 ..
        uint8_t* base = page + h * head_bytes;
        uint16_t* vc = reinterpret_cast<uint16_t*>(base + L::v_codes(P)) + (o >> 2) * HD;
        if (pairs) {
            // row r gets both tokens' quad r & 1 (see swap16)
            float q0 = __builtin_bit_cast(float, lo), q1 = __builtin_bit_cast(float, hi);
            swap16(q0, q1);
            *reinterpret_cast<uint32_t*>(vc + (2 * l + ((lane / LR) & 1)) * 4 + (o & 2)) =
                __builtin_bit_cast(uint32_t, q0) | (__builtin_bit_cast(uint32_t, q1) << 16);
        } else if (kept) {
            vc[2 * l * 4 + (o & 3)] = (uint16_t)lo;
            vc[(2 * l + 1) * 4 + (o & 3)] = (uint16_t)hi;
        }
        if (kept && (l & 3) == 0) {
            uint16_t* vp = reinterpret_cast<uint16_t*>(base + L::v_params(P)) +
                           ((o >> 2) * (HD / kKv4Group) + (l >> 2)) * 8 + (o & 3);
            vp[0] = (uint16_t)d16;
            vp[4] = (uint16_t)m16;
        }
    }
}

// Lanes as in the append: one wave reads the K and V values of one head in
// 512 / HD slots.  8192 slots of 8 heads of 128, 44 MB, in 10.4 us
// (4.2 TB/s; K and V in a wave each 11.8).
template <int HD>
__global__ __launch_bounds__(kBlk) void kv4_read_kernel(Kv4View c, const int32_t* __restrict__ slots, int count,
                                                        uint16_t* __restrict__ k_out, uint16_t* __restrict__ v_out) {
    constexpr int LR = HD / 8, kRows = kWave / LR;
    using L = Kv4Layout<HD>;
    const int lane = threadIdx.x & (kWave - 1), l = lane % LR;
    const uint32_t unit = blockIdx.x * (kBlk / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t group = unit / (uint32_t)c.kv_heads;
    const int kvh = (int)(unit - group * c.kv_heads);
    const long long t = (long long)group * kRows + lane / LR;
    if (t >= count) return;
    const int slot = slots[t];
    const int P = 1 << c.page_shift, o = slot & (P - 1);
    u32x4 k{0u, 0u, 0u, 0u}, v = k;
    if (slot >= 0 && (slot >> c.page_shift) < c.num_pages) {
        const uint8_t* base = kv4_head<HD>(c, slot >> c.page_shift, kvh);
        const uint32_t w = *reinterpret_cast<const uint32_t*>(base + o * L::kCodes + 4 * l);
        const f16x2 dm =
            as_h2(*reinterpret_cast<const uint32_t*>(base + L::k_params(P) + o * L::kParams + (l & ~3)));
        const uint16_t* vc = reinterpret_cast<const uint16_t*>(base + L::v_codes(P)) + (o >> 2) * HD + (o & 3);
        const _Float16* vp = reinterpret_cast<const _Float16*>(base + L::v_params(P)) +
                             ((o >> 2) * (HD / kKv4Group) + (l >> 2)) * 8 + (o & 3);
        const _Float16 d = vp[0], m = vp[4];
        const uint32_t lo = vc[8 * l], hi = vc[8 * l + 4];
        f16x2 e[4];
        kv4_pairs(w, f16x2{dm.x, dm.x}, f16x2{dm.y, dm.y}, e);
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = __builtin_bit_cast(uint32_t, e[i]);
        kv4_pairs(lo | (hi << 16), f16x2{d, d}, f16x2{m, m}, e);   // pair i: dims i and i + 4 of the lane
        const f16x2 in_order[4] = {{e[0].x, e[1].x}, {e[2].x, e[3].x}, {e[0].y, e[1].y}, {e[2].y, e[3].y}};
        v = __builtin_bit_cast(u32x4, in_order);
    }
    const size_t at = ((size_t)t * c.kv_heads + kvh) * HD + 8 * l;
    __builtin_nontemporal_store(k, reinterpret_cast<u32x4*>(k_out + at));
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(v_out + at));
}

// ---------------------------------------------------------------------------
// Position first[s] + kept[s][j] of sequence s moves to first[s] + j.  One workgroup
// per (kv head, sequence, cache), and one more for the V codes, which are as many
// bytes as the rest, takes its moves in order, some hundred at a time:
// all are read before any is written, so that a position which one of them takes
// may be where another comes from.  Later moves come from behind (kept ascends), so
// the next ones are read before these are written.
// kQuad lanes take four positions of the target in a row: for K 16 bytes of a token's
// codes or its params, for V a word of the four tokens' codes or params, gathered from
// four places and stored at once.  Where the tokens come from and go to is looked up
// for kAhead of them at a time, a thread a token.
// Bound by HBM: 3500 of 8000 positions of 4 sequences, 8 heads of 128, in 12 caches, 187
// MB to read and as many to write, in 114 to 122 us.  V's quads, of which nearly all have
// a position that stays, are read whole, and K's lines of two: 272 MB read by the
// counters, 3.8 to 4 TB/s in all.  (A wave a token with 2-byte pieces of V: 1227 us.  One
// turn's reads ahead instead of two: 118 for 114.)
// ---------------------------------------------------------------------------
constexpr int kKeepWaves = 8, kAhead = 2048;
template <int HD>
struct KeepTurn {
    static constexpr int kQuad = HD / 4;   // lanes of four tokens
    static constexpr int kSteps = 4;
    static constexpr int kTokens = kSteps * 4 * (kWave / kQuad);   // of a wave
    static_assert(kAhead % (kKeepWaves * kTokens) == 0);
};
template <int HD>
__global__ __launch_bounds__(kKeepWaves * kWave) void kv4_keep_kernel(Kv4View c, Kv4Keep a) {
    using L = Kv4Layout<HD>;
    using T = KeepTurn<HD>;
    constexpr int kSteps = T::kSteps, kTokens = T::kTokens;
    constexpr int kCodeLanes = HD / 8, kKLanes = kCodeLanes + 4;   // of K: 16-byte pieces, then params
    constexpr int kVCodes = HD / 4, kVParams = HD / 16;            // words of V a quad of tokens
    static_assert(kKLanes + kVParams <= T::kQuad && kVCodes <= T::kQuad);
    // the parts of pages (their first byte << 8 | row) that tokens come from and go to;
    // -1 for none
    __shared__ __align__(16) long long from_at[kAhead], to_at[kAhead];
    const bool codes = blockIdx.x & 1;   // of V
    const int kvh = blockIdx.x / 2, seq = blockIdx.y;
    c.pages = a.pages[blockIdx.z];
    const int n = min(a.counts[seq], a.max_count), first = a.first[seq];
    if (n <= 0 || first < 0) return;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int l = lane % T::kQuad, quad = lane / T::kQuad;
    const int32_t* kept = a.kept + (size_t)seq * a.kept_stride;
    const int32_t* table = a.page_table + (size_t)seq * a.pages_per_seq;
    const int P = 1 << c.page_shift, lead = first & 3;   // target positions of the first quad that stay
    const int turn = blockDim.x / kWave * kTokens;
    const int end = lead + n;

    auto part_of = [&](long long position) {
        const long long at = position >> c.page_shift;
        const int page = at < a.pages_per_seq ? table[at] : -1;
        if (page < 0 || page >= c.num_pages) return -1ll;
        return (long long)(kv4_head<HD>(c, page, kvh) - c.pages) << 8 | (position & (P - 1));
    };
    // a lane's bytes of a token in row o of its part: lane_at + (o >> lane_shift) *
    // lane_row, and for V 2 (o & 3) more
    const bool is_k = !codes && l < kKLanes, is_v = codes || (!is_k && l < kKLanes + kVParams);
    const bool k_codes = is_k && l < kCodeLanes;
    const int lane_shift = is_k ? 0 : 2, lane_and = is_k ? 0 : 3;
    const int lane_row = k_codes ? L::kCodes : is_k ? L::kParams : 8 * (codes ? kVCodes : kVParams);
    const int lane_at = k_codes  ? l % (HD / 32) * 16
                        : is_k   ? L::k_params(P)
                        : codes  ? L::v_codes(P) + 8 * l
                                 : L::v_params(P) + 8 * (l - kKLanes);
    auto place = [&](long long part) {
        const int o = (int)part & 255;
        return c.pages + (part >> 8) + (lane_at + (o >> lane_shift) * lane_row + 2 * (o & lane_and));
    };
    const int k_token = k_codes ? l / (HD / 32) : l - kCodeLanes;   // of the quad
    const bool wide = HD == 128 || k_codes;                          // 16 bytes of K, else 8
    const int my_quad = wave * kTokens + quad * 4;
    constexpr int kStride = 4 * (kWave / T::kQuad);   // of a step's tokens
    // without branches on what moves: the cache's first bytes are read in the place of none
    auto load = [&](int t, u32x4 (&v)[kSteps]) {
        const long long* at = from_at + t + my_quad;
        if (is_k) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const uint8_t* src = place(max(at[s * kStride + k_token], 0ll));
                if (wide) {
                    v[s] = *reinterpret_cast<const u32x4*>(src);
                } else {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(src);
                    v[s].x = w.x;
                    v[s].y = w.y;
                }
            }
        } else if (is_v) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v[s][k] = *reinterpret_cast<const uint16_t*>(place(max(at[s * kStride + k], 0ll)));
        }
    };
    auto store = [&](int t, const u32x4 (&v)[kSteps]) {
        const long long* at = to_at + t + my_quad;
        if (is_k) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const long long to = at[s * kStride + k_token];
                if (to < 0) continue;
                if (wide)
                    *reinterpret_cast<u32x4*>(place(to)) = v[s];
                else
                    *reinterpret_cast<u32x2*>(place(to)) = u32x2{v[s].x, v[s].y};
            }
        } else if (is_v) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                long long to[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) to[k] = at[s * kStride + k];
                if ((to[0] | to[1] | to[2] | to[3]) >= 0) {
                    *reinterpret_cast<u32x2*>(place(to[0])) = u32x2{v[s].x | v[s].y << 16, v[s].z | v[s].w << 16};
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (to[k] >= 0) *reinterpret_cast<uint16_t*>(place(to[k])) = (uint16_t)v[s][k];
                }
            }
        }
    };

    u32x4 v[kSteps], w[kSteps];
    for (int t0 = 0; t0 < end; t0 += kAhead) {   // (all bounds are the same for the workgroup's waves)
        const int some = min(kAhead, (end - t0 + turn - 1) / turn * turn);
        __syncthreads();
        for (int i = threadIdx.x; i < some; i += blockDim.x) {
            const int j = t0 + i - lead, source = j >= 0 && j < n ? kept[j] : -1;
            long long from = -1, to = -1;
            if (j >= 0 && source > j) {
                from = part_of((long long)first + source);
                to = part_of((long long)first + j);
            }
            from_at[i] = from;
            to_at[i] = from < 0 ? -1 : to;
        }
        __syncthreads();
        // two turns' tokens on their way while a third's are stored
        auto go = [&](int t, u32x4 (&x)[kSteps]) {
#pragma unroll
            for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(x[s]));   // in registers, not on the way,
            lds_only_barrier();                                              // before another wave may write there
            store(t, x);
            if (t + 2 * turn < some) load(t + 2 * turn, x);
        };
        load(0, v);
        if (turn < some) load(turn, w);
        for (int t = 0; t < some; t += 2 * turn) {
            go(t, v);
            if (t + turn < some) go(t + turn, w);
        }
    }
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

// Heads of a wave: as many of 8, 4 or 2 as leave four waves per SIMD, else one.
// 8192 tokens of 32/8 heads: 45.2 us with 16, 43.7 with 8, 48.4 with 4.
hipError_t launch_kv4_append(const Kv4View& c, const Kv4Append& a, hipStream_t s) {
    const long long groups = (a.tokens + 512 / c.head_dim - 1) / (512 / c.head_dim);
    auto waves = [&](int per) { return groups * ((a.heads + per - 1) / per + 2 * ((c.kv_heads + per - 1) / per)); };
    int per = 8;
    while (per > 1 && waves(per) < kEnoughWaves) per /= 2;
    const dim3 grid((unsigned)((waves(per) + kBlk / kWave - 1) / (kBlk / kWave)));
    if (c.head_dim == 128)
        launch_kernel(kv4_append_kernel<128>, grid, dim3(kBlk), 0, s, c, a, per);
    else
        launch_kernel(kv4_append_kernel<64>, grid, dim3(kBlk), 0, s, c, a, per);
    return hipGetLastError();
}

hipError_t launch_kv4_read(const Kv4View& c, const int32_t* slots, int count, uint16_t* k_out, uint16_t* v_out,
                           hipStream_t s) {
    const dim3 grid(blocks_for(count, c.head_dim, c.kv_heads));
    if (c.head_dim == 128)
        launch_kernel(kv4_read_kernel<128>, grid, dim3(kBlk), 0, s, c, slots, count, k_out, v_out);
    else
        launch_kernel(kv4_read_kernel<64>, grid, dim3(kBlk), 0, s, c, slots, count, k_out, v_out);
    return hipGetLastError();
}

hipError_t launch_kv4_keep(const Kv4View& c, const Kv4Keep& a, hipStream_t s) {
    const dim3 grid(2 * c.kv_heads, a.nseq, a.layers);
    const int tokens = c.head_dim == 128 ? KeepTurn<128>::kTokens : KeepTurn<64>::kTokens;
    const int waves = std::min<long long>(kKeepWaves, ((long long)a.max_count + 3 + tokens - 1) / tokens);
    if (c.head_dim == 128)
        launch_kernel(kv4_keep_kernel<128>, grid, dim3(waves * kWave), 0, s, c, a);
    else
        launch_kernel(kv4_keep_kernel<64>, grid, dim3(waves * kWave), 0, s, c, a);
    return hipGetLastError();
}

}  // namespace citlali::hip
