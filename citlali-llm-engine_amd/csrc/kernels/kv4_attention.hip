// kv4_attention.hip -- causal attention over the paged cache of 4-bit keys and
// values.
#include "kv4.hpp"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace citlali::hip {
namespace {

// The queries of sequence `seq`: rows start .. start + n - 1 of q, the cached
// positions that exist, and how many of them query i sees (see()).
struct Kv4Seq {
    int start, n, context, cap;
    __device__ int see(int i) const { return min(context - n + i + 1, cap); }
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attention& a, int seq) {
    Kv4Seq s;
    int end;
    if (a.query_start != nullptr) {
        s.start = min(max(a.query_start[seq], 0), a.tokens);
        end = min(max(a.query_start[seq + 1], s.start), a.tokens);
    } else {
        s.start = seq;
        end = seq + 1;
    }
    s.n = end - s.start;
    s.context = a.context_lens[seq];
    s.cap = a.max_context;
    return s;
}

constexpr int kBlk = 256, kWaves = kBlk / kWave;
constexpr float kShift = 14.f;   // weights are kept times 2^14

// ---------------------------------------------------------------------------
// Few rows: one workgroup per (chunk of positions, kv head, sequence) serves
// every query of the sequence for every head of the kv head's group, at most
// 16 kCols rows (row r: query r / group, head r % group), so the cache is read
// once.  The four waves take tiles of 32 positions in turn; no LDS until they
// merge:
//  * S^T[position][row] = K Q^T by v_mfma_f32_16x16x32_f16, 16 positions at a
//    time: lane (col, grp) of the A operand holds position col's dims
//    grp * HD/4 .. + HD/4 - 1, one 16-byte (head_dim 64: 8-byte) load of codes
//    with one (d, m); Q, the B operand, is held in the same dim order.
//  * online softmax down each column (row of Q): a lane has 8 of a tile's 32
//    positions, the maximum takes two permlane swaps, the sum stays per lane
//    until the end.
//  * O^T[dim][row] += V^T P^T: the lanes' weights are the B operand as they
//    stand (k index = grp 4 + i of the first 16 positions, then of the second);
//    V lies in groups of four tokens, so lane (c, grp) loads the codes of its
//    four positions and HD / 16 dims together, each word two positions' dims,
//    and gets the A operand's pairs without a transposition.
// Bound by the cache's bytes: 5 KB a tile of head_dim 128 against about 300
// vector instructions, a good half of what a CU issues meanwhile at 6 TB/s.
// ---------------------------------------------------------------------------
template <int HD, int kCols>
__global__ __launch_bounds__(kBlk, kCols == 1 ? 4 : 2) void kv4_decode_kernel(Kv4View c, Kv4Attention a, int chunk, int n_splits,
                                                          float scale_log2) {
    using L = Kv4Layout<HD>;
    using Vec = std::conditional_t<HD == 128, u32x4, u32x2>;   // a lane's codes of 16 positions
    constexpr int kSteps = HD / 32, kDims = HD / 16;   // MFMA steps of a score; dims (and O tiles) of a V lane
    // the waves' merge, rows_most of each: [wave][row][HD + 4], sums behind HD
    extern __shared__ __align__(16) float lds[];
    const int rows_most = a.max_query * (a.heads / c.kv_heads);

    const int split = blockIdx.x, kvh = blockIdx.y, seq = blockIdx.z;
    const Kv4Seq s = kv4_seq(a, seq);
    const int asked = min(s.n, a.max_query);
    if (asked <= 0) return;
    const int group = a.heads / c.kv_heads, rows = asked * group;
    const int most = max(0, s.see(asked - 1));   // positions any row sees
    const int c0 = split * chunk, c1 = min(most, c0 + chunk);
    if (c0 >= most && split > 0) return;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int col = lane & 15, grp = lane >> 4;

    // page of 16 .. positions j of the chunk's pages: lane j (a chunk has at most 64)
    const int first_page = c0 >> c.page_shift;
    int my_page = -1;
    if (((first_page + lane) << c.page_shift) < c1) {
        my_page = a.page_table[(size_t)seq * a.pages_per_seq + first_page + lane];
        if (my_page >= c.num_pages) my_page = -1;
    }
    half8 q[kCols][kSteps];
    int see[kCols];
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
        const int r = col + 16 * n, i = r / group;
        const bool real = r < rows;
        see[n] = real ? s.see(i) : 0;
        const uint16_t* qr = a.q + (size_t)(s.start + (real ? i : 0)) * a.q_stride +
                             (size_t)(kvh * group + (real ? r - i * group : 0)) * HD + grp * (HD / 4);
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            u32x4 v = *reinterpret_cast<const u32x4*>(qr + 8 * t);
            if (!real) v = u32x4{0u, 0u, 0u, 0u};
            q[n][t] = __builtin_bit_cast(half8, v);
        }
    }
    const int least = s.see(0);   // positions every row sees

    const int P = 1 << c.page_shift;
    // The page of the 16 positions at p (-1: none).  Past the chunk it is the
    // chunk's first: every load is unconditional, so that the compiler's waits
    // count exactly, and in bounds.
    auto page_of = [&](int p) {
        const int page = __builtin_amdgcn_readlane(my_page, ((p < c1 ? p : c0) >> c.page_shift) - first_page);
        return p < c1 ? page : -1;
    };
    auto head_at = [&](int p) {
        const int page = __builtin_amdgcn_readlane(my_page, ((p < c1 ? p : c0) >> c.page_shift) - first_page);
        return kv4_head<HD>(c, max(page, 0), kvh);
    };
    Vec xk[2], xv[2];
    uint32_t xkp[2];
    u32x4 xvp[2];
    auto load_k = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint8_t* base = head_at(t + 16 * u);
            const int o = (t + 16 * u) & (P - 1) & ~15;
            xk[u] = *reinterpret_cast<const Vec*>(base + (o + col) * L::kCodes + grp * (HD / 8));
            xkp[u] = *reinterpret_cast<const uint32_t*>(base + L::k_params(P) + (o + col) * L::kParams +
                                                        (HD == 128 ? grp : grp >> 1) * 4);
        }
    };
    auto load_v = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint8_t* base = head_at(t + 16 * u);
            const int o = (t + 16 * u) & (P - 1) & ~15;
            xv[u] = *reinterpret_cast<const Vec*>(base + L::v_codes(P) + ((o >> 2) + grp) * (4 * L::kCodes) +
                                                  col * (HD / 8));
            xvp[u] = *reinterpret_cast<const u32x4*>(base + L::v_params(P) + ((o >> 2) + grp) * (4 * L::kParams) +
                                                     col / (512 / HD) * 16);
        }
    };

    f32x4 o[kCols][kDims];
    float m_run[kCols], l_run[kCols];
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
        m_run[n] = -INFINITY;
        l_run[n] = 0.f;
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    load_k(c0 + 32 * wave);
    load_v(c0 + 32 * wave);
    __builtin_amdgcn_sched_barrier(0);
    for (int t = c0 + 32 * wave; t < c1; t += 32 * kWaves) {
        const int there = (page_of(t) >= 0) | (page_of(t + 16) >= 0) << 1;
        const bool whole = there == 3 && t + 32 <= least;
        f32x4 sc[kCols][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int n = 0; n < kCols; ++n) sc[n][u] = f32x4{0.f, 0.f, 0.f, 0.f};
            const f16x2 dm = as_h2(xkp[u]);
            const f16x2 d{dm.x, dm.x}, m{dm.y, dm.y};
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                f16x2 e[4];
                kv4_pairs(xk[u][st], d, m, e);
                const half8 k = __builtin_bit_cast(half8, e);
#pragma unroll
                for (int n = 0; n < kCols; ++n)
                    sc[n][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[n][st], sc[n][u], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(t + 32 * kWaves);   // in flight through the softmax and V
        __builtin_amdgcn_sched_barrier(0);
        half8 pw[kCols];
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
            if (!whole) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool seen = ((there >> u) & 1) && t + 16 * u + 4 * grp + i < min(see[n], c1);
                        sc[n][u][i] = seen ? sc[n][u][i] : -INFINITY;
                    }
            }
            float mt = fmaxf(fmaxf(fmaxf(sc[n][0][0], sc[n][0][1]), fmaxf(sc[n][0][2], sc[n][0][3])),
                             fmaxf(fmaxf(sc[n][1][0], sc[n][1][1]), fmaxf(sc[n][1][2], sc[n][1][3])));
            mt = max32(max16(mt)) * scale_log2;
            if (__builtin_amdgcn_ballot_w64(mt > m_run[n]) != 0) {
                const float m_new = fmaxf(m_run[n], mt);
                const float f = m_run[n] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[n] - m_new);
                m_run[n] = m_new;
                l_run[n] *= f;
#pragma unroll
                for (int d = 0; d < kDims; ++d) o[n][d] *= f;
            }
            const float off = kShift - (m_run[n] == -INFINITY ? 0.f : m_run[n]);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(sc[n][u][i], scale_log2, off));
                    l_run[n] += w;
                    pw[n][4 * u + i] = (_Float16)w;
                }
        }
        if (!whole) {   // positions no row may use: their V counts as 0, whatever it holds
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int left = (there >> u) & 1 ? c1 - (t + 16 * u + 4 * grp) : 0;   // of this lane's four
                const uint32_t lo = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
                const uint32_t hi = left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
                xvp[u] &= u32x4{lo, hi, lo, hi};
            }
        }
#pragma unroll
        for (int h = 0; h < kDims / 4; ++h) {
            f16x2 e[4][4];   // [token pair][dim]
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int y = 0; y < 2; ++y)
                    kv4_pairs(xv[u][2 * h + y], as_h2(xvp[u][y]), as_h2(xvp[u][2 + y]), e[2 * u + y]);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const f16x2 w[4] = {e[0][d], e[1][d], e[2][d], e[3][d]};
                const half8 v = __builtin_bit_cast(half8, w);
#pragma unroll
                for (int n = 0; n < kCols; ++n)
                    o[n][4 * h + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pw[n], o[n][4 * h + d], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v(t + 32 * kWaves);
        __builtin_amdgcn_sched_barrier(0);
    }

    // merge the waves
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
        l_run[n] = sum32(sum16(l_run[n]));
        const int r = col + 16 * n;
        if (r >= rows) continue;
        float* to = lds + (wave * rows_most + r) * (HD + 4);
        if (grp == 0) {
            to[HD] = m_run[n];
            to[HD + 1] = l_run[n];
        }
        // lane (col, grp) has dims kDims (4 grp + i) + d of its column
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < kDims; d += 4)
                *reinterpret_cast<f32x4*>(to + kDims * (4 * grp + i) + d) =
                    f32x4{o[n][d][i], o[n][d + 1][i], o[n][d + 2][i], o[n][d + 3][i]};
    }
    __syncthreads();
    const bool alone = most <= chunk;
    for (int idx = threadIdx.x; idx < rows * (HD / 4); idx += kBlk) {
        const int r = idx / (HD / 4), d = idx % (HD / 4) * 4, i = r / group;
        const float* from = lds + r * (HD + 4);
        const int step = rows_most * (HD + 4);
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, from[w * step + HD]);
        float l = 0.f;
        f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float m = from[w * step + HD];
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
            l += from[w * step + HD + 1] * f;
            acc += *reinterpret_cast<const f32x4*>(from + w * step + d) * f;
        }
        const size_t head = (size_t)kvh * group + (r - i * group);
        if (alone) {
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
            u32x2 w;
            w.x = f2h_rne(acc.x * inv) | ((uint32_t)f2h_rne(acc.y * inv) << 16);
            w.y = f2h_rne(acc.z * inv) | ((uint32_t)f2h_rne(acc.w * inv) << 16);
            *reinterpret_cast<u32x2*>(a.out + (size_t)(s.start + i) * a.out_stride + head * HD + d) = w;
        } else {
            const size_t at = ((size_t)(s.start + i) * a.heads + head) * n_splits + split;
            *reinterpret_cast<f32x4*>(a.workspace + at * HD + d) = acc;
            if (d == 0) {
                float* ml = a.workspace + (size_t)a.tokens * a.heads * n_splits * HD + 2 * at;
                ml[0] = M;
                ml[1] = l;
            }
        }
    }
}

// Log-sum-exp merge of the chunks of one (query, head) by one wave, HD / 64
// dims a lane.
template <int HD>
__global__ __launch_bounds__(kBlk) void kv4_merge_kernel(Kv4Attention a, int chunk, int n_splits) {
    constexpr int kPer = HD / kWave;
    const int seq = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    const Kv4Seq s = kv4_seq(a, seq);
    const int asked = min(s.n, a.max_query);
    const int unit = blockIdx.x * kWaves + threadIdx.x / kWave;
    const int i = unit / a.heads, head = unit - i * a.heads;
    if (i >= asked) return;
    const int most = s.see(asked - 1);
    if (most <= chunk) return;   // written by the chunk itself
    const int n = (most + chunk - 1) / chunk;
    const size_t at = ((size_t)(s.start + i) * a.heads + head) * n_splits;
    const float* part = a.workspace + at * HD + lane * kPer;
    const f32x2* ml = reinterpret_cast<const f32x2*>(a.workspace + (size_t)a.tokens * a.heads * n_splits * HD) + at;
    float M = -INFINITY;
    for (int j = lane; j < n; j += kWave) M = fmaxf(M, ml[j].x);
    M = wave_max(M);
    float l = 0.f, acc[kPer] = {};
    for (int j0 = 0; j0 < n; j0 += kWave) {
        float f = 0.f;
        if (j0 + lane < n) {
            const f32x2 v = ml[j0 + lane];
            f = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - M);
            l += v.y * f;
        }
        const int here = min(kWave, n - j0);
        for (int j = 0; j < here; ++j) {
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), j));
#pragma unroll
            for (int e = 0; e < kPer; ++e) acc[e] = fmaf(part[(size_t)(j0 + j) * HD + e], w, acc[e]);
        }
    }
    l = wave_sum(l);
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    uint16_t* out = a.out + (size_t)(s.start + i) * a.out_stride + (size_t)head * HD + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) out[e] = f2h_rne(acc[e] * inv);
}

// One wave per (query, sequence, head): lane = position for the scores, lane =
// dims for the values.
template <int HD>
__global__ __launch_bounds__(kWave) void kv4_attention_rows_kernel(Kv4View c, Kv4Attention a, float scale) {
    using L = Kv4Layout<HD>;
    const int i = blockIdx.x, seq = blockIdx.y, head = blockIdx.z, lane = threadIdx.x;
    const Kv4Seq s = kv4_seq(a, seq);
    if (i >= s.n) return;
    const int see = s.see(i), kvh = head / (a.heads / c.kv_heads), P = 1 << c.page_shift;
    __shared__ float qs[HD], ps[kWave];
    __shared__ const uint8_t* bases[kWave];
    for (int d = lane; d < HD; d += kWave)
        qs[d] = h2f(a.q[(size_t)(s.start + i) * a.q_stride + (size_t)head * HD + d]) * scale;
    __syncthreads();
    float m_run = -INFINITY, l_run = 0.f, acc[HD / kWave] = {};
    for (int p0 = 0; p0 < see; p0 += kWave) {
        const int p = p0 + lane, o = p & (P - 1);
        int page = -1;
        if (p < see) page = a.page_table[(size_t)seq * a.pages_per_seq + (p >> c.page_shift)];
        if (page >= c.num_pages) page = -1;
        float x = -INFINITY;
        const uint8_t* base = page >= 0 ? kv4_head<HD>(c, page, kvh) : nullptr;
        if (page >= 0) {
            x = 0.f;
            for (int w8 = 0; w8 < HD / 8; ++w8) {
                const f16x2 dm =
                    as_h2(*reinterpret_cast<const uint32_t*>(base + L::k_params(P) + o * L::kParams + w8 / 4 * 4));
                f16x2 v[4];
                kv4_pairs(*reinterpret_cast<const uint32_t*>(base + o * L::kCodes + 4 * w8), f16x2{dm.x, dm.x},
                          f16x2{dm.y, dm.y}, v);
                for (int e = 0; e < 4; ++e)
                    x += (float)v[e].x * qs[8 * w8 + 2 * e] + (float)v[e].y * qs[8 * w8 + 2 * e + 1];
            }
        }
        const float m = fmaxf(m_run, wave_max(x));
        const float w = m == -INFINITY ? 0.f : expf(x - m), f = m == -INFINITY ? 1.f : expf(m_run - m);
        l_run = l_run * f + wave_sum(w);
        m_run = m;
        ps[lane] = w;
        bases[lane] = base;
        __syncthreads();
        for (int e = 0; e < HD / kWave; ++e) {
            const int d = lane + e * kWave;
            acc[e] *= f;
            for (int j = 0; j < kWave; ++j) {
                const uint8_t* b = bases[j];
                if (b == nullptr) continue;
                const int oj = (p0 + j) & (P - 1);
                const uint32_t word =
                    reinterpret_cast<const uint16_t*>(b + L::v_codes(P))[((oj >> 2) * (HD / 4) + d / 4) * 4 + (oj & 3)];
                const _Float16* vp = reinterpret_cast<const _Float16*>(b + L::v_params(P)) +
                                     ((oj >> 2) * (HD / kKv4Group) + d / kKv4Group) * 8 + (oj & 3);
                const _Float16 v = __builtin_fmaf16((_Float16)(float)((word >> (4 * (d & 3))) & 15u), vp[0], vp[4]);
                acc[e] += ps[j] * (float)v;
            }
        }
        __syncthreads();
    }
    for (int e = 0; e < HD / kWave; ++e)
        a.out[(size_t)(s.start + i) * a.out_stride + (size_t)head * HD + lane + e * kWave] =
            f2h_rne(l_run > 0.f ? acc[e] / l_run : 0.f);
}


// Positions a workgroup takes: whole turns of its four waves, few enough for a
// lane per page, and about eight workgroups per CU where the bound allows.
constexpr int kChunkStep = 32 * kWaves, kChunkMost = 1024, kTargetBlocks = 2048;
struct Kv4Plan {
    bool few;   // the few-row kernel, else one wave per row
    int cols, chunk, n_splits;
};
Kv4Plan kv4_plan(int max_context, int max_query, int nseq, int heads, int kv_heads) {
    Kv4Plan p{};
    const long long rows = (long long)max_query * (heads / kv_heads);
    p.few = rows <= 32;
    p.cols = rows <= 16 ? 1 : 2;
    const long long want = ((long long)max_context * nseq * kv_heads + kTargetBlocks - 1) / kTargetBlocks;
    p.chunk = (int)std::min<long long>(kChunkMost, std::max<long long>(1, (want + kChunkStep - 1) / kChunkStep) * kChunkStep);
    p.n_splits = (max_context + p.chunk - 1) / p.chunk;
    return p;
}

}  // namespace

size_t kv4_attention_workspace(int max_context, int max_query, int nseq, int tokens, int heads, int kv_heads,
                               int head_dim) {
    const Kv4Plan p = kv4_plan(max_context, max_query, nseq, heads, kv_heads);
    if (!p.few || p.n_splits == 1) return 0;
    return (size_t)tokens * heads * p.n_splits * (head_dim + 2) * sizeof(float);
}

namespace {
template <int HD>
hipError_t launch_for(const Kv4View& c, const Kv4Attention& a, hipStream_t s) {
    const Kv4Plan p = kv4_plan(a.max_context, a.max_query, a.nseq, a.heads, c.kv_heads);
    const float scale = 1.f / sqrtf((float)HD);
    if (!p.few) {
        launch_kernel(kv4_attention_rows_kernel<HD>, dim3(a.max_query, a.nseq, a.heads), dim3(kWave), 0, s, c, a, scale);
        return hipGetLastError();
    }
    const float scale_log2 = scale * 1.44269504088896340736f;
    const dim3 grid(p.n_splits, c.kv_heads, a.nseq);
    const size_t lds = (size_t)kWaves * a.max_query * (a.heads / c.kv_heads) * (HD + 4) * sizeof(float);
    if (p.cols == 1) {
        launch_kernel_in_call(p.n_splits == 1, kv4_decode_kernel<HD, 1>, grid, dim3(kBlk), lds, s, c, a, p.chunk,
                              p.n_splits, scale_log2);
    } else {
        const hipError_t e = allow_lds<kv4_decode_kernel<HD, 2>>((int)lds);
        if (e != hipSuccess) return e;
        launch_kernel_in_call(p.n_splits == 1, kv4_decode_kernel<HD, 2>, grid, dim3(kBlk), lds, s, c, a, p.chunk,
                              p.n_splits, scale_log2);
    }
    if (p.n_splits > 1)
        launch_kernel(kv4_merge_kernel<HD>, dim3((a.max_query * a.heads + kWaves - 1) / kWaves, a.nseq), dim3(kBlk), 0,
                      s, a, p.chunk, p.n_splits);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_kv4_attention(const Kv4View& c, const Kv4Attention& a, hipStream_t s) {
    return c.head_dim == 128 ? launch_for<128>(c, a, s) : launch_for<64>(c, a, s);
}

}  // namespace citlali::hip
