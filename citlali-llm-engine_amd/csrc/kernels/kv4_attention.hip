// kv4_attention.hip -- causal attention over the paged cache of 4-bit keys and
// values.
#include "kv4.hpp"

#include <math.h>

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

}  // namespace

size_t kv4_attention_workspace(int, int, int, int, int, int, int) { return 0; }

hipError_t launch_kv4_attention(const Kv4View& c, const Kv4Attention& a, hipStream_t s) {
    const dim3 grid(a.max_query, a.nseq, a.heads);
    const float scale = 1.f / sqrtf((float)c.head_dim);
    if (c.head_dim == 128)
        launch_kernel(kv4_attention_rows_kernel<128>, grid, dim3(kWave), 0, s, c, a, scale);
    else
        launch_kernel(kv4_attention_rows_kernel<64>, grid, dim3(kWave), 0, s, c, a, scale);
    return hipGetLastError();
}

}  // namespace citlali::hip
