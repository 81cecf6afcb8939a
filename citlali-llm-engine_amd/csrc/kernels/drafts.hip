// drafts.hip -- trees of drafted tokens: which rows see which, and from the
// model's logits the path that stays and the token after it.
#include "device_common.hpp"
#include "launch.hpp"

#include <limits.h>
#include <math.h>

#include <algorithm>

namespace citlali::hip {
namespace {

// ---------------------------------------------------------------------------
// Masks and positions.  One workgroup per sequence, a thread per row, by
// doubling: after step t a row's mask holds itself and the 2^t - 1 rows above it,
// and `above` is the row 2^t up.
// ---------------------------------------------------------------------------
constexpr int kNone = -1, kBad = -2;   // nothing above in the tree; a parent that is not an earlier row

__global__ __launch_bounds__(kMaxTree) void draft_tree_kernel(DraftTree a, int words) {
    __shared__ uint64_t mask[kMaxTree / 64][kMaxTree];
    __shared__ int above[kMaxTree];
    const int seq = blockIdx.x, i = threadIdx.x;
    const DraftRows rows = draft_rows(a.query_start, seq, a.tokens, a.max_query);
    const bool real = i < rows.n;
    int up = real ? a.parents[rows.start + i] : kNone;
    const int context = a.context_lens[seq];
    if (up < kNone || up >= i) up = real ? kBad : kNone;
    above[i] = up;
    for (int w = 0; w < words; ++w) mask[w][i] = i / 64 == w ? 1ull << (i % 64) : 0ull;
    __syncthreads();
    for (int reach = 1; reach < rows.n; reach *= 2) {
        uint64_t more[kMaxTree / 64];
        int next = up;
        if (up >= 0) {
            for (int w = 0; w < kMaxTree / 64; ++w) more[w] = w < words ? mask[w][up] : 0ull;
            next = above[up];
        }
        __syncthreads();
        if (up >= 0) {
            for (int w = 0; w < kMaxTree / 64; ++w)
                if (w < words) mask[w][i] |= more[w];
            above[i] = up = next;
        }
        __syncthreads();
    }
    if (!real) return;
    int depth = 0;
    for (int w = 0; w < words; ++w) {
        const uint64_t m = up == kBad ? 0ull : mask[w][i];
        depth += __popcll(m);
        a.masks[(size_t)(rows.start + i) * words + w] = m;
    }
    if (a.positions) a.positions[rows.start + i] = up == kBad ? -1 : max(context, 0) - rows.total + depth - 1;
}

// ---------------------------------------------------------------------------
// Verification.  p = softmax(x / T) of a row; everything that decides is in 64
// bits: a token drawn by the first running sum above u times the total is
// misplaced where the sums are off by more than u's distance to the next border,
// of which a row has as many as tokens (151936 of them at an error of 2^-26, what
// 32 bits give: 1 draw in 200).
// ---------------------------------------------------------------------------
constexpr int kBlk = 256, kWaves = kBlk / kWave;
constexpr int kPer = 32, kSeg = kPer * kWave;   // logits of a lane, and of a wave: a segment

// 2^z, z <= 0 (0 from -1100 on).  2^f = 1 + f g(f), g by Chebyshev's interpolant of
// degree 8 on [-1/2, 1/2]: 2^0 is 1, the rest off by 3.7e-14 at most.
__device__ __forceinline__ double exp2_64(double z) {
    z = fmax(z, -1100.);
    const double k = rint(z), f = z - k;
    double r = 1.0203121063391729e-07;
    r = fma(r, f, 1.3255224878668817e-06);
    r = fma(r, f, 1.525268684626772e-05);
    r = fma(r, f, 0.00015403455852453838);
    r = fma(r, f, 0.0013333558179043112);
    r = fma(r, f, 0.009618129159402558);
    r = fma(r, f, 0.055504108664760424);
    r = fma(r, f, 0.2402265069581299);
    r = fma(r, f, 0.6931471805599453);
    r = fma(r, f, 1.);
    return ldexp(r, (int)k);
}
// Weight of a logit x against one of m >= x; c = log2(e) / T.
__device__ __forceinline__ double weight(float x, float m, double c) {
    return x == -INFINITY ? 0. : exp2_64(((double)x - (double)m) * c);
}

template <typename T, typename F>
__device__ __forceinline__ T wave_fold(T v, F f) {
    for (int o = 1; o < kWave; o <<= 1) v = f(v, __shfl_xor(v, o, kWave));
    return v;
}
__device__ __forceinline__ double wave_sum64(double v) {
    return wave_fold(v, [](double a, double b) { return a + b; });
}

template <bool kHalf>
__device__ __forceinline__ float logit(const void* row, int i) {
    if constexpr (kHalf)
        return h2f(static_cast<const uint16_t*>(row)[i]);
    else
        return static_cast<const float*>(row)[i];
}
template <bool kHalf>
__device__ __forceinline__ const void* logit_row(const void* logits, long long stride, int r) {
    return static_cast<const char*>(logits) + (size_t)r * stride * (kHalf ? 2 : 4);
}

// What a segment of a row comes to: its largest logit (NaN where the row has no
// distribution), the sum of the weights against it, and the first id that has it
// (greedy rows only).
struct alignas(16) Segment {
    double sum;
    float top;
    int first;
};
// Where a sequence's path ended.
struct alignas(16) PathEnd {
    double s, s_draft;
    float m, m_draft;
    int row;     // of the logits
    int rest;    // 1: the token comes from max(p - q, 0)
    double c;
};
struct Work {
    Segment* segments;   // [rows (, then drafts')][segs]
    PathEnd* ends;       // [nseq]
    double* rest;        // [nseq][segs]
};
__host__ __device__ inline Work work_of(const VerifyDrafts& a, int segs) {
    Work w;
    w.segments = static_cast<Segment*>(a.workspace);
    w.ends = reinterpret_cast<PathEnd*>(w.segments + (size_t)a.rows * (a.draft ? 2 : 1) * segs);
    w.rest = reinterpret_cast<double*>(w.ends + (a.draft ? a.nseq : 0));
    return w;
}

__device__ __forceinline__ float temperature(const VerifyDrafts& a, int seq) {
    return a.temperatures ? a.temperatures[seq] : 1.f;
}
constexpr double kLog2e = 1.4426950408889634074;

// Workgroup (4 segments, row, sequence), a segment a wave.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void verify_sums_kernel(VerifyDrafts a, int segs) {
    constexpr int kVec = kHalf ? 8 : 4, kLoads = kPer / kVec;
    const int seq = blockIdx.z;
    const bool draft = (int)blockIdx.y >= a.max_query;
    const int i = blockIdx.y - (draft ? a.max_query : 0);
    const DraftRows rows = draft_rows(a.query_start, seq, a.rows, a.max_query);
    if (i >= rows.n || (draft && i + 1 >= rows.n)) return;   // the last row's draft has no child
    const int lane = threadIdx.x & (kWave - 1);
    const int seg = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (seg >= segs) return;
    const float t = temperature(a, seq);
    const int r = rows.start + i;
    const void* row = draft ? logit_row<kHalf>(a.draft, a.draft_stride, r) : logit_row<kHalf>(a.logits, a.stride, r);
    const int id0 = seg * kSeg;
    float x[kPer];
    if (id0 + kSeg <= a.vocab) {
        const char* at = static_cast<const char*>(row) + (size_t)id0 * (kHalf ? 2 : 4) + lane * 16;
#pragma unroll
        for (int l = 0; l < kLoads; ++l) {
            u32x4 v = *reinterpret_cast<const u32x4_a2*>(at + l * kWave * 16);
#pragma unroll
            for (int e = 0; e < kVec; ++e)
                x[l * kVec + e] = kHalf ? h2f((uint16_t)(v[e / 2] >> (e % 2 * 16))) : __uint_as_float(v[e]);
        }
    } else {
#pragma unroll
        for (int l = 0; l < kPer; ++l) {
            const int id = id0 + (l / kVec * kWave + lane) * kVec + l % kVec;
            x[l] = id < a.vocab ? logit<kHalf>(row, id) : -INFINITY;
        }
    }
    float top = x[0];
#pragma unroll
    for (int l = 1; l < kPer; ++l) top = __builtin_elementwise_maximum(top, x[l]);   // a NaN stays
    const bool bad = __builtin_amdgcn_ballot_w64(!(top < INFINITY)) != 0;
    top = wave_max(top);
    Segment out{0., bad ? NAN : top, 0};
    if (!bad && top > -INFINITY) {
        if (t > 0.f) {
            const double c = kLog2e / (double)t, m = top;
            double s[2] = {0., 0.};
#pragma unroll
            for (int l = 0; l < kPer; ++l) s[l % 2] += exp2_64(((double)x[l] - m) * c);
            out.sum = wave_sum64(s[0] + s[1]);
        } else {
            int first = INT_MAX;
#pragma unroll
            for (int l = kPer - 1; l >= 0; --l)
                if (x[l] == top) first = id0 + (l / kVec * kWave + lane) * kVec + l % kVec;
            out.first = wave_fold(first, [](int p, int q) { return min(p, q); });
            out.sum = 1.;
        }
    }
    if (lane == 0) work_of(a, segs).segments[((size_t)(draft ? a.rows : 0) + r) * segs + seg] = out;
}

// Largest logit, sum and first id of a row from its segments, by one wave.
struct RowSum {
    double s;
    float m;   // NaN: no distribution
    int first;
};
__device__ RowSum join_segments(const Segment* at, int segs, bool greedy, double c, int lane) {
    float m = -INFINITY;
    double s = 0.;
    int first = INT_MAX;
    bool bad = false;
    for (int j = lane; j < segs; j += kWave) {
        const Segment g = at[j];
        bad |= g.top != g.top;
        if (!(g.top > -INFINITY)) continue;
        if (greedy) {
            if (g.top > m) {
                m = g.top;
                first = g.first;
            }
        } else if (g.top > m) {
            s = fma(s, m == -INFINITY ? 0. : weight(m, g.top, c), g.sum);
            m = g.top;
        } else {
            s = fma(g.sum, weight(g.top, m, c), s);
        }
    }
    RowSum r;
    r.m = wave_max(m);
    bad = __builtin_amdgcn_ballot_w64(bad) != 0 || r.m == -INFINITY;
    if (greedy) {
        r.first = wave_fold(m == r.m ? first : INT_MAX, [](int p, int q) { return min(p, q); });
        r.s = 1.;
    } else {
        r.first = 0;
        r.s = wave_sum64(m == -INFINITY ? 0. : s * weight(m, r.m, c));
    }
    if (bad) r.m = NAN;
    return r;
}

// Running sum over the threads, and the workgroup's total.
struct Scan {
    double before, total;
};
__device__ Scan block_scan(double v, double* room) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    double run = v;
    for (int o = 1; o < kWave; o <<= 1) {
        const double w = __shfl_up(run, o, kWave);
        if (lane >= o) run += w;
    }
    __syncthreads();
    if (lane == kWave - 1) room[wave] = run;
    __syncthreads();
    Scan s{run - v, 0.};
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) s.before += room[w];
        s.total += room[w];
    }
    return s;
}

// The first id whose running sum of weights exceeds u times their total; -1 where
// the total is 0.  value(j): sum of segment j's weights; weight_of(id).
template <typename V, typename W>
__device__ int pick(int vocab, int segs, float u, V value, W weight_of) {
    __shared__ double room[kWaves];
    __shared__ int found, last;
    __shared__ double found_before;
    u = u >= 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
    double total = 0.;
    for (int j0 = 0; j0 < segs; j0 += kBlk) {
        const int j = j0 + threadIdx.x;
        total += block_scan(j < segs ? value(j) : 0., room).total;
    }
    if (!(total > 0.)) return -1;
    const double t = (double)u * total;
    if (threadIdx.x == 0) {
        found = INT_MAX;
        last = -1;
    }
    double base = 0.;
    for (int j0 = 0; j0 < segs; j0 += kBlk) {
        const int j = j0 + threadIdx.x;
        const double v = j < segs ? value(j) : 0.;
        const Scan s = block_scan(v, room);
        if (v > 0.) {
            if (base + s.before + v > t) atomicMin(&found, j);
            atomicMax(&last, j);
        }
        __syncthreads();
        const bool here = found == j;
        if (here) found_before = base + s.before;
        base += s.total;
        if (found < INT_MAX) break;   // uniform
    }
    __syncthreads();
    // (where rounding leaves no segment, the last one that has any)
    const int seg = found < INT_MAX ? found : last;
    const double before = found < INT_MAX ? found_before : 0., bar = found < INT_MAX ? t : INFINITY;
    __syncthreads();
    if (threadIdx.x == 0) {
        found = INT_MAX;
        last = -1;
    }
    constexpr int kRun = kSeg / kBlk;
    const int id0 = seg * kSeg + (int)threadIdx.x * kRun;
    double w[kRun], sum = 0.;
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
        w[e] = id0 + e < vocab ? weight_of(id0 + e) : 0.;
        sum += w[e];
    }
    double run = before + block_scan(sum, room).before;
    int mine = INT_MAX;
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
        run += w[e];
        if (w[e] > 0.) {
            if (run > bar && mine == INT_MAX) mine = id0 + e;
            atomicMax(&last, id0 + e);
        }
    }
    if (mine < INT_MAX) atomicMin(&found, mine);
    __syncthreads();
    return found < INT_MAX ? found : last;
}

// One workgroup per sequence: the rows' sums, the drafted tokens' probabilities,
// the path, and the next token but where it comes from what q leaves of p.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void verify_walk_kernel(VerifyDrafts a, int segs) {
    __shared__ RowSum target[kMaxTree], drafted[kMaxTree];
    __shared__ int parent[kMaxTree], token[kMaxTree], gone[kMaxTree];
    __shared__ double p[kMaxTree], bar[kMaxTree];
    __shared__ int end_row, end_gone;
    const int seq = blockIdx.x, lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const DraftRows rows = draft_rows(a.query_start, seq, a.rows, a.max_query);
    const Work work = work_of(a, segs);
    if (rows.n <= 0) {
        if (a.paths)
            for (int i = threadIdx.x; i < a.max_query; i += kBlk) a.paths[(size_t)seq * a.max_query + i] = -1;
        if (threadIdx.x == 0) {
            if (a.counts) a.counts[seq] = 0;
            a.next_tokens[seq] = -1;
            if (a.draft) work.ends[seq].rest = 0;
        }
        return;
    }
    const float t = temperature(a, seq);
    const bool greedy = !(t > 0.f);
    const double c = greedy ? 0. : kLog2e / (double)t;
    const Segment* segments = work.segments + (size_t)rows.start * segs;
    const Segment* draft_segments = segments + (size_t)a.rows * segs;
    for (int i = wave; i < rows.n; i += kWaves) {
        const RowSum r = join_segments(segments + (size_t)i * segs, segs, greedy, c, lane);
        if (lane == 0) target[i] = r;
        if (a.draft && i + 1 < rows.n) {
            const RowSum d = join_segments(draft_segments + (size_t)i * segs, segs, greedy, c, lane);
            if (lane == 0) drafted[i] = d;
        }
    }
    __syncthreads();
    const int i = threadIdx.x;
    float u = 0.f;
    if (i < rows.n) {
        const int r = rows.start + i;
        int up = a.parents ? a.parents[r] : i - 1;
        if (up < 0 || up >= i) up = -1;
        const int x = up >= 0 ? a.tokens[r] : -1;
        u = a.uniforms[r];
        u = u >= 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f;
        double mine = 0., against = 1.;
        if (up >= 0 && x >= 0 && x < a.vocab) {
            const RowSum s = target[up];
            if (s.m == s.m) {
                if (greedy)
                    mine = x == s.first;
                else
                    mine = weight(logit<kHalf>(logit_row<kHalf>(a.logits, a.stride, rows.start + up), x), s.m, c) / s.s;
            }
            if (a.draft) {
                const RowSum d = drafted[up];
                if (d.m != d.m)
                    against = INFINITY;   // no distribution: rejected
                else if (greedy)
                    against = x == d.first;
                else
                    against =
                        weight(logit<kHalf>(logit_row<kHalf>(a.draft, a.draft_stride, rows.start + up), x), d.m, c) / d.s;
            }
        }
        parent[i] = up;
        token[i] = x;
        p[i] = mine;
        bar[i] = a.draft ? (u == 0.f && against == INFINITY ? INFINITY : (double)u * against) : (double)u;
        if (a.token_probs) a.token_probs[r] = (float)mine;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int current = 0, count = 1, lost = 0;
        double left = 1.;
        if (a.paths) a.paths[(size_t)seq * a.max_query] = 0;
        for (int k = 1; k < rows.n; ++k) {
            if (parent[k] != current) continue;
            double mine = p[k];
            for (int g = 0; g < lost; ++g)
                if (gone[g] == token[k]) mine = 0.;
            if (bar[k] * (a.draft ? 1. : left) < mine) {
                current = k;
                if (a.paths) a.paths[(size_t)seq * a.max_query + count] = k;
                ++count;
                lost = 0;
                left = 1.;
            } else {
                left -= mine;
                gone[lost++] = token[k];
            }
        }
        if (a.counts) a.counts[seq] = count;
        if (a.paths)
            for (int k = count; k < a.max_query; ++k) a.paths[(size_t)seq * a.max_query + k] = -1;
        end_row = current;
        end_gone = lost;
    }
    __syncthreads();
    const int f = end_row, lost = end_gone;
    const RowSum s = target[f];
    const bool rest = a.draft && lost > 0 && s.m == s.m && !greedy && drafted[f].m == drafted[f].m;
    if (a.draft && threadIdx.x == 0) {
        PathEnd e{};
        e.rest = rest;
        if (rest) {
            e.s = s.s;
            e.m = s.m;
            e.s_draft = drafted[f].s;
            e.m_draft = drafted[f].m;
            e.row = rows.start + f;
            e.c = c;
        }
        work.ends[seq] = e;
    }
    if (rest) return;
    int next = -1;
    if (s.m != s.m) {
        // no distribution
    } else if (greedy) {
        next = s.first;
    } else {
        const void* row = logit_row<kHalf>(a.logits, a.stride, rows.start + f);
        Segment* mine = work.segments + ((size_t)rows.start + f) * segs;
        auto of = [&](int id) { return weight(logit<kHalf>(row, id), s.m, c); };
        auto value = [&](int j) {
            const Segment g = mine[j];
            return g.top > -INFINITY ? g.sum * weight(g.top, s.m, c) : 0.;
        };
        const int out = a.draft ? 0 : lost;   // rejected tokens to leave out
        auto left_of = [&](int id) {
            for (int g = 0; g < out; ++g)
                if (gone[g] == id) return 0.;
            return of(id);
        };
        // their segments anew, without them, by a wave each
        auto resum = [&](bool all) {
            for (int g = wave; g < out; g += kWaves) {
                if (gone[g] < 0 || gone[g] >= a.vocab) continue;
                const int seg = gone[g] / kSeg, id1 = min(a.vocab, (seg + 1) * kSeg);
                double sum = 0.;
                for (int id = seg * kSeg + lane; id < id1; id += kWave) sum += all ? of(id) : left_of(id);
                sum = wave_sum64(sum);
                if (lane == 0) mine[seg] = Segment{sum, s.m, 0};
            }
            __syncthreads();
        };
        if (out > 0) resum(false);
        next = pick(a.vocab, segs, a.uniforms[rows.start], value, left_of);
        if (next < 0) {   // nothing is left
            __syncthreads();
            resum(true);
            next = pick(a.vocab, segs, a.uniforms[rows.start], value, of);
        }
    }
    if (threadIdx.x == 0) a.next_tokens[seq] = next;
}

template <bool kHalf>
struct Rest {   // max(p - q, 0)
    const void *row, *draft_row;
    PathEnd e;
    double inv, inv_draft;
    __device__ Rest(const VerifyDrafts& a, const PathEnd& end)
        : row(logit_row<kHalf>(a.logits, a.stride, end.row)),
          draft_row(logit_row<kHalf>(a.draft, a.draft_stride, end.row)), e(end), inv(1. / end.s),
          inv_draft(1. / end.s_draft) {}
    __device__ double operator()(int id) const {
#pragma clang fp contract(off)   // equal p and q leave nothing
        return fmax(weight(logit<kHalf>(row, id), e.m, e.c) * inv -
                        weight(logit<kHalf>(draft_row, id), e.m_draft, e.c) * inv_draft,
                    0.);
    }
};

// Workgroup (4 segments, sequence): what q leaves of p where a draft was rejected.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void verify_rest_kernel(VerifyDrafts a, int segs) {
    const int seq = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    const int seg = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const Work work = work_of(a, segs);
    const PathEnd e = work.ends[seq];
    if (!e.rest || seg >= segs) return;
    const Rest<kHalf> rest(a, e);
    const int id1 = min(a.vocab, (seg + 1) * kSeg);
    double sum = 0.;
#pragma unroll 4
    for (int id = seg * kSeg + lane; id < id1; id += kWave) sum += rest(id);
    sum = wave_sum64(sum);
    if (lane == 0) work.rest[(size_t)seq * segs + seg] = sum;
}

template <bool kHalf>
__global__ __launch_bounds__(kBlk) void verify_pick_kernel(VerifyDrafts a, int segs) {
    const int seq = blockIdx.x;
    const Work work = work_of(a, segs);
    const PathEnd e = work.ends[seq];
    if (!e.rest) return;
    const DraftRows rows = draft_rows(a.query_start, seq, a.rows, a.max_query);
    const Rest<kHalf> rest(a, e);
    const float u = a.uniforms[rows.start];
    int next = pick(a.vocab, segs, u, [&](int j) { return work.rest[(size_t)seq * segs + j]; }, rest);
    if (next < 0) {   // nothing is left
        const Segment* mine = work.segments + (size_t)e.row * segs;
        auto value = [&](int j) {
            const Segment g = mine[j];
            return g.top > -INFINITY ? g.sum * weight(g.top, e.m, e.c) : 0.;
        };
        __syncthreads();
        next = pick(a.vocab, segs, u, value, [&](int id) { return weight(logit<kHalf>(rest.row, id), e.m, e.c); });
    }
    if (threadIdx.x == 0) a.next_tokens[seq] = next;
}

int segments_of(int vocab) { return (vocab + kSeg - 1) / kSeg; }

template <bool kHalf>
void launch_for(const VerifyDrafts& a, hipStream_t s) {
    const int segs = segments_of(a.vocab), blocks = (segs + kWaves - 1) / kWaves;
    launch_kernel_in_call(false, verify_sums_kernel<kHalf>, dim3(blocks, a.max_query * (a.draft ? 2 : 1), a.nseq),
                          dim3(kBlk), 0, s, a, segs);
    launch_kernel_in_call(!a.draft, verify_walk_kernel<kHalf>, dim3(a.nseq), dim3(kBlk), 0, s, a, segs);
    if (!a.draft) return;
    launch_kernel_in_call(false, verify_rest_kernel<kHalf>, dim3(blocks, a.nseq), dim3(kBlk), 0, s, a, segs);
    launch_kernel(verify_pick_kernel<kHalf>, dim3(a.nseq), dim3(kBlk), 0, s, a, segs);
}

}  // namespace

hipError_t launch_draft_tree(const DraftTree& a, hipStream_t s) {
    const int words = (a.max_query + 63) / 64;
    launch_kernel(draft_tree_kernel, dim3(a.nseq), dim3(64 * words), 0, s, a, words);
    return hipGetLastError();
}

size_t verify_drafts_workspace(int nseq, int rows, int vocab, bool drafts) {
    const size_t segs = segments_of(vocab);
    size_t bytes = (size_t)rows * (drafts ? 2 : 1) * segs * sizeof(Segment);
    if (drafts) bytes += nseq * (sizeof(PathEnd) + segs * sizeof(double));
    return bytes;
}

hipError_t launch_verify_drafts(const VerifyDrafts& a, hipStream_t s) {
    if (a.half)
        launch_for<true>(a, s);
    else
        launch_for<false>(a, s);
    return hipGetLastError();
}

}  // namespace citlali::hip
