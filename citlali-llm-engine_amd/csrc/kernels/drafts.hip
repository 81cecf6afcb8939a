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
// and `above` is the row 2^t up.  128 trees of 256 rows are 1 MB, written in 4 to 5 us,
// eight rows' in 2: the launch and two round trips.  (A walk up the tree takes as many
// LDS reads in a row as it is deep.)
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
// Sums of segments of 2048 logits first, a wave each, then a workgroup per sequence for
// all that is in turn: the path, and the draw of its token.
// After the sums, five rows take 8 us, a chain of four with drafts 8.5, a tree of 40
// 11.5: one round trip and one reduction after another.
// ---------------------------------------------------------------------------
constexpr int kBlk = 256, kWaves = kBlk / kWave;
constexpr int kPer = 32, kSeg = kPer * kWave;   // logits of a lane, and of a wave: a segment
__device__ __forceinline__ int segment_of(int id) {   // below 0 for an id below 0
    static_assert(kSeg == 1 << 11);
    return id >> 11;
}

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
// The same for many z = d c: z is n / 256 + r with a whole n, 2^(n / 256) comes from a
// table of 256 and 2^r, |r| <= 1/512, by a polynomial of degree 3; off by 1e-13 at
// most, 2^0 is 1.  Adding 1.5 * 2^44 rounds z to 256ths and leaves n in the low bits;
// entry j's upper half is less by j << 12, so that n << 12 added to it is the
// exponent.  d is kept from -1000 / c on: 2^-1000 for all below.
struct Exp2Table {
    static constexpr int kEntries = 256;
    const double* table;   // of LDS
    double c, least;
    // by kThreads threads; they meet without waiting for their loads
    template <int kThreads>
    __device__ void make(double* room, double c_) {
        table = room;
        c = c_;
        least = -1000. / c_;
        for (int j = threadIdx.x; j < kEntries; j += kThreads) {
            u32x2 w = __builtin_bit_cast(u32x2, exp2_64(j * (1. / kEntries) - 1.));
            w.y += (1u << 20) - ((uint32_t)j << 12);   // (times 2)
            room[j] = __builtin_bit_cast(double, w);
        }
        lds_only_barrier();
    }
    struct Parts {
        double e, p;   // whose product it is
    };
    __device__ Parts parts(double d) const {
        d = fmax(d, least);
        constexpr double kRound = 0x1.8p44;
        const double t = fma(d, c, kRound), r = fma(d, c, kRound - t);
        const uint32_t n = __builtin_bit_cast(u32x2, t).x;
        u32x2 w = __builtin_bit_cast(u32x2, table[n & (kEntries - 1)]);
        w.y += n << 12;
        return {__builtin_bit_cast(double, w),
                fma(fma(fma(0.05550411247958329, r, 0.24022653447679007), r, 0.6931471805599453), r, 1.)};
    }
    __device__ double operator()(double d) const {
        const Parts v = parts(d);
        return v.e * v.p;
    }
    __device__ double add(double sum, double d) const {
        const Parts v = parts(d);
        return fma(v.e, v.p, sum);
    }
};
// Weight of a logit x against one of m >= x; c = log2(e) / T.
__device__ __forceinline__ double weight(float x, float m, double c) {
    return x == -INFINITY ? 0. : exp2_64(((double)x - (double)m) * c);
}

// ---- 64-bit moves between lanes --------------------------------------------------
template <int Ctrl, int kRows = 0xF>
__device__ __forceinline__ double dpp64(double v) {   // 0 where no lane is meant
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(double, u32x2{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, Ctrl, kRows, 0xF, false),
                                            (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, Ctrl, kRows, 0xF, false)});
}
__device__ __forceinline__ double lane64(double v, int lane) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(double, u32x2{(uint32_t)__builtin_amdgcn_readlane((int)w.x, lane),
                                            (uint32_t)__builtin_amdgcn_readlane((int)w.y, lane)});
}
// Sum over each row of 16 lanes, in all of them.
__device__ __forceinline__ double row_sum64(double v) {
    v += dpp64<kDppXor1>(v);
    v += dpp64<kDppXor2>(v);
    v += dpp64<DppRor<4>::value>(v);
    return v + dpp64<DppRor<8>::value>(v);
}
__device__ __forceinline__ double wave_sum64(double v) {
    v = row_sum64(v);
    return (lane64(v, 0) + lane64(v, 16)) + (lane64(v, 32) + lane64(v, 48));
}
// Sum over the lanes up to this one.
__device__ __forceinline__ double wave_scan64(double v) {
    v += dpp64<0x111>(v);   // row_shr 1, 2, 4, 8
    v += dpp64<0x112>(v);
    v += dpp64<0x114>(v);
    v += dpp64<0x118>(v);
    v += dpp64<0x142, 0xA>(v);   // lane 15 of a row to the next row, then lane 31 to the upper half
    return v + dpp64<0x143, 0xC>(v);
}
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp<kDppXor1>(v));
    v = fmaxf(v, dpp<kDppXor2>(v));
    v = fmaxf(v, dpp<DppRor<4>::value>(v));
    return fmaxf(v, dpp<DppRor<8>::value>(v));
}
__device__ __forceinline__ int row_min(int v) {
    for (int o = 1; o < 16; o <<= 1) v = min(v, __shfl_xor(v, o, kWave));
    return v;
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

// 0: greedy.  An infinite one as 2^200, at which finite logits, 2^129 apart at most, all
// weigh 1 (their exponents are below 2^-70) and -inf still nothing.
__device__ __forceinline__ double temperature(const VerifyDrafts& a, int seq) {
    const float t = a.temperatures ? a.temperatures[seq] : 1.f;
    return t > 0.f ? fmin((double)t, 0x1p200) : 0.;
}
constexpr double kLog2e = 1.4426950408889634074;

// A segment's logits as one wave has them: element e of a lane is id
// seg * kSeg + (e / kVec * 64 + lane) * kVec + e % kVec; -inf behind the last id.
template <bool kHalf>
struct Logits {
    static constexpr int kVec = kHalf ? 8 : 4, kLoads = kPer / kVec;
    u32x4 w[kLoads];   // fp32, or pairs of fp16
    __device__ void load(const void* row, int vocab, int seg, int lane) {
        const int id0 = seg * kSeg;
        constexpr int kSize = kHalf ? 2 : 4;
        if (id0 + kSeg <= vocab) {
            const char* at = static_cast<const char*>(row) + (size_t)id0 * kSize + lane * 16;
#pragma unroll
            for (int l = 0; l < kLoads; ++l) w[l] = *reinterpret_cast<const u32x4_a2*>(at + l * kWave * 16);
            return;
        }
        if (vocab >= kVec) {   // the row's last: what would reach behind it is read from before and moved down
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
                const int id = id_of(seg, l * kVec, lane);
                w[l] = *reinterpret_cast<const u32x4_a2*>(static_cast<const char*>(row) +
                                                          (size_t)min(id, vocab - kVec) * kSize);
            }
#pragma unroll
            for (int l = 0; l < kLoads; ++l) {
                const int by = id_of(seg, l * kVec, lane) - (vocab - kVec);
                w[l] = by <= 0 ? w[l] : by >= kVec ? u32x4{kNone, kNone, kNone, kNone} : moved(w[l], by);
            }
            return;
        }
#pragma unroll
        for (int l = 0; l < kLoads; ++l)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int id = id_of(seg, l * kVec + i * (kVec / 4), lane);
                if constexpr (kHalf) {
                    const uint16_t* x = static_cast<const uint16_t*>(row);
                    w[l][i] = (id < vocab ? x[id] : kNone & 0xffffu) | (id + 1 < vocab ? x[id + 1] : kNone >> 16) << 16;
                } else {
                    w[l][i] = id < vocab ? static_cast<const uint32_t*>(row)[id] : kNone;
                }
            }
    }
    static constexpr uint32_t kNone = kHalf ? 0xfc00fc00u : 0xff800000u;   // -inf
    // elements `by` .. of v, -inf behind them
    __device__ static u32x4 moved(u32x4 v, int by) {
        const int words = kHalf ? by >> 1 : by;
        if (words & 2) v = u32x4{v.z, v.w, kNone, kNone};
        if (words & 1) v = u32x4{v.y, v.z, v.w, kNone};
        if (kHalf && (by & 1))
            v = u32x4{v.x >> 16 | v.y << 16, v.y >> 16 | v.z << 16, v.z >> 16 | v.w << 16, v.w >> 16 | kNone << 16};
        return v;
    }
    __device__ float at(int e) const {
        const uint32_t v = w[e / kVec][kHalf ? e % kVec / 2 : e % kVec];
        return kHalf ? h2f((uint16_t)(e & 1 ? v >> 16 : v)) : __uint_as_float(v);
    }
    __device__ static int id_of(int seg, int e, int lane) {
        return seg * kSeg + (e / kVec * kWave + lane) * kVec + e % kVec;
    }
};

// Workgroup (4 segments, row, sequence), a segment a wave; every logit is read once.
// Bound by 64-bit instructions in fp16 (ten a logit, beside the table's read; the vector
// unit is busy for 77%): 14 trees of up to 40 rows of 151936, 131 MB, in 31 to 33 us.  By
// the reads in fp32: 40 chains of up to 6 and their drafts' logits, 200 MB, in 35 to 37
// (5.4 TB/s).  150 chains of up to 4 with drafts of 32003 in fp16, 47 MB, in 20.  By
// exp2_64 alone the first takes 85.  64 rows of 151936 to draw from: 11 in fp32, 9 in
// fp16, in calls of 17.7 and 16.0.  Several segments a wave, the next one loaded ahead,
// are no faster.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void verify_sums_kernel(VerifyDrafts a, int segs) {
    __shared__ double table[Exp2Table::kEntries];
    const int seq = blockIdx.z;
    const bool draft = (int)blockIdx.y >= a.max_query;
    const int i = blockIdx.y - (draft ? a.max_query : 0);
    const DraftRows rows = draft_rows(a.query_start, seq, a.rows, a.max_query);
    if (i >= rows.n || (draft && i + 1 >= rows.n)) return;   // the last row's draft has no child
    const int lane = threadIdx.x & (kWave - 1);
    const int seg = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const double t = temperature(a, seq);
    const int r = rows.start + i;
    Logits<kHalf> x;
    x.load(draft ? logit_row<kHalf>(a.draft, a.draft_stride, r) : logit_row<kHalf>(a.logits, a.stride, r), a.vocab,
           min(seg, segs - 1), lane);
    Exp2Table exp2;
    exp2.make<kBlk>(table, kLog2e / t);
    if (seg >= segs) return;
    float top = x.at(0);
#pragma unroll
    for (int e = 1; e < kPer; ++e) top = __builtin_elementwise_maximum(top, x.at(e));   // a NaN stays
    const bool bad = __builtin_amdgcn_ballot_w64(!(top < INFINITY)) != 0;
    top = wave_max(top);
    Segment out{0., bad ? NAN : top, 0};
    if (!bad && top > -INFINITY) {
        if (t > 0.) {
            double s[2] = {0., 0.};
#pragma unroll
            for (int e = 0; e < kPer; ++e) s[e % 2] = exp2.add(s[e % 2], (double)x.at(e) - (double)top);
            out.sum = wave_sum64(s[0] + s[1]);
        } else {
            int first = INT_MAX;
#pragma unroll
            for (int e = kPer - 1; e >= 0; --e)
                if (x.at(e) == top) first = x.id_of(seg, e, lane);
            first = row_min(first);
            out.first = min(min(__builtin_amdgcn_readlane(first, 0), __builtin_amdgcn_readlane(first, 16)),
                            min(__builtin_amdgcn_readlane(first, 32), __builtin_amdgcn_readlane(first, 48)));
        }
    }
    if (lane == 0) work_of(a, segs).segments[((size_t)(draft ? a.rows : 0) + r) * segs + seg] = out;
}

// ---- a draw by a workgroup of kWalk threads ---------------------------------------
constexpr int kWalk = 512, kWalkWaves = kWalk / kWave;
constexpr int kRun = kSeg / kWalk;   // ids of a thread

__device__ __forceinline__ float unit(float u) { return u >= 0.f ? fminf(u, 0x1.fffffep-1f) : 0.f; }

// The first of `count` values whose running sum exceeds t(total), and the sum before
// it; where rounding leaves none, the last that is above 0, with t infinite; -1 where
// the total is 0.  By every wave for itself: 64 blocks of them at a time, then the
// block that has it.
struct Place {
    int at;
    double before, t;
};
template <typename V>
__device__ __forceinline__ Place find_place(int count, float u, V value) {
    const int lane = threadIdx.x & (kWave - 1);
    Place f{0, 0., -1.};
    for (int n = count;;) {   // n values from f.at on
        const int each = (n + kWave - 1) / kWave;
        double v = 0.;
        for (int k = 0; k < each; ++k) {
            const int j = lane * each + k;
            v += j < n ? value(f.at + j) : 0.;
        }
        const double upto = wave_scan64(v);
        if (f.t < 0.) {
            const double total = lane64(upto, kWave - 1);
            if (!(total > 0.)) return {-1, 0., 0.};
            f.t = (double)unit(u) * total;
        }
        // (of those with a value: rounding does not order the sums, and the one of a lane
        // without may exceed the one before it)
        uint64_t who = __builtin_amdgcn_ballot_w64(v > 0. && f.before + upto > f.t);
        if (who == 0) {
            who = __builtin_amdgcn_ballot_w64(v > 0.);
            if (who == 0) return {-1, 0., 0.};
            who = 1ull << (63 - __builtin_clzll(who));
            f.t = INFINITY;
        }
        const int l = __builtin_ctzll(who);
        f.before += lane64(upto - v, l);
        f.at += l * each;
        if (each == 1) return f;
        n = min(each, n - l * each);
    }
}

// The first id whose running sum of weights exceeds u times their total; -1 where
// the total is 0.  value(j): the sum of segment j's weights; weights(id, w): those of
// the kRun ids from `id` on.
template <typename V, typename W>
__device__ int pick(int segs, float u, V value, W weights) {
    __shared__ double sums[kWalkWaves];
    __shared__ int hits[kWalkWaves], lasts[kWalkWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const Place f = find_place(segs, u, value);
    if (f.at < 0) return -1;
    const int id0 = f.at * kSeg + (int)threadIdx.x * kRun;
    double w[kRun], sum = 0.;
    weights(id0, w);
#pragma unroll
    for (int e = 0; e < kRun; ++e) sum += w[e];
    const double upto = wave_scan64(sum);
    if (lane == kWave - 1) sums[wave] = upto;
    __syncthreads();
    double run = f.before;
#pragma unroll
    for (int k = 0; k < kWalkWaves - 1; ++k) run += k < wave ? sums[k] : 0.;
    run += upto - sum;
    int hit = INT_MAX, last = -1;
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
        run += w[e];
        if (w[e] > 0.) {
            last = id0 + e;
            hit = hit == INT_MAX && run > f.t ? last : hit;
        }
    }
    // the wave's first hit, and its last id with a weight: for where rounding leaves no hit
    const uint64_t who = __builtin_amdgcn_ballot_w64(hit < INT_MAX), have = __builtin_amdgcn_ballot_w64(last >= 0);
    if (lane == 0) {
        hits[wave] = INT_MAX;
        lasts[wave] = -1;
    }
    wave_lds_sync();
    if (who != 0 && lane == __builtin_ctzll(who)) hits[wave] = hit;
    if (have != 0 && lane == 63 - __builtin_clzll(have)) lasts[wave] = last;
    __syncthreads();
    int first = INT_MAX, end = -1;
#pragma unroll
    for (int k = 0; k < kWalkWaves; ++k) {
        first = min(first, hits[k]);
        end = max(end, lasts[k]);
    }
    return first < INT_MAX ? first : end;
}
// kRun logits of a row from id on, -inf behind the last.
template <bool kHalf>
__device__ __forceinline__ void load_run(const void* row, int id, int vocab, float (&x)[kRun]) {
    static_assert(kRun == 4);
    if (id + kRun <= vocab) {
        if constexpr (kHalf) {
            const u32x2 v = *reinterpret_cast<const u32x2_a2*>(static_cast<const uint16_t*>(row) + id);
#pragma unroll
            for (int e = 0; e < kRun; ++e) x[e] = h2f((uint16_t)(v[e / 2] >> (e % 2 * 16)));
        } else {
            const u32x4 v = *reinterpret_cast<const u32x4_a2*>(static_cast<const float*>(row) + id);
#pragma unroll
            for (int e = 0; e < kRun; ++e) x[e] = __uint_as_float(v[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < kRun; ++e) {
            const float v = logit<kHalf>(row, min(id + e, vocab - 1));
            x[e] = id + e < vocab ? v : -INFINITY;
        }
    }
}

// Largest logit, sum and first id of a row.
struct RowSum {
    double s;
    float m;   // NaN: no distribution
    int first;
};
// A row's segments joined by 16 lanes.
constexpr int kRowLanes = 16;
__device__ RowSum join_segments(const Segment* at, int segs, bool greedy, double c) {
    constexpr int kBatch = 5;
    const int lane = threadIdx.x & (kWave - 1);
    float m = -INFINITY;
    double s = 0.;
    int first = INT_MAX;
    bool bad = false;
    for (int j0 = lane % kRowLanes; j0 < segs; j0 += kBatch * kRowLanes) {
        Segment g[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int j = j0 + b * kRowLanes;
            g[b] = at[min(j, segs - 1)];
            if (j >= segs) g[b].top = -INFINITY;
        }
        float most = m;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            bad |= g[b].top != g[b].top;
            most = fmaxf(most, g[b].top);
        }
        if (greedy) {
            int here = INT_MAX;   // (the lowest ids come first)
#pragma unroll
            for (int b = kBatch - 1; b >= 0; --b)
                if (g[b].top == most) here = g[b].first;
            first = most > m ? here : first;
        } else if (most > -INFINITY) {
            s *= weight(m, most, c);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) s = fma(g[b].sum, weight(g[b].top, most, c), s);
        }
        m = most;
    }
    RowSum r{0., row_max(m), 0};
    if (greedy)
        r.first = row_min(m == r.m ? first : INT_MAX);
    else if (r.m > -INFINITY)
        r.s = row_sum64(s * weight(m, r.m, c));
    const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
    if ((any >> (lane & 48) & 0xffff) != 0 || r.m == -INFINITY) r.m = NAN;
    return r;
}

// max(p - q, 0) of the row where a path ended.
template <bool kHalf>
struct Rest {
    const void *row, *draft_row;
    PathEnd e;
    double inv, inv_draft;
    __device__ Rest(const VerifyDrafts& a, const PathEnd& end)
        : row(logit_row<kHalf>(a.logits, a.stride, end.row)),
          draft_row(logit_row<kHalf>(a.draft, a.draft_stride, end.row)), e(end), inv(1. / end.s),
          inv_draft(1. / end.s_draft) {}
    __device__ double of(double w, double w_draft) const {
#pragma clang fp contract(off)   // equal p and q leave nothing
        return fmax(w * inv - w_draft * inv_draft, 0.);
    }
    // of one id
    __device__ double of(float x, float d, const Exp2Table& exp2) const {
        const double dx = (double)x - (double)e.m, dd = (double)d - (double)e.m_draft;
        const double w = exp2(dx), w_draft = exp2(dd);
        return of(dx > exp2.least ? w : 0., dd > exp2.least ? w_draft : 0.);
    }
    // of kRun ids from id on: the same numbers as in their segment's sum, so that one which
    // is above 0 has an id that is
    __device__ void run(int id, int vocab, const Exp2Table& exp2, double (&w)[kRun]) const {
        float x[kRun], d[kRun];
        load_run<kHalf>(row, id, vocab, x);
        load_run<kHalf>(draft_row, id, vocab, d);
#pragma unroll
        for (int k = 0; k < kRun; ++k) w[k] = of(x[k], d[k], exp2);
    }
};
// A segment of it, by one wave.
template <bool kHalf>
struct RestLogits {
    Logits<kHalf> x, d;
    __device__ void load(const Rest<kHalf>& r, int vocab, int seg, int lane) {
        x.load(r.row, vocab, seg, lane);
        d.load(r.draft_row, vocab, seg, lane);
    }
    __device__ double sum(const Rest<kHalf>& r, const Exp2Table& exp2) const {
        double sum[2] = {0., 0.};
#pragma unroll
        for (int k = 0; k < kPer; ++k) sum[k % 2] += r.of(x.at(k), d.at(k), exp2);
        return wave_sum64(sum[0] + sum[1]);
    }
};
// Rows of up to kAloneSegs segments, two a wave: the workgroup that finds the path sums
// what q leaves of them too (150 sequences of 32003 tokens: 19 us in all), without the
// two launches that take longer rows'.  Calls with every draft rejected, fp32, so and by
// those launches: of 16000 tokens 1 sequence 17.1 / 18.7 us, 40 21.5 / 23.2, 150 30.3 /
// 34.8; of 32003 150 43.8 / 47.2, 256 62.3 / 66.1, but few sequences leave CUs idle: 1
// 22.1 / 18.5, 40 28.7 / 26.2.
constexpr int kAloneSegs = 2 * kWalkWaves;

// ---------------------------------------------------------------------------
// One workgroup per sequence: the rows' sums, the drafted tokens' probabilities, the
// path, and the next token but where it comes from what q leaves of p.
// ---------------------------------------------------------------------------
template <bool kHalf>
__global__ __launch_bounds__(kWalk) void verify_walk_kernel(VerifyDrafts a, int segs) {
    __shared__ RowSum sums[2 * kMaxTree];   // the rows', then their drafts'
    __shared__ int parent[kMaxTree], token[kMaxTree], gone[kMaxTree], path[kMaxTree];
    __shared__ double p[kMaxTree], bar[kMaxTree], gone_p[kMaxTree], gone_sum[kMaxTree];
    __shared__ double end_left;
    __shared__ double table[Exp2Table::kEntries], rest_sum[kAloneSegs];
    __shared__ int end_row, end_lost, end_count;
    const int seq = blockIdx.x, lane = threadIdx.x & (kWave - 1), tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const DraftRows rows = draft_rows(a.query_start, seq, a.rows, a.max_query);
    const Work work = work_of(a, segs);
    if (rows.n <= 0) {
        if (a.paths)
            for (int i = tid; i < a.max_query; i += kWalk) a.paths[(size_t)seq * a.max_query + i] = -1;
        if (tid == 0) {
            if (a.counts) a.counts[seq] = 0;
            a.next_tokens[seq] = -1;
            if (a.draft) work.ends[seq].rest = 0;
        }
        return;
    }
    const double heat = temperature(a, seq);
    const bool greedy = !(heat > 0.);
    const double c = greedy ? 0. : kLog2e / heat;
    const float u0 = a.uniforms[rows.start];
    // a row's draft and its logits, on their way beside the rows' sums
    int up = -1, x = -1;
    float u = 0.f, x_logit = -INFINITY, x_draft = -INFINITY;
    if (tid < rows.n) {
        const int r = rows.start + tid;
        up = a.parents ? a.parents[r] : tid - 1;
        if (up < 0 || up >= tid) up = -1;
        x = up >= 0 ? a.tokens[r] : -1;
        u = unit(a.uniforms[r]);
        if (x < 0 || x >= a.vocab) x = -1;
        if (x >= 0) {
            x_logit = logit<kHalf>(logit_row<kHalf>(a.logits, a.stride, rows.start + up), x);
            if (a.draft) x_draft = logit<kHalf>(logit_row<kHalf>(a.draft, a.draft_stride, rows.start + up), x);
        }
    }
    const int joined = rows.n + (a.draft ? rows.n - 1 : 0);
    for (int v = tid / kRowLanes; v < joined; v += kWalk / kRowLanes) {
        const bool of_draft = v >= rows.n;
        const int i = of_draft ? v - rows.n : v;
        const RowSum r = join_segments(
            work.segments + ((size_t)(of_draft ? a.rows : 0) + rows.start + i) * segs, segs, greedy, c);
        if (tid % kRowLanes == 0) sums[(of_draft ? kMaxTree : 0) + i] = r;
    }
    __syncthreads();
    if (tid < rows.n) {
        double mine = 0., against = 1.;
        if (x >= 0) {
            const RowSum s = sums[up];
            if (s.m == s.m) mine = greedy ? x == s.first : weight(x_logit, s.m, c) / s.s;
        }
        if (a.draft && up >= 0) {
            const RowSum d = sums[kMaxTree + up];
            against = d.m != d.m ? INFINITY   // no distribution: rejected
                      : x < 0    ? 0.
                      : greedy   ? x == d.first
                                 : weight(x_draft, d.m, c) / d.s;
        }
        parent[tid] = up;
        token[tid] = x;
        p[tid] = mine;
        bar[tid] = against == INFINITY ? INFINITY : (double)u * against;
        if (a.token_probs) a.token_probs[rows.start + tid] = (float)mine;
    }
    __syncthreads();
    if (wave == 0) {   // the path; the lanes have 64 rows at a time
        int above = -1, mark = -1;
        double chance = 0., limit = 0.;
        auto look_at = [&](int from) {
            const int i = min(from + lane, rows.n - 1);
            above = from + lane < rows.n ? parent[i] : -1;
            mark = token[i];
            chance = p[i];
            limit = bar[i];
        };
        int current = 0, at = 0, from = 0, count = 1, lost = 0;
        double left = 1.;
        look_at(0);
        for (;;) {
            const uint64_t who = __builtin_amdgcn_ballot_w64(above == current && from + lane > at);
            if (who == 0) {
                from += kWave;
                if (from >= rows.n) break;
                look_at(from);
                continue;
            }
            const int l = __builtin_ctzll(who), its_mark = __builtin_amdgcn_readlane(mark, l);
            at = from + l;
            bool again = false;   // rejected before
            for (int g = lane; g < lost; g += kWave) again |= gone[g] == its_mark;
            const double mine = __builtin_amdgcn_ballot_w64(again) != 0 ? 0. : lane64(chance, l);
            if (lane64(limit, l) * (a.draft ? 1. : left) < mine) {
                current = at;
                if (lane == 0) path[count] = at;
                ++count;
                lost = 0;
                left = 1.;
            } else {
                left -= mine;
                if (lane == 0) {
                    gone[lost] = its_mark;
                    gone_p[lost] = mine;
                }
                ++lost;
                wave_lds_sync();
            }
        }
        if (lane == 0) {
            path[0] = 0;
            end_row = current;
            end_lost = lost;
            end_count = count;
            end_left = left;
        }
    }
    __syncthreads();
    const int f = end_row, lost = end_lost;
    if (a.paths)
        for (int i = tid; i < a.max_query; i += kWalk)
            a.paths[(size_t)seq * a.max_query + i] = i < end_count ? path[i] : -1;
    if (a.counts && tid == 0) a.counts[seq] = end_count;
    const RowSum s = sums[f];
    bool rest = false;
    if (a.draft) {
        const RowSum d = sums[kMaxTree + f];
        rest = lost > 0 && s.m == s.m && !greedy && d.m == d.m;
        const PathEnd end = rest ? PathEnd{s.s, d.s, s.m, d.m, rows.start + f, 1, c} : PathEnd{};
        if (tid == 0) work.ends[seq] = end;
        if (rest && segs > kAloneSegs) return;
        if (rest) {
            const Rest<kHalf> left(a, end);
            Exp2Table exp2;
            exp2.make<kWalk>(table, c);
            for (int seg = wave; seg < segs; seg += kWalkWaves) {
                RestLogits<kHalf> l;
                l.load(left, a.vocab, seg, lane);
                const double sum = l.sum(left, exp2);
                if (lane == 0) rest_sum[seg] = sum;
            }
            __syncthreads();
            const int next = pick(
                segs, u0, [&](int j) { return rest_sum[j]; },
                [&](int id, double (&w)[kRun]) { left.run(id, a.vocab, exp2, w); });
            if (next >= 0) {
                if (tid == 0) a.next_tokens[seq] = next;
                return;
            }
            __syncthreads();   // nothing is left: the token comes from p
        }
    }
    int next = -1;
    if (s.m == s.m) {
        if (greedy) {
            next = s.first;
        } else {
            const void* row = logit_row<kHalf>(a.logits, a.stride, rows.start + f);
            const Segment* mine = work.segments + ((size_t)rows.start + f) * segs;
            const int out = a.draft ? 0 : lost;   // rejected tokens, left out
            // What is left of their segments, a wave each: the sum less their weights, an
            // error of 2^-43 of p in all; summed anew without them where that counts, with
            // less than a sixteenth of p left, or leaves hardly more than it.  A segment of
            // several is summed for the first.  A call with 4, 60 or 255 children of one row
            // of 151936 tokens, all rejected with a fiftieth of p left: 20, 157 and 443 us
            // with tokens all over the row, 54 and 188 with the last two in one segment (by
            // a sum for each token, every id against every token: 27, 916 and 13800).
            for (int g = wave; g < out; g += kWalkWaves) {
                const int seg = segment_of(__builtin_amdgcn_readfirstlane(gone[g]));
                bool again = seg < 0;
                for (int k = lane; k < g; k += kWave) again |= segment_of(gone[k]) == seg;
                if (__builtin_amdgcn_ballot_w64(again) != 0) continue;
                const Segment whole = mine[seg];
                const double all = whole.sum * weight(whole.top, s.m, c);
                double sum = all;
                if (end_left >= 0.0625)
#pragma unroll 8
                    for (int k = 0; k < out; ++k) sum -= segment_of(gone[k]) == seg ? gone_p[k] * s.s : 0.;
                if (end_left < 0.0625 || !(sum >= all * 0x1p-40)) {
                    const int id0 = seg * kSeg, id1 = min(a.vocab, id0 + kSeg);
                    uint32_t is_out = 0;   // which of the lane's ids, every 64th
                    static_assert(kPer == 32);
#pragma unroll 8
                    for (int k = 0; k < out; ++k) {
                        const int id = gone[k] - id0;
                        is_out |= segment_of(id) == 0 && id % kWave == lane ? 1u << id / kWave : 0u;
                    }
                    sum = 0.;
#pragma unroll 4
                    for (int id = id0 + lane; id < id1; id += kWave) {
                        const double v = weight(logit<kHalf>(row, id), s.m, c);
                        sum += is_out & 1u ? 0. : v;
                        is_out >>= 1;
                    }
                    sum = wave_sum64(sum);
                }
                if (lane == 0) gone_sum[g] = sum;
            }
            if (out > 0) __syncthreads();
            auto draw = [&](int left_out) {
                auto value = [&](int j) {
                    const Segment g = mine[j];
                    const double v = g.top > -INFINITY ? g.sum * weight(g.top, s.m, c) : 0.;
                    int first = -1;   // of its rejected tokens
#pragma unroll 8
                    for (int k = left_out - 1; k >= 0; --k) first = segment_of(gone[k]) == j ? k : first;
                    return first < 0 ? v : gone_sum[first];
                };
                return pick(segs, u0, value, [&](int id, double (&w)[kRun]) {
                    float l[kRun];
                    load_run<kHalf>(row, id, a.vocab, l);
#pragma unroll 4
                    for (int k = 0; k < left_out; ++k)
#pragma unroll
                        for (int e = 0; e < kRun; ++e) l[e] = gone[k] == id + e ? -INFINITY : l[e];
#pragma unroll
                    for (int e = 0; e < kRun; ++e) w[e] = weight(l[e], s.m, c);
                });
            };
            next = draw(out);
            if (next < 0) {   // nothing is left
                __syncthreads();
                next = draw(0);
            }
        }
    }
    if (tid == 0) a.next_tokens[seq] = next;
}

// Workgroup (4 segments, sequence): what q leaves of p where a draft was rejected.  40
// sequences of 151936 tokens, 49 MB at most: 9 us, and 5 for the pick.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void verify_rest_kernel(VerifyDrafts a, int segs) {
    __shared__ double table[Exp2Table::kEntries];
    const int seq = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    const int seg = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const Work work = work_of(a, segs);
    const PathEnd e = work.ends[seq];
    if (!e.rest) return;
    const Rest<kHalf> rest(a, e);
    RestLogits<kHalf> x;
    x.load(rest, a.vocab, min(seg, segs - 1), lane);
    Exp2Table exp2;
    exp2.make<kBlk>(table, e.c);
    if (seg >= segs) return;
    const double sum = x.sum(rest, exp2);
    if (lane == 0) work.rest[(size_t)seq * segs + seg] = sum;
}

template <bool kHalf>
__global__ __launch_bounds__(kWalk) void verify_pick_kernel(VerifyDrafts a, int segs) {
    __shared__ double table[Exp2Table::kEntries];
    const int seq = blockIdx.x;
    const Work work = work_of(a, segs);
    const PathEnd e = work.ends[seq];
    if (!e.rest) return;
    Exp2Table exp2;
    exp2.make<kWalk>(table, e.c);
    const DraftRows rows = draft_rows(a.query_start, seq, a.rows, a.max_query);
    const float u = a.uniforms[rows.start];
    const Rest<kHalf> rest(a, e);
    int next = pick(
        segs, u, [&](int j) { return work.rest[(size_t)seq * segs + j]; },
        [&](int id, double (&w)[kRun]) { rest.run(id, a.vocab, exp2, w); });
    if (next < 0) {   // nothing is left
        __syncthreads();
        const Segment* mine = work.segments + (size_t)e.row * segs;
        auto value = [&](int j) {
            const Segment g = mine[j];
            return g.top > -INFINITY ? g.sum * weight(g.top, e.m, e.c) : 0.;
        };
        next = pick(segs, u, value, [&](int id, double (&w)[kRun]) {
            float x[kRun];
            load_run<kHalf>(rest.row, id, a.vocab, x);
#pragma unroll
            for (int k = 0; k < kRun; ++k) w[k] = weight(x[k], e.m, e.c);
        });
    }
    if (threadIdx.x == 0) a.next_tokens[seq] = next;
}

int segments_of(int vocab) { return (vocab + kSeg - 1) / kSeg; }

template <bool kHalf>
void launch_for(const VerifyDrafts& a, hipStream_t s) {
    const int segs = segments_of(a.vocab), blocks = (segs + kWaves - 1) / kWaves;
    launch_kernel_in_call(false, verify_sums_kernel<kHalf>, dim3(blocks, a.max_query * (a.draft ? 2 : 1), a.nseq),
                          dim3(kBlk), 0, s, a, segs);
    const bool last = !a.draft || segs <= kAloneSegs;
    launch_kernel_in_call(last, verify_walk_kernel<kHalf>, dim3(a.nseq), dim3(kWalk), 0, s, a, segs);
    if (last) return;
    launch_kernel_in_call(false, verify_rest_kernel<kHalf>, dim3(blocks, a.nseq), dim3(kBlk), 0, s, a, segs);
    launch_kernel(verify_pick_kernel<kHalf>, dim3(a.nseq), dim3(kWalk), 0, s, a, segs);
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
