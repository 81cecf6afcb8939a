// kv4_attention.hip -- attention over the paged cache of 4-bit keys and values:
// causal, or of a tree of drafted tokens.
#include "kv4.hpp"

#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

namespace citlali::hip {
namespace {

// The largest of three (a NaN stays): one v_maximum3_f32.  Not asm: its operands
// come from matrix instructions, and only for an instruction of its own does the
// compiler keep the wait states between the two.  Not fmaxf: that first makes a
// quiet NaN of each operand.
__device__ __forceinline__ float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// l + the sum of eight weights as the product with V takes them: what their
// rounding to fp16 does is then in numerator and denominator alike.
__device__ __forceinline__ float add_weights(half8 w, float l) {
    const u32x4 pairs = __builtin_bit_cast(u32x4, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) l = dot2(pairs[i], 0x3c003c00u, l);   // times 1, 1
    return l;
}

// The queries of sequence `seq`: rows start .. start + n - 1 of q, the cached
// positions that exist, how many of them query i sees some of (see()), and how
// many every query from i on sees all of (all()).  In a tree the n last positions
// are the rows' own; which of them a row sees its mask says.
template <bool kTree>
struct Kv4Seq {
    int start, n, context, cap;
    __device__ int see(int i) const { return min(kTree ? context : context - n + i + 1, cap); }
    __device__ int all(int i) const { return kTree ? min(before(), cap) : see(i); }
    __device__ int before() const { return context - n; }
};
// Bits p .. p + 31 of a row's mask: set before it (p < 0), clear behind it.
__device__ __forceinline__ uint32_t tree_bits(const uint32_t* row, int words, int p) {
    auto word = [&](int k) { return k < 0 ? 0xffffffffu : k < words ? row[k] : 0u; };
    return __builtin_amdgcn_alignbit(word((p >> 5) + 1), word(p >> 5), p & 31);
}
template <bool kTree>
__device__ __forceinline__ Kv4Seq<kTree> kv4_seq(const Kv4Attention& a, int seq) {
    Kv4Seq<kTree> s;
    int end;
    if (a.query_start != nullptr) {
        s.start = min(max(a.query_start[seq], 0), a.tokens);
        end = min(max(a.query_start[seq + 1], s.start), a.tokens);
    } else {
        s.start = seq;
        end = seq + 1;
    }
    s.n = end - s.start;
    s.context = max(a.context_lens[seq], 0);
    s.cap = a.max_context;
    return s;
}

// Chunks of a sequence whose rows all see some of its last positions; one where there
// are no positions.
__device__ __forceinline__ int kv4_chunks(const Kv4Seq<true>& s, int chunk) {
    return max(1, (min(s.context, s.cap) + chunk - 1) / chunk);
}

// V of four positions that some rows do not see: a weight of 0 would not keep a
// NaN from them.  Clears the scales (d of four positions, then m) of those whose
// m is NaN -- their codes are 0 -- and returns them as bits.
__device__ __forceinline__ uint32_t kv4_hide_nan(u32x4& dm) {
    uint32_t nan = 0;
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        const bool lo = (dm[2 + y] & 0x7fffu) > 0x7c00u, hi = (dm[2 + y] & 0x7fff0000u) > 0x7c000000u;
        const uint32_t keep = (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
        dm[y] &= keep;
        dm[2 + y] &= keep;
        nan |= ((lo ? 1u : 0u) | (hi ? 2u : 0u)) << (2 * y);
    }
    return nan;
}

// The sequence of workgroup x (of a layer of nseq sequences).  An XCD deals its
// workgroups to its four shader engines in strict turn, those without work
// too, so a sequence's place has to change from layer to layer: by nseq where
// that is odd, else by one more (16 long contexts 87.7 -> 82.0 us, 24 sequences
// of 20 rows 40.3 -> 36.8).
__device__ __forceinline__ int seq_of(int x, int layer, int nseq) {
    return (x + (nseq & 1 ? 0 : layer)) % nseq;
}

constexpr int kBlk = 256, kWaves = kBlk / kWave;
constexpr float kShift = 14.f;   // weights are kept times 2^14 (base 2)
// The maximum that weights refer to moves only when it is exceeded by kSlack (base
// 2; kSlackScore of a score); beyond kFar a reference is taken off the scores first.
constexpr float kSlack = 4.f, kFar = 1024.f;
template <int HD>
constexpr float kSlackScore = kSlack * 0.693147181f * (HD == 128 ? 11.3137085f : 8.f);   // kSlack / scale_log2

// 2^((a - b) scale) of scores a <= b, of which -inf is none at all.  The maxima
// that weights and sums refer to are kept as scores: a difference of scores is as
// exact as they are, one of their multiples of scale_log2 need not be, and from
// 2^25 on (queries and keys of some thousands) is off by any factor.
__device__ __forceinline__ float score_factor(float a, float b, float scale_log2) {
    return a == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((a - b) * scale_log2);
}

// ---------------------------------------------------------------------------
// Few rows: one workgroup per (chunk of positions, kv head, sequence) serves
// every query of the sequence for every head of the kv head's group, at most
// 16 kCols rows (row r: query r / group, head r % group), so the cache is read
// once.  The waves, four or eight, take tiles of 32 positions in turn, without LDS
// until they merge:
//  * S^T[position][row] = K Q^T by v_mfma_f32_16x16x32_f16, 16 positions at a
//    time: lane (col, grp) of the A operand holds position col's dims
//    grp * HD/4 .. + HD/4 - 1, one 16-byte (head_dim 64: 8-byte) load of codes
//    with one (d, m); Q, the B operand, is held in the same dim order (in LDS
//    beyond 16 rows: that leaves registers for three waves per SIMD at 32).  Three of
//    the tree's instances do not quite fit theirs: heads of 128 at 17 to 32 rows spill 36
//    bytes a lane, 8 of them read again in every turn before V is asked for, at 16 rows
//    8 and heads of 64 at 33 to 48 rows 16, outside the loop over the prefix.
//  * online softmax down each column (row of Q): a lane has 8 of a tile's 32
//    positions, the maximum takes two permlane swaps, the sum stays per lane
//    until the end.
//  * O^T[dim][row] += V^T P^T: the lanes' weights are the B operand as they
//    stand (k index = grp 4 + i of the first 16 positions, then of the second),
//    rounded to fp16 -- times 2^14, so that weights down to 2^-28 of the largest
//    keep all their bits (of a tree's row times 2^10 to 2^14, as far as its reference
//    lags behind the largest score: down to 2^-24); their sum takes them so too.  V lies in groups of
//    four tokens, so lane (c, grp) loads the codes of its four positions and
//    HD / 16 dims together, each word two positions' dims, and gets the A
//    operand's pairs without a transposition.
// Bound by the cache's bytes where contexts are long; else by the round trips of a
// workgroup's start and by the unequal lengths of the one round of workgroups: the
// vector unit (about 300 instructions a tile of 5 KB at head_dim 128, 215 a tile of
// 2.5 KB at 64) is busy for half of the time in each causal case below but the first.
// 32/8 heads of 128: 16 sequences of 4096 .. 32768
// positions, 403 MB, in 78 us (5.1 TB/s), 64 of 200 .. 4000, 174 MB, in 38.7 (4.5);
// 20 rows, 24 sequences of 500 .. 6000, 101 MB, in 31.0; 16/8 heads of 64, 100
// sequences of 150 .. 1500, 52.6 MB, in 17.6.
// Of a tree (kTree): 48 sequences of 200 .. 4000, 28 to 48 rows of 32/8 heads of 128,
// 154 MB, in 63 to 66; 25 of 176 .. 2500, 34 to 66 rows of 16/8 of 64, 22 MB, in 22.7.
// No unit is busy for half of it (vector units 43% and 33%, matrix units 14% and 9%): a
// chunk's start and end, 5 us of 16 in the first, and CUs with five chunks where others
// have four.  Chains of up to 8 as trees, 32 rows, and by the causal kernel: calls of 24
// sequences of 200 .. 4000 36.3 and 35.9 us, of 64 69.7 and 68.1; of up to 4, 16 rows,
// 24.7 and 24.8, 47.4 and 47.7.
// ---------------------------------------------------------------------------
template <int HD, int kCols, bool kTree, int kWaves = 4>
__global__ __launch_bounds__(kWaves * kWave, kWaves > 4 ? 2 : kCols == 1 ? 4
                                             : kCols == 2 || (kTree && HD == 64 && kCols == 3) ? 3 : 2)
void kv4_decode_kernel(Kv4View c, Kv4Attention a, int chunk, int n_splits, float scale_log2) {
    constexpr int kBlk = kWaves * kWave;
    using L = Kv4Layout<HD>;
    using Vec = std::conditional_t<HD == 128, u32x4, u32x2>;   // a lane's codes of 16 positions
    constexpr int kSteps = HD / 32, kDims = HD / 16;   // MFMA steps of a score; dims (and O tiles) of a V lane
    // the waves' merge of 16 rows: [wave][row][HD + 4], sums behind HD
    extern __shared__ __align__(16) float lds[];

    // every sequence's first chunks before the second ones: the chunks that
    // short sequences lack then leave all XCDs alike
    const int split = blockIdx.y, kvh = blockIdx.x % c.kv_heads, seq = seq_of(blockIdx.x / c.kv_heads, split, a.nseq);
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, grp = lane >> 4;
    // the chunk's pages, one a lane (a chunk has at most 64), with the lengths
    // still on their way
    const int c0 = split * chunk, first_page = c0 >> c.page_shift;
    int my_page = a.page_table[(size_t)seq * a.pages_per_seq + min(first_page + lane, a.pages_per_seq - 1)];
    const Kv4Seq<kTree> s = kv4_seq<kTree>(a, seq);
    const int asked = min(s.n, a.max_query);
    if (asked <= 0) return;
    const int group = a.heads / c.kv_heads, rows = asked * group;
    const int most = max(0, s.see(asked - 1));   // positions any row sees
    const int c1 = min(most, c0 + chunk);
    if (c0 >= most && split > 0) return;
    if (((first_page + lane) << c.page_shift) >= c1 || my_page >= c.num_pages) my_page = -1;
    constexpr bool kQInLds = kCols > 1;
    half8 q[kQInLds ? 1 : kCols][kSteps];
    int see[kCols];   // positions a row sees; in a tree the row (-1: none)
    half8* const q_lds = reinterpret_cast<half8*>(lds);   // [column tile][step][lane]
    u32x4 mine[kTree && kQInLds ? kCols : 1];             // (a row that is none has another's)
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
        const int r = col + 16 * n, i = r / group;
        const bool real = r < rows;
        see[n] = kTree ? (real ? s.start + i : -1) : real ? s.see(i) : 0;
        const uint16_t* qr = a.q + (size_t)(s.start + (real ? i : 0)) * a.q_stride +
                             (size_t)(kvh * group + (real ? r - i * group : 0)) * HD + grp * (HD / 4);
        if constexpr (kTree && kQInLds) {   // a piece a wave, written once all are on their way
            mine[n] = *reinterpret_cast<const u32x4*>(qr + 8 * (wave % kSteps));
            continue;
        }
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
            u32x4 v = *reinterpret_cast<const u32x4*>(qr + 8 * t);
            if (!real) v = u32x4{0u, 0u, 0u, 0u};
            if constexpr (kQInLds) {
                if ((n * kSteps + t) % kWaves == wave)
                    q_lds[(n * kSteps + t) * kWave + lane] = __builtin_bit_cast(half8, v);
            } else {
                q[n][t] = __builtin_bit_cast(half8, v);
            }
        }
    }
    const int least = s.all(0);   // positions every row sees

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
    // uniform addresses plus a lane's own offsets
    const uint32_t at_k = col * L::kCodes + grp * (HD / 8), at_kp = col * L::kParams + (HD == 128 ? grp : grp >> 1) * 4;
    const uint32_t at_v = grp * (4 * L::kCodes) + col * (HD / 8);
    const uint32_t at_vp = grp * (4 * L::kParams) + col / (512 / HD) * 16;
    const uint8_t* at_head[2];
    auto read = [](auto* to, const uint8_t* from) {
        *to = __builtin_nontemporal_load(reinterpret_cast<decltype(to)>(const_cast<uint8_t*>(from)));
    };
    auto load_k = [&](int t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int o = (t + 16 * u) & (P - 1) & ~15;
            at_head[u] = head_at(t + 16 * u);
            read(&xk[u], at_head[u] + o * L::kCodes + at_k);
            read(&xkp[u], at_head[u] + L::k_params(P) + o * L::kParams + at_kp);
        }
    };
    auto load_v = [&](int t) {   // of the positions that load_k took last
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int o = (t + 16 * u) & (P - 1) & ~15;
            read(&xv[u], at_head[u] + L::v_codes(P) + o * L::kCodes + at_v);
            read(&xvp[u], at_head[u] + L::v_params(P) + o * L::kParams + at_vp);
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
    if constexpr (kTree && kQInLds) {
#pragma unroll
        for (int n = 0; n < kCols; ++n)
            if (wave / kSteps == n % (kWaves / kSteps))
                q_lds[(n * kSteps + wave % kSteps) * kWave + lane] = __builtin_bit_cast(half8, mine[n]);
    }
    if constexpr (kQInLds) lds_only_barrier();
    __builtin_amdgcn_sched_barrier(0);
    // A tree's tiles with positions of its rows have a loop of their own: with the masks
    // in one the compiler keeps less in registers (64 rows of 16384 positions on the
    // prompt kernel, below: 121 us for 95).
    int t = c0 + 32 * wave;
#pragma unroll
    for (int phase = kTree ? 0 : 1; phase < 2; ++phase)
    for (const bool tail = kTree && phase == 1; t < (kTree && !tail ? min(c1, s.before() - 31) : c1);
         t += 32 * kWaves) {
        const int there = (page_of(t) >= 0) | (page_of(t + 16) >= 0) << 1;
        const bool whole = there == 3 && t + 32 <= least;
        f32x4 sc[kCols][2];
        int q_at = lane;
        if constexpr (kQInLds) asm volatile("" : "+v"(q_at));   // read in every turn, not kept
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
                for (int n = 0; n < kCols; ++n) {
                    const half8 row = kQInLds ? q_lds[(n * kSteps + st) * kWave + q_at] : q[kQInLds ? 0 : n][st];
                    sc[n][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, row, sc[n][u], 0, 0, 0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(t + 32 * kWaves);   // in flight through the softmax and V
        __builtin_amdgcn_sched_barrier(0);
        half8 pw[kCols];
        uint32_t sees[kTree ? kCols : 1];   // of a tree's row, the tile's positions
#pragma unroll
        for (int n = 0; n < kCols; ++n) {
            if constexpr (kTree && kCols > 1) {   // (48 trees of 28 to 48 rows: 69.1 -> 66.1 us)
                pw[n] = half8{};
                if (16 * n >= rows) continue;   // none of the sequence's rows
            }
            if (!whole) {
                asm volatile("");   // a branch: most tiles skip it
                if (kTree && tail)
                    sees[n] = see[n] < 0 ? 0u
                                         : tree_bits(a.masks + (size_t)see[n] * a.mask_words, a.mask_words,
                                                     t - s.before());
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = 16 * u + 4 * grp + i;
                        const bool seen = ((there >> u) & 1) && t + p < (kTree ? c1 : min(see[n], c1)) &&
                                          (!kTree || !tail || (sees[kTree ? n : 0] >> p & 1));
                        sc[n][u][i] = seen ? sc[n][u][i] : -INFINITY;
                    }
            }
            float mt = max3(max3(sc[n][0][0], sc[n][0][1], sc[n][0][2]), sc[n][0][3], sc[n][1][0]);
            mt = max3(mt, sc[n][1][1], max3(sc[n][1][2], sc[n][1][3], sc[n][1][3]));
            mt = max32(max16(mt));
            // (rows of a tree in the prompt kernel's way, see there)
            if (__builtin_amdgcn_ballot_w64(kTree ? mt - m_run[n] > kSlackScore<HD> : mt > m_run[n]) != 0) {
                const float m_new = fmaxf(m_run[n], mt);
                const float f = score_factor(m_run[n], m_new, scale_log2);
                m_run[n] = m_new;
                l_run[n] *= f;
#pragma unroll
                for (int d = 0; d < kDims; ++d) o[n][d] *= f;
            }
            const float ref = m_run[n] == -INFINITY ? 0.f : m_run[n];
            float off = 0.f;
            if constexpr (kTree) {
                off = fmaf(-ref, scale_log2, kShift - kSlack);
                if (__builtin_amdgcn_ballot_w64(fabsf(off) > kFar) != 0) {
                    asm volatile("");
                    sc[n][0] -= ref;
                    sc[n][1] -= ref;
                    off = kShift - kSlack;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    pw[n][4 * u + i] = (_Float16)__builtin_amdgcn_exp2f(
                        kTree ? fmaf(sc[n][u][i], scale_log2, off) : fmaf(sc[n][u][i] - ref, scale_log2, kShift));
            l_run[n] = add_weights(pw[n], l_run[n]);
        }
        if (!whole) {   // positions no row may use: their V counts as 0, whatever it holds
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int left = (there >> u) & 1 ? c1 - (t + 16 * u + 4 * grp) : 0;   // of this lane's four
                const uint32_t lo = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
                const uint32_t hi = left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
                xvp[u] &= u32x4{lo, hi, lo, hi};
            }
            // NaN in V: only for the rows that see it
            const uint32_t nan = kv4_hide_nan(xvp[0]) | kv4_hide_nan(xvp[1]) << 4;
            if (__builtin_amdgcn_ballot_w64(nan != 0) != 0) {
                int first = INT_MAX;   // position of the first one in the lane's dims of O, a group
                uint32_t where = 0;    // in a tree, of all of them in the tile
#pragma unroll 1
                for (int g = 0; g < HD / kKv4Group; ++g)
#pragma unroll 1
                    for (int b = 0; b < 8; ++b) {
                        const uint64_t who =
                            __builtin_amdgcn_ballot_w64(col / (512 / HD) == g && ((nan >> b) & 1) != 0);
                        if (who == 0 || (HD == 128 ? grp : grp >> 1) != g) continue;
                        first = min(first, t + 16 * (b / 4) + 4 * (__builtin_ctzll(who) / 16) + b % 4);
                        if (kTree && tail)
                            for (int y = 0; y < 4; ++y)
                                where |= (who >> (16 * y) & 0xffff) != 0 ? 1u << (16 * (b / 4) + 4 * y + b % 4) : 0u;
                    }
#pragma unroll
                for (int n = 0; n < kCols; ++n)
#pragma unroll
                    for (int d = 0; d < kDims; ++d)
                        if (!kTree ? see[n] > first : tail ? (sees[kTree ? n : 0] & where) != 0 : first < INT_MAX)
                            o[n][d] = f32x4{NAN, NAN, NAN, NAN};
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

    // merge the waves, 16 rows at a time
    const bool alone = most <= chunk;
#pragma unroll
    for (int n = 0; n < kCols; ++n) {
        if (16 * n >= rows) break;   // uniform
        if (kCols > 1) __syncthreads();   // Q, or the rows before, are read
        const float l_sum = sum32(sum16(l_run[n]));
        float* to = lds + (wave * 16 + col) * (HD + 4);
        if (grp == 0) {
            to[HD] = m_run[n];
            to[HD + 1] = l_sum;
        }
        // lane (col, grp) has dims kDims (4 grp + i) + d of its column
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int d = 0; d < kDims; d += 4)
                *reinterpret_cast<f32x4*>(to + kDims * (4 * grp + i) + d) =
                    f32x4{o[n][d][i], o[n][d + 1][i], o[n][d + 2][i], o[n][d + 3][i]};
        __syncthreads();
        for (int idx = threadIdx.x; idx < min(rows - 16 * n, 16) * (HD / 4); idx += kBlk) {
            const int r = 16 * n + idx / (HD / 4), d = idx % (HD / 4) * 4, i = r / group;
            const float* from = lds + idx / (HD / 4) * (HD + 4);
            const int step = 16 * (HD + 4);
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) M = fmaxf(M, from[w * step + HD]);
            float l = 0.f;
            f32x4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float m = from[w * step + HD];
                const float f = score_factor(m, M, scale_log2);
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
}

// Log-sum-exp merge of the chunks of one (query, head) by kTeam waves: HD / 4
// lanes read a chunk's sums 16 bytes each, the teams of a wave (and the waves)
// take different chunks, kBatch at once.  The first batch is read before the
// number of chunks is known (all lie in the workspace), so that the kernel is
// one round trip behind the lengths.  Up to 8 chunks (head_dim 64: 16) it takes 3.2
// to 4.7 us by one wave, by four 3.6 to 7.3; 32 chunks of 16 x 32 heads 4.7 by four,
// 6.4 by one.
template <int HD, int kTeam, bool kTree, int kBatch = 4>
__global__ __launch_bounds__(kBlk) void kv4_merge_kernel(Kv4Attention a, int group, int tile_rows, int chunk,
                                                         int n_splits, float scale_log2) {
    constexpr int kLanes = HD / 4, kTeams = kTeam * kWave / kLanes;
    __shared__ __align__(16) float lds[kTeam > 1 ? kTeam : 1][HD];
    const int seq = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int unit = kTeam > 1 ? blockIdx.x : blockIdx.x * kWaves + wave;
    const int i = unit / a.heads, head = unit - i * a.heads;
    if (i >= a.max_query) return;
    const Kv4Seq<kTree> s = kv4_seq<kTree>(a, seq);
    const size_t token = min(s.start + i, a.tokens - 1);   // i may be past the sequence's queries
    const size_t at = (token * a.heads + head) * n_splits;
    const int team = (kTeam > 1 ? wave * (kWave / kLanes) : 0) + lane / kLanes, d = lane % kLanes * 4;
    const float* part = a.workspace + at * HD + d;
    const f32x2* ml = reinterpret_cast<const f32x2*>(a.workspace + (size_t)a.tokens * a.heads * n_splits * HD) + at;
    f32x4 v[kBatch];
    f32x2 w[kBatch];
    auto load = [&](int j0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int j = min(j0 + u * kTeams + team, n_splits - 1);
            v[u] = *reinterpret_cast<const f32x4*>(part + (size_t)j * HD);
            w[u] = ml[j];
        }
    };
    load(0);
    f32x2 mine = ml[min(lane, n_splits - 1)];
    const int asked = min(s.n, a.max_query);
    if (i >= asked) return;
    // the positions that the rows of its workgroups saw
    const int tile = (i * group + head % group) / tile_rows;
    const int most = s.see((int)(min((long long)asked * group, (tile + 1ll) * tile_rows) - 1) / group);
    if (most <= chunk) return;   // written by the chunk itself
    const int n = (most + chunk - 1) / chunk;
    float M = lane < n ? mine.x : -INFINITY;
    for (int j = lane + kWave; j < n; j += kWave) M = fmaxf(M, ml[j].x);
    M = wave_max(M);
    auto factor = [&](float m) { return score_factor(m, M, scale_log2); };
    float l = lane < n ? mine.y * factor(mine.x) : 0.f;
    for (int j = lane + kWave; j < n; j += kWave) l += ml[j].y * factor(ml[j].x);
    l = wave_sum(l);
    f32x4 acc{0.f, 0.f, 0.f, 0.f};
    for (int j0 = 0; j0 < n; j0 += kBatch * kTeams) {
        if (j0 > 0) load(j0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (j0 + u * kTeams + team < n) acc += v[u] * factor(w[u].x);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (kLanes == 16) acc[e] = sum16(acc[e]);
        acc[e] = sum32(acc[e]);
    }
    if constexpr (kTeam > 1) {
        if (lane < kLanes) *reinterpret_cast<f32x4*>(&lds[wave][d]) = acc;
        __syncthreads();
        if (wave != 0) return;
        acc = *reinterpret_cast<const f32x4*>(&lds[0][d]);
#pragma unroll
        for (int o = 1; o < kTeam; ++o) acc += *reinterpret_cast<const f32x4*>(&lds[o][d]);
    }
    if (lane >= kLanes) return;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    u32x2 out;
    out.x = f2h_rne(acc.x * inv) | ((uint32_t)f2h_rne(acc.y * inv) << 16);
    out.y = f2h_rne(acc.z * inv) | ((uint32_t)f2h_rne(acc.w * inv) << 16);
    *reinterpret_cast<u32x2*>(a.out + (size_t)(s.start + i) * a.out_stride + (size_t)head * HD + d) = out;
}

// ---------------------------------------------------------------------------
// Many rows (prompts): one workgroup per (chunk of positions, 128 rows, kv
// head, sequence), 32 rows a wave, tiles of 64 positions.  Bound by the matrix
// products and what goes on beside them:
//  * the workgroup turns a tile's codes into fp16 once, for all its rows: each
//    wave takes 16 positions' K and V (one page), loaded two tiles ahead, into
//    one of two LDS buffers while the other is used; one barrier a tile.  That
//    work is set between the score products, which do not depend on it.
//  * K in LDS as [8 dims][position][8] and V as [16 positions][half][dim][8
//    positions]: the A operands of v_mfma_f32_32x32x16_f16 are 16-byte reads
//    of consecutive lanes, without bank conflicts.
//  * S^T = K Q^T: column = row of Q = lane & 31, so the softmax of a row is one
//    lane's 32 scores and its partner's 32 lanes away, and the weights are the
//    B operand of O^T = V^T P^T as they stand: lane half h has the positions
//    8 a + 4 h + b of 32 (a, b = 0..3), the order V is laid in.
//  * V's dim HD/16 c + n lies at 16 n + c, so that the 16 lanes that write one n
//    use different banks.
//  * the maximum a row's weights refer to moves only when it is exceeded by
//    kSlack (base 2), which spares O its rescaling in most tiles (593 us for the
//    case below against 599 without, six fresh prompts 88 against 91).
//  * kParts = 2: eight waves, four for every other tile, each with buffers of
//    their own; the second four's sums join the first's at the end.  For grids
//    that leave a CU one workgroup, whose waves would wait for their own reads.
// 2048 queries behind 14336 positions, 32/8 heads of 128 (515 GFLOP): 573 to
// 578 us, 893 TFLOP/s (a large fp16 product: 1162), the matrix units busy for 36%
// of it and the vector units for 46%; of 631 us of an early form the products
// alone took 330, and 256 rows by eight waves as long as 128 by four.
// Four trees of 190 to 300 rows behind 22452 .. 32000 positions, 40/8 heads (115 GFLOP):
// 181 to 200 us, 570 to 630 TFLOP/s, with 78% of the row tiles' rows filled.
// ---------------------------------------------------------------------------
constexpr int kRowTile = 128, kTile = 64;   // rows of a workgroup; positions of a step
// A row tile of a tree that has no more rows (kPairs): a wave has half of the positions of
// a step for 32 of them, and the halves join at the end (heads of 128: 25 sequences of 32
// to 64 rows behind 150 to 2500 positions 44.3 -> 39.2 us, 64 behind 200 to 2000 75.8 ->
// 63.9, 25 of 80 to 160 rows 83.5 -> 69.3; in tiles of 64 throughout, 300 rows take 255 us
// for 200: the codes' way to fp16 is half of a step).
constexpr int kPairRows = 64;
constexpr int kPromptNotes = 10 * kWaves;   // words that a part's waves leave one another
typedef float f32x16 __attribute__((ext_vector_type(16)));

// Rows row0 .. of sequence seq's `rows`, against its positions c0 .. c1 - 1 (of `most`).
template <int HD, int kParts, bool kTree, bool kPairs>
__device__ __forceinline__ void kv4_prompt_tile(const Kv4View& c, const Kv4Attention& a, int chunk, int n_splits,
                                                float scale_log2, const Kv4Seq<kTree>& s, int seq, int kvh, int group,
                                                int split, int rows, int row0, int most, int c0, int c1) {
    using L = Kv4Layout<HD>;
    using Vec = std::conditional_t<HD == 128, u32x4, u32x2>;
    constexpr int kHalf = kPairs ? 1 : 2;              // a wave's positions of a step, by 32
    constexpr int kWords = HD / 32;                    // words of codes a thread has of a position (K) or of 4 (V)
    constexpr int kHalves = HD * kTile;                // of K (or V) in a buffer
    extern __shared__ __align__(16) float lds[];
    const int part = kParts == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / kBlk);
    uint16_t* const buf = reinterpret_cast<uint16_t*>(lds) + part * 4 * kHalves;   // [2][K, V][kHalves]
    // [2][4 waves]: bit 0, the 16 positions have a page; bit 1, nan_at says where V is
    // NaN first (in a tree: at which of the 16)
    int* const notes = reinterpret_cast<int*>(reinterpret_cast<uint16_t*>(lds) + kParts * 4 * kHalves);
    int* const there_at = notes + part * kPromptNotes;
    int* const nan_at = there_at + 2 * kWaves;                           // [2][4 waves][4 groups of dims]
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) % kWaves;   // of the part
    const int col = lane & 31, half = lane >> 5;

    // this lane's row of Q
    const int row1 = row0 + 32 * (kPairs ? wave & 1 : wave), u0 = kPairs ? wave >> 1 : 0;   // the wave's, of both
    const int r = row1 + col;
    const bool real = r < rows;
    const int i = real ? r / group : 0;
    const size_t head = (size_t)kvh * group + (real ? r - i * group : 0);
    const int see = real ? min(s.see(i), c1) : 0;
    half8 q[HD / 16];
    {
        const uint16_t* qr = a.q + (size_t)(s.start + i) * a.q_stride + head * HD + 8 * half;
#pragma unroll
        for (int t = 0; t < HD / 16; ++t) {
            u32x4 v = *reinterpret_cast<const u32x4*>(qr + 16 * t);
            if (!real) v = u32x4{0u, 0u, 0u, 0u};
            q[t] = __builtin_bit_cast(half8, v);
        }
    }
    // positions that every / any row of the wave sees
    const int r_last = min(rows - 1, row1 + 31);
    const int wave_least = r_last < row1 + 31 ? 0 : min(s.all((row1) / group), c1);
    const int wave_most = row1 >= rows ? 0 : min(s.see(r_last / group), c1);

    const int least = min(s.all(row0 / group), c1);   // positions that every row of the workgroup sees

    // ---- the wave's 16 positions of a tile: pages, loads, dequantisation ----
    const int P = 1 << c.page_shift;
    const int last_page = (max(c1, 1) - 1) >> c.page_shift;
    const int32_t* table = a.page_table + (size_t)seq * a.pages_per_seq;
    int window = c0 >> c.page_shift;   // lane j has page window + j of the table, then of the 64 after them
    auto pages_from = [&](int first) { return table[min(first + lane, last_page)]; };
    int pages = pages_from(window), pages_next = pages_from(window + kWave);
    const int t16 = lane & 15, g = lane >> 4;            // K: position, quarter of the dims
    const int vb = ((g & 1) << 1) | (g >> 1);            // V: block of 4 positions, dims HD/16 t16 ..
    Vec xk, xv;
    uint32_t xkp;
    u32x4 xvp;
    const uint32_t at_k = t16 * L::kCodes + g * (HD / 8), at_kp = t16 * L::kParams + (HD == 128 ? g : g >> 1) * 4;
    const uint32_t at_v = vb * (4 * L::kCodes) + t16 * (HD / 8), at_vp = vb * (4 * L::kParams) + t16 / (512 / HD) * 16;
    int x_there = 0, x_nan = 0, x_pos = 0;
    auto load = [&](int t) {
        const int p = t + 16 * wave, at = min(p >> c.page_shift, last_page);
        if (at >= window + kWave) {   // uniform
            window += kWave;
            pages = pages_next;
            pages_next = pages_from(window + kWave);
        }
        const int page = __builtin_amdgcn_readlane(pages, at - window);
        x_there = p < c1 && page >= 0 && page < c.num_pages;
        x_pos = p;
        const uint8_t* base = kv4_head<HD>(c, x_there ? page : 0, kvh);
        const int o = p & (P - 1);
        xk = *reinterpret_cast<const Vec*>(base + o * L::kCodes + at_k);
        xkp = *reinterpret_cast<const uint32_t*>(base + L::k_params(P) + o * L::kParams + at_kp);
        xv = *reinterpret_cast<const Vec*>(base + L::v_codes(P) + o * L::kCodes + at_v);
        xvp = *reinterpret_cast<const u32x4*>(base + L::v_params(P) + o * L::kParams + at_vp);
    };
    // Before store(b): V of positions that no row, or not every row, sees.
    auto hide = [&](int b) {
        x_nan = 0;
        if (x_there && x_pos + 16 <= least) return;   // uniform
        // positions past the chunk or without a page: V counts as 0, whatever it holds
        const int left = x_there ? c1 - (x_pos + 4 * vb) : 0;
        const uint32_t lo = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
        const uint32_t hi = left >= 4 ? 0xffffffffu : left == 3 ? 0xffffu : 0u;
        xvp &= u32x4{lo, hi, lo, hi};
        const uint32_t nan = kv4_hide_nan(xvp);
        if (__builtin_amdgcn_ballot_w64(nan != 0) == 0) return;
        x_nan = 2;
#pragma unroll 1
        for (int dims = 0; dims < HD / kKv4Group; ++dims) {
            int first = nan != 0 && t16 / (512 / HD) == dims ? x_pos + 4 * vb + __builtin_ctz(nan) : INT_MAX;
            if constexpr (kTree) first = t16 / (512 / HD) == dims ? (int)(nan << 4 * vb) : 0;
            for (int d = 1; d < kWave; d <<= 1) {
                const int other = __shfl_xor(first, d, kWave);
                first = kTree ? first | other : min(first, other);
            }
            if (lane == 0) nan_at[(b * kWaves + wave) * 4 + dims] = first;
        }
    };
    auto store = [&](int b) {
        uint16_t* kb = buf + b * 2 * kHalves;
        uint16_t* vbuf = kb + kHalves;
        const f16x2 dm = as_h2(xkp);
        const f16x2 d{dm.x, dm.x}, m{dm.y, dm.y};
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            f16x2 e[4];
            kv4_pairs(xk[w], d, m, e);
            *reinterpret_cast<half8*>(kb + ((g * kWords + w) * kTile + 16 * wave + t16) * 8) =
                __builtin_bit_cast(half8, e);
        }
#pragma unroll
        for (int h = 0; h < kWords / 2; ++h) {
            f16x2 e[2][4];
#pragma unroll
            for (int y = 0; y < 2; ++y)
                kv4_pairs(xv[2 * h + y], as_h2(xvp[y]), as_h2(xvp[2 + y]), e[y]);
#pragma unroll
            for (int n = 0; n < 4; ++n)
                *reinterpret_cast<u32x2*>(vbuf + (((2 * wave + (vb & 1)) * HD) + (4 * h + n) * 16 + t16) * 8 +
                                          (vb >> 1) * 4) =
                    u32x2{__builtin_bit_cast(uint32_t, e[0][n]), __builtin_bit_cast(uint32_t, e[1][n])};
        }
        if (lane == 0) there_at[b * kWaves + wave] = x_there | x_nan;
    };

    f32x16 o[HD / 32];
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    // kTail: of a tree, positions of its rows among the tile's
    auto process = [&](int t, int b, auto kTail) __attribute__((always_inline)) {
        hide(b ^ 1);
        if (t + 32 * u0 >= wave_most) {   // uniform: no row of the wave sees the tile
            store(b ^ 1);
            return;
        }
        const uint16_t* kb = buf + b * 2 * kHalves;
        const uint16_t* vbuf = kb + kHalves;
        int there = 0;   // two bits a wave
#pragma unroll
        for (int w = 0; w < kWaves; ++w) there |= there_at[b * kWaves + w] << (2 * w);
        there = __builtin_amdgcn_readfirstlane(there);
        constexpr int kThere = kPairs ? 0xf : 0xff;   // bits of the wave's positions
        there = there >> 4 * u0 & kThere;
        const bool whole = (there & 0x55) == (0x55 & kThere) && t + 32 * (u0 + kHalf) <= wave_least;
        __builtin_amdgcn_sched_barrier(0);
        f32x16 sc[kHalf];
#pragma unroll
        for (int u = 0; u < kHalf; ++u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[u][e] = 0.f;
#pragma unroll
            for (int st = 0; st < HD / 16; ++st) {
                const half8 k =
                    *reinterpret_cast<const half8*>(kb + ((2 * st + half) * kTile + 32 * (u0 + u) + col) * 8);
                sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[st], sc[u], 0, 0, 0);
            }
        }
        store(b ^ 1);   // the next tile's codes beside this one's products
#pragma unroll
        // an LDS read, a product, 8 vector instructions and a write at a time (kPairs: twice the last two)
        for (int n = 0; n < kHalf * HD / 16; ++n) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 16 / kHalf, 0);
            __builtin_amdgcn_sched_group_barrier(0x200, 2 / kHalf, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        uint32_t sees[kTail ? kHalf : 1];   // of a tree's row, the wave's positions
        if (!whole) {
            if constexpr (kTail) {
                const uint32_t* row = a.masks + (size_t)(s.start + i) * a.mask_words;
#pragma unroll
                for (int u = 0; u < kHalf; ++u)
                    sees[u] = real ? tree_bits(row, a.mask_words, t + 32 * (u0 + u) - s.before()) : 0u;
            }
#pragma unroll
            for (int u = 0; u < kHalf; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int p = 32 * u + 8 * (e / 4) + 4 * half + e % 4;
                    const bool seen = t + 32 * u0 + p < see && ((there >> (p >> 4) * 2) & 1) &&
                                      (!kTail || (sees[kTail ? u : 0] >> (p & 31) & 1));
                    sc[u][e] = seen ? sc[u][e] : -INFINITY;
                }
        }
        if ((there & 0xaa) != 0) {   // NaN in V: only for the rows that see it
#pragma unroll
            for (int y = 0; y < 2; ++y) {   // elements e with e / 4 % 2 = y are of one group of dims
                int first = INT_MAX;
                bool meets = false;   // in a tree: the row sees one of them
#pragma unroll 1
                for (int w = 0; w < 2 * kHalf; ++w)
                    if ((there >> (2 * w)) & 2) {
                        const int at = nan_at[(b * kWaves + 2 * u0 + w) * 4 + (HD == 128 ? 2 * y + half : y)];
                        if constexpr (kTail)
                            meets |= ((w < 2 ? sees[0] : sees[kHalf - 1]) >> (16 * (w & 1)) & (uint32_t)at) != 0;
                        else if constexpr (kTree)
                            meets |= at != 0;
                        else
                            first = min(first, at);
                    }
#pragma unroll
                for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (e / 4 % 2 == y) o[d][e] = (kTree ? meets : see > first) ? NAN : o[d][e];
            }
        }
        float mt = -INFINITY;
#pragma unroll
        for (int u = 0; u < kHalf; ++u)
#pragma unroll
            for (int e = 0; e < 16; e += 2) mt = max3(mt, sc[u][e], sc[u][e + 1]);
        mt = max32(mt);
        if (__builtin_amdgcn_ballot_w64(mt - m_run > kSlackScore<HD>) != 0) {
            const float m_new = fmaxf(m_run, mt);
            const float f = score_factor(m_run, m_new, scale_log2);
            m_run = m_new;
            l_run *= f;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) o[d] *= f;
        }
        // A weight is 2^((score - ref) scale + shift), here as one fma with off =
        // shift - ref scale (with the difference first, as few rows take it: 603 us
        // for 584).  Beyond kFar the rounding of off would count, 2^-15 of a weight
        // there; those tiles take the difference first.
        const float ref = m_run == -INFINITY ? 0.f : m_run;
        float off = fmaf(-ref, scale_log2, kShift - kSlack);
        if (__builtin_amdgcn_ballot_w64(fabsf(off) > kFar) != 0) {
            asm volatile("");   // a branch: most tiles skip it
#pragma unroll
            for (int u = 0; u < kHalf; ++u) sc[u] -= ref;
            off = kShift - kSlack;
        }
        half8 pw[2 * kHalf];
#pragma unroll
        for (int u = 0; u < kHalf; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                pw[2 * u + e / 8][e % 8] = (_Float16)__builtin_amdgcn_exp2f(fmaf(sc[u][e], scale_log2, off));
#pragma unroll
        for (int st = 0; st < 2 * kHalf; ++st) l_run = add_weights(pw[st], l_run);
#pragma unroll
        for (int st = 0; st < 2 * kHalf; ++st)
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                const half8 v = *reinterpret_cast<const half8*>(
                    vbuf + ((2 * (2 * u0 + st) + half) * HD + 32 * d + col) * 8);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pw[st], o[d], 0, 0, 0);
            }
    };

    constexpr int kTurn = kParts * kTile;
    const int mine = part * kTile;
    load(c0 + mine);
    hide(0);
    store(0);
    load(c0 + mine + kTurn);
    __syncthreads();
    int t = c0, b = 0;
    auto turn = [&](auto kTail) __attribute__((always_inline)) {
        process(t + mine, b, kTail);
        load(t + mine + 2 * kTurn);
        __syncthreads();
        t += kTurn;
        b ^= 1;
    };
    if constexpr (kTree)
        while (t < c1 && t + kTurn <= s.before()) turn(std::false_type{});
    while (t < c1) turn(std::bool_constant<kTree>{});

    // ---- out: O^T's rows back in dim order through LDS, a wave's rows at a time ----
    float l = sum32(l_run);
    // another wave's sums, lane by lane through LDS, join this one's
    auto give = [&](float* sums, float* ml) {
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) sums[(16 * d + e) * kWave] = o[d][e];
        ml[0] = m_run;
        ml[1] = l;
    };
    auto take = [&](const float* sums, const float* ml) {
        const float m = fmaxf(m_run, ml[0]);
        const float f0 = score_factor(m_run, m, scale_log2), f1 = score_factor(ml[0], m, scale_log2);
        m_run = m;
        l = l * f0 + ml[1] * f1;
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = o[d][e] * f0 + sums[(16 * d + e) * kWave] * f1;
    };
    if constexpr (kParts == 2) {   // the second part's, through its own buffers
        float* const sums = lds + 2 * kHalves + wave * (HD / 2) * kWave + lane;
        float* const ml = reinterpret_cast<float*>(notes + 2 * kPromptNotes) + 2 * (wave * kWave + lane);
        if (part == 1) give(sums, ml);
        __syncthreads();
        if (part == 1) return;
        take(sums, ml);
    }
    constexpr int kPitch = HD + 8;
    if constexpr (kPairs) {   // the second half of the positions', behind the rows' buffers below
        float* const sums = lds + 32 * kPitch + (wave & 1) * (HD / 2) * kWave + lane;
        float* const ml = lds + 32 * kPitch + HD * kWave + 2 * ((wave & 1) * kWave + lane);
        static_assert((32 * kPitch + HD * kWave + 4 * kWave) * 4 <= 4 * kHalves * 2);
        if (u0 == 1) give(sums, ml);
        __syncthreads();
        if (u0 == 1) return;
        take(sums, ml);
    }
    const bool alone = most <= chunk;
    if (alone) {
        uint16_t* rowbuf = buf + wave * 32 * kPitch;
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int slot = 32 * d + 8 * (e / 4) + 4 * half + e % 4;
                rowbuf[col * kPitch + slot % 16 * (HD / 16) + slot / 16] = f2h_rne(o[d][e] * inv);
            }
        wave_lds_sync();
        for (int idx = lane; idx < 32 * (HD / 8); idx += kWave) {
            const int rr = idx / (HD / 8), r1 = row1 + rr, piece = idx % (HD / 8);
            if (r1 >= rows) break;
            const int i1 = r1 / group;
            *reinterpret_cast<u32x4*>(a.out + (size_t)(s.start + i1) * a.out_stride +
                                      ((size_t)kvh * group + (r1 - i1 * group)) * HD + 8 * piece) =
                *reinterpret_cast<const u32x4*>(rowbuf + rr * kPitch + 8 * piece);
        }
        return;
    }
    if (!real) return;
    const size_t at = ((size_t)(s.start + i) * a.heads + head) * n_splits + split;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int slot = 32 * d + 8 * (e / 4) + 4 * half + e % 4;
            a.workspace[at * HD + slot % 16 * (HD / 16) + slot / 16] = o[d][e];
        }
    if (half == 0) {
        float* ml = a.workspace + (size_t)a.tokens * a.heads * n_splits * HD + 2 * at;
        ml[0] = m_run;
        ml[1] = l;
    }
}

template <int HD, int kParts, bool kTree>
__global__ __launch_bounds__(kParts * kBlk, 2) void kv4_prompt_kernel(Kv4View c, Kv4Attention a, int chunk,
                                                                      int n_splits, float scale_log2) {
    // kv heads side by side, so that the workgroups of one meet in an XCD's L2
    // where there are eight of them; row tiles with the most positions first,
    // every sequence's before the next tile (6 prompts of 100 .. 2500 tokens:
    // 88 us against 85 with one sequence's tiles after another's, but 29.5 against
    // 35.1 for two of 761, 43 against 50 for three pieces of 636 behind a prefix)
    const int kvh = blockIdx.x % c.kv_heads;
    const int group = a.heads / c.kv_heads, tiles = (a.max_query * group + kRowTile - 1) / kRowTile;
    const int rest = blockIdx.z * gridDim.y + blockIdx.y;
    const int seq = seq_of(blockIdx.x / c.kv_heads, rest, a.nseq);
    const Kv4Seq<kTree> s = kv4_seq<kTree>(a, seq);
    int split, tile;
    if constexpr (kTree) {   // every sequence's last chunk, the short one, last (kTreeBlocks' case: 304 -> 207 us)
        tile = rest % tiles;
        split = rest / tiles - (n_splits - kv4_chunks(s, chunk));
        if (split < 0) return;
    } else {
        split = rest % n_splits;
        tile = tiles - 1 - rest / n_splits;
    }
    const int rows = min(s.n, a.max_query) * group, row0 = tile * kRowTile;
    if (tile < 0 || row0 >= rows) return;
    const int most = max(0, s.see((min(rows, row0 + kRowTile) - 1) / group));
    const int c0 = split * chunk, c1 = min(most, c0 + chunk);
    if (c0 >= most && split > 0) return;
    auto go = [&](auto pairs) __attribute__((always_inline)) {
        kv4_prompt_tile<HD, kParts, kTree, pairs>(c, a, chunk, n_splits, scale_log2, s, seq, kvh, group, split, rows,
                                                  row0, most, c0, c1);
    };
    if constexpr (kTree)
        if (rows - row0 <= kPairRows) return go(std::true_type{});
    go(std::false_type{});
}

// us below: 8 kv heads, head_dim 128, wall clock per call.
// Which kernel: the few-row kernel up to 48 rows, where it beats the prompt
// kernel from about 300 positions on and does not lose before (16 sequences of
// 2000 / 6000 positions, few-row against prompt kernel: 32 rows 24 / 39 against
// 30 / 59, 40 rows 26 / 54 against 32 / 67; built for 64 rows 37 / 82 against
// 33 / 68).
constexpr int kFewRows = 48;
// Trees with heads of 64 go up to 80 rows: few-row against prompt kernel, calls of 8 kv
// heads, with up to 50, 66 and 80 rows of 2 heads: 25 sequences of 176 to 2500
// positions 26.6 / 30.7, 34.9 / 36.9, 34.5 / 36.8; 100 of 150 to 1500 50.6 / 60.8, 60.6 /
// 60.5, 68.2 / 74.8; one of 16000 17.4 / 18.4, 19.4 / 19.4, 19.8 / 19.9; but 64 of 200 to 2000 47.4 /
// 47.1, 52.8 / 49.9, 59.8 / 57.9, and 8 of them 17.2 / 17.4, 20.3 / 19.3, 20.9 / 20.3: up
// to 17% less, 6% more where the grid falls badly.
// Heads of 128 spill at 64 rows: 34 us for 21 with one sequence, 108 for 80 with 64.
constexpr int kFewTreeRows64 = 80;
constexpr int few_rows(bool tree, int head_dim) { return tree && head_dim == 64 ? kFewTreeRows64 : kFewRows; }
// Its chunks: whole turns of the four waves, as long as leaves one round of
// resident workgroups (four, three or two per CU for 16, 32 or 48 rows), at
// most 1024 positions (a lane per page) and at least 256 (16 sequences of 2000
// positions, 15 rows: chunks of 128 16.3, 256 13.6, 512 13.3).  Short contexts
// stay in one chunk, without a merge (64 sequences of 4 rows: 512 positions
// 12.1 against 20.9 in chunks, 768 15.3 against 23.7; one sequence of 42 rows and
// 512 positions 14.1 against 13.0, 768 17.4 against 13.5).
constexpr int kChunkStep = 32 * kWaves, kChunkLeast = 256, kChunkMost = 1024, kFewBlocks = 1024;
constexpr int kAlone = 768, kAloneWide = 512;   // positions of one chunk, up to 16 rows and above
// The prompt kernel splits the positions only where its row tiles leave CUs
// without work: chunks of 192 on up to one workgroup per CU, of 512 up to two
// (64 rows of 600 positions 15.2, 21.2 with 512 alone; 4 sequences of 64 rows and
// 1000 positions 16.3, 33.0; 2 prompts of 500 x 4 rows behind 500 positions, which
// fill the CUs, 34.9, and 46.3 with 192 up to two).
constexpr int kPromptBlocks = 256, kPromptChunk = 192, kPromptChunkFull = 512;
// Two parts up to 384 workgroups, one and a half per CU, that take all of more than
// 256 positions (one prompt of 32/8 heads: 1100 tokens, 280 workgroups, 33.8
// against 40.8 with one part, 1500, 376, 44.0 against 53.4, 2048, 512, 59.6
// against 62.7; but two of 1024, 512, 40.7 against 39.1, four of 700, 704, 43.5
// against 36.3, 288 workgroups of half of 1390 positions 54.6 against 48.5, 312 of
// 44 positions 11.7 against 9.4).
constexpr int kTwoPartBlocks = 384, kTwoPartContext = 256;
// Trees have few rows behind contexts of any length: the prompt kernel's grid is cut
// finer than a prompt's, into about kTreeBlocks workgroups were all contexts the
// longest (four sequences of 38 to 60 rows of 5 heads behind 22452 to 32000 positions:
// kernel and merge 208 us, cut for one round of workgroups 263, into 1280 229; 25 of up
// to 64 rows of heads of 128 behind 150 to 2500 39.5, into 1024 45).  The merge takes one
// wave a head from kMergeUnits heads on (180 rows of 40 heads in 15 parts: 12.1 us, by
// four waves 18.5).
constexpr int kTreeBlocks = 700, kMergeUnits = 2048;
// Trees that one workgroup per CU serves have eight waves in each, so that a chunk takes
// half the turns (32/8 heads, with four waves and with eight: 4 sequences of 8000
// positions and 16 rows 20.1 and 15.7 us, 32 rows 29.0 and 18.8, 48 29.7 and 22.6; 16 of
// 1000 with 32 19.0 and 15.5; one of 1000 with 16 10.6 and 10.2.  Two such workgroups
// per CU: 16 of 2000 with 48 rows 31.6, 26.6 with four waves).
constexpr int kWideWaves = 8, kWideBlocks = 256;
struct Kv4Plan {
    bool few;
    int cols, tiles, chunk, n_splits, waves;   // waves: of a workgroup with few rows
};
Kv4Plan kv4_plan(bool tree, int max_context, int max_query, int nseq, int heads, int kv_heads, int head_dim) {
    Kv4Plan p{};
    const long long rows = (long long)max_query * (heads / kv_heads);
    p.few = rows <= few_rows(tree, head_dim);
    p.cols = p.few ? (int)(rows + 15) / 16 : 0;
    p.tiles = (int)((rows + kRowTile - 1) / kRowTile);
    auto whole = [](long long positions, int step) { return (int)((positions + step - 1) / step * step); };
    if (p.few) {
        // (a tree's columns without rows cost little, so its grid counts on three per CU
        // with heads of 64: 25 of 48 rows and 2500 positions 28.2 us, on two 31.7)
        const int blocks = p.cols == 1                               ? kFewBlocks
                           : p.cols == 2 || (tree && head_dim == 64) ? kFewBlocks * 3 / 4
                                                                     : kFewBlocks / 2;
        const long long share = ((long long)max_context * nseq * kv_heads + blocks - 1) / blocks;
        p.chunk = max_context <= (p.cols == 1 || p.cols > 3 ? kAlone : kAloneWide)
                      ? whole(max_context, kChunkStep)
                      : whole(std::max<long long>(kChunkLeast, std::min<long long>(kChunkMost, share)), kChunkStep);
    } else {
        const long long blocks = (long long)p.tiles * kv_heads * nseq;
        auto least = [&](long long most, int chunk) { return std::min<long long>(most / blocks, max_context / chunk); };
        const long long splits =
            tree ? std::max(1ll, least(kTreeBlocks, kPromptChunk))
                 : std::max({1ll, least(kPromptBlocks, kPromptChunk), least(2 * kPromptBlocks, kPromptChunkFull)});
        p.chunk = whole((max_context + splits - 1) / splits, kTile);
    }
    p.waves = kWaves;
    const long long units = (long long)kv_heads * nseq;
    if (tree && p.few && units * ((max_context + kChunkMost - 1) / kChunkMost) <= kWideBlocks) {
        p.waves = kWideWaves;
        const int step = 32 * kWideWaves;
        const long long share = (max_context * units + kWideBlocks - 1) / kWideBlocks;
        const bool alone = max_context <= kAloneWide || (max_context <= kChunkMost && share > kChunkLeast);
        p.chunk = whole(alone ? max_context : std::max<long long>(kChunkLeast, std::min<long long>(kChunkMost, share)),
                        step);
    }
    p.n_splits = (max_context + p.chunk - 1) / p.chunk;
    return p;
}

template <int HD, bool kTree>
hipError_t launch_for(const Kv4View& c, const Kv4Attention& a, hipStream_t s) {
    const Kv4Plan p = kv4_plan(kTree, a.max_context, a.max_query, a.nseq, a.heads, c.kv_heads, HD);
    const float scale_log2 = 1.44269504088896340736f / sqrtf((float)HD);
    const int group = a.heads / c.kv_heads;
    const bool last = p.n_splits == 1;
    if (!p.few) {
        const int units = p.tiles * p.n_splits, y = std::min(units, 32768);   // at most 65535 in y
        const dim3 grid(c.kv_heads * a.nseq, y, (units + y - 1) / y);
        const int part = 4 * HD * kTile * (int)sizeof(uint16_t) + kPromptNotes * (int)sizeof(int);
        const bool two = last && a.max_context > kTwoPartContext &&
                         (long long)units * c.kv_heads * a.nseq <= kTwoPartBlocks;
        const int lds = two ? 2 * part + 2 * kBlk * (int)sizeof(float) : part;
        auto with = [&](auto parts) {
            constexpr auto kernel = kv4_prompt_kernel<HD, parts, kTree>;
            const hipError_t e = allow_lds<kernel>(lds);
            if (e == hipSuccess)
                launch_kernel_in_call(last, kernel, grid, dim3(parts * kBlk), lds, s, c, a, p.chunk, p.n_splits,
                                      scale_log2);
            return e;
        };
        const hipError_t e = two ? with(std::integral_constant<int, 2>{}) : with(std::integral_constant<int, 1>{});
        if (e != hipSuccess) return e;
    } else {
        const dim3 grid(c.kv_heads * a.nseq, p.n_splits);
        const int lds = p.waves * 16 * (HD + 4) * (int)sizeof(float);   // the merge; Q takes less
        static_assert(few_rows(kTree, HD) * HD * 2 <= kWaves * 16 * (HD + 4) * 4);
        auto go = [&](auto kernel, int waves) {
            launch_kernel_in_call(last, kernel, grid, dim3(waves * kWave), lds, s, c, a, p.chunk, p.n_splits,
                                  scale_log2);
        };
        auto with = [&](auto cols) {
            if constexpr (16 * cols - 15 > few_rows(kTree, HD)) {
                return hipErrorInvalidValue;   // (no plan has them)
            } else {
                if constexpr (kTree) {
                    if (p.waves == kWideWaves) {
                        constexpr auto kernel = kv4_decode_kernel<HD, cols, true, kWideWaves>;
                        const hipError_t e = allow_lds<kernel>(lds);
                        if (e == hipSuccess) go(kernel, kWideWaves);
                        return e;
                    }
                }
                go(kv4_decode_kernel<HD, cols, kTree>, kWaves);
                return hipSuccess;
            }
        };
        const hipError_t e = p.cols == 1   ? with(std::integral_constant<int, 1>{})
                             : p.cols == 2 ? with(std::integral_constant<int, 2>{})
                             : p.cols == 3 ? with(std::integral_constant<int, 3>{})
                             : p.cols == 4 ? with(std::integral_constant<int, 4>{})
                                           : with(std::integral_constant<int, 5>{});
        if (e != hipSuccess) return e;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || last) return e;
    const long long units = (long long)a.max_query * a.heads;
    const int tile_rows = p.few ? few_rows(kTree, HD) : kRowTile;
    const dim3 one((unsigned)((units + kWaves - 1) / kWaves), a.nseq);   // a wave a head
    auto merge = [&](auto kernel, dim3 grid) {
        launch_kernel(kernel, grid, dim3(kBlk), 0, s, a, group, tile_rows, p.chunk, p.n_splits, scale_log2);
        return hipGetLastError();
    };
    // one wave covers 4 chunks a lane group at once; with more of them four waves share a head
    if constexpr (kTree) {   // of few chunks, 2: none is read twice (48 x 384 heads of 4 chunks 9.6 -> 8.1 us)
        if (p.n_splits <= 2 * kWave / (HD / 4)) return merge(kv4_merge_kernel<HD, 1, true, 2>, one);
    }
    if (p.n_splits <= 4 * kWave / (HD / 4) || (kTree && units * a.nseq > kMergeUnits))
        return merge(kv4_merge_kernel<HD, 1, kTree>, one);
    return merge(kv4_merge_kernel<HD, kWaves, kTree>, dim3((unsigned)units, a.nseq));
}

}  // namespace

size_t kv4_attention_workspace(bool tree, int max_context, int max_query, int nseq, int tokens, int heads,
                               int kv_heads, int head_dim) {
    const Kv4Plan p = kv4_plan(tree, max_context, max_query, nseq, heads, kv_heads, head_dim);
    if (p.n_splits == 1) return 0;
    return (size_t)tokens * heads * p.n_splits * (head_dim + 2) * sizeof(float);
}

hipError_t launch_kv4_attention(const Kv4View& c, const Kv4Attention& a, hipStream_t s) {
    if (a.masks) return c.head_dim == 128 ? launch_for<128, true>(c, a, s) : launch_for<64, true>(c, a, s);
    return c.head_dim == 128 ? launch_for<128, false>(c, a, s) : launch_for<64, false>(c, a, s);
}

}  // namespace citlali::hip
