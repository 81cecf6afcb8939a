// logprobs.hip -- log probability and rank of a given token, entropy and the
// most likely tokens of each row of logits, in one pass over them.
//
// With m a row's maximum, s = sum e^(x - m) and t = sum e^(x - m) (x - m):
//   log p(x) = x - m - log s        H = log s - t / s
// Every lane keeps (m, s, t) of its own logits, 16 at a time: the maximum
// first, then one rescaling, then their exponentials, added in pairs.  A row is
// cut into pieces of whole waves; lanes, waves and workgroups join by
//   (m, s, t) + (m', s', t'):  s f + s' f',  f (t + s (m - M)) + ...,  f = e^(m - M).
//
// The most likely tokens are kept as 64-bit keys (ordered bits of the logit,
// then the complement of the id, so that equal logits go by the lower id):
// lane i of a wave has the wave's i-th largest.  Logits below the k-th cost one
// comparison per 16; those above it are gathered in LDS, and 64 of them are
// sorted across the lanes and merged at a time.  The order is total, so the
// result does not depend on the cut.
//
// Bound by reading the logits; beside them a wave issues about 11 instructions
// per 64 logits, one of them the exponential.
#include "device_common.hpp"
#include "launch.hpp"

#include <limits.h>
#include <math.h>

#include <algorithm>

namespace citlali::hip {
namespace {

constexpr int kBlk = 256, kWaves = kBlk / kWave;
constexpr int kPer = 16;                    // logits of a lane in a step
constexpr int kStep = kPer * kWave;         // of a wave
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// Larger logit first, then the lower id; 0 is a NaN, before nothing.  -0.0
// counts as +0.0.
__device__ __forceinline__ uint64_t logit_key(float x, int id) {
    if (x != x) return 0ull;
    const uint32_t u = __float_as_uint(x + 0.f);
    return ((uint64_t)(u ^ (uint32_t)((int32_t)u >> 31 | 0x80000000)) << 32) | (uint32_t)~(uint32_t)id;
}
__device__ __forceinline__ float key_logit(uint64_t k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// ---- a wave's largest keys --------------------------------------------------
// Larger of a lane's and its partner's key where `up`, else the smaller.
__device__ __forceinline__ uint64_t exchange(uint64_t v, int stride, bool up) {
    const uint64_t w = __shfl_xor((unsigned long long)v, stride, kWave);
    return (v > w) == up ? v : w;
}
__device__ __forceinline__ uint64_t sort_descending(uint64_t v, int lane) {
#pragma unroll
    for (int size = 2; size <= kWave; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1)
            v = exchange(v, stride, ((lane & stride) == 0) == ((lane & size) == 0 || size == kWave));
    return v;
}
// The 64 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t merge_descending(uint64_t a, uint64_t b, int lane) {
    const uint64_t w = __shfl((unsigned long long)b, kWave - 1 - lane, kWave);
    uint64_t v = a > w ? a : w;
#pragma unroll
    for (int stride = kWave >> 1; stride > 0; stride >>= 1) v = exchange(v, stride, (lane & stride) == 0);
    return v;
}
__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return ((uint64_t)hi << 32) | lo;
}

struct TopKeys {
    uint64_t mine = 0;    // lane i: the i-th largest
    uint64_t floor = 0;   // only keys above it can be among the k largest (uniform)
    int waiting = 0;      // keys in `room` (uniform)
    uint64_t* room;       // 64 of LDS, the wave's own
    int lane, k;

    __device__ void flush() {
        wave_lds_sync();
        const uint64_t v = lane < waiting ? room[lane] : 0ull;
        wave_lds_sync();
        mine = merge_descending(mine, sort_descending(v, lane), lane);
        const uint64_t kth = lane_key(mine, k - 1);
        floor = kth > floor ? kth : floor;
        waiting = 0;
    }
    __device__ void add(uint64_t key) {
        uint64_t who = __builtin_amdgcn_ballot_w64(key > floor);
        if (who == 0) return;
        if (waiting + __popcll(who) > kWave) {
            flush();
            who = __builtin_amdgcn_ballot_w64(key > floor);
        }
        if (key > floor)
            room[waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] =
                key;
        waiting += __popcll(who);
    }
    // Before many keys at once, of which `best` are the lanes' largest: at
    // least k of them reach the k-th largest of those.
    __device__ void raise(uint64_t best) {
        const uint64_t kth = lane_key(sort_descending(best, lane), k - 1);
        if (kth > floor) floor = kth - 1;
    }
};

// ---- sums --------------------------------------------------------------------
struct Sums {
    float m, s, t;   // t in base 2: sum e^(x - m) log2(e) (x - m)
};
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float M = fmaxf(a.m, b.m);
    // a side without a logit above -inf has s and t 0 (or NaN, which stays)
    const float da = a.m == -INFINITY ? 0.f : (a.m - M) * kLog2e, db = b.m == -INFINITY ? 0.f : (b.m - M) * kLog2e;
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    // a factor of 0 takes its side's terms with it (its distance may be infinite)
    const float ta = fa == 0.f ? 0.f * a.s : fa * fmaf(a.s, da, a.t), tb = fb == 0.f ? 0.f * b.s : fb * fmaf(b.s, db, b.t);
    return {M, a.s * fa + b.s * fb, ta + tb};
}
__device__ __forceinline__ Sums wave_join(Sums v) {
    for (int o = 1; o < kWave; o <<= 1)
        v = join(v, Sums{__shfl_xor(v.m, o, kWave), __shfl_xor(v.s, o, kWave), __shfl_xor(v.t, o, kWave)});
    return v;
}

__device__ __forceinline__ float pair_sum(const float (&v)[kPer]) {
    float w[kPer / 2];
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) w[i] = v[2 * i] + v[2 * i + 1];
#pragma unroll
    for (int n = kPer / 4; n > 0; n >>= 1)
#pragma unroll
        for (int i = 0; i < n; ++i) w[i] += w[i + n];
    return w[0];
}

__device__ __forceinline__ void add_logits(Sums& a, const float (&x)[kPer]) {
    float mx = a.m;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mx = fmaxf(mx, x[i]);
    const float M = mx == -INFINITY ? 0.f : mx;
    const float d = a.m == -INFINITY ? 0.f : (a.m - M) * kLog2e, f = __builtin_amdgcn_exp2f(d);
    float e[kPer], z[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const float y = (x[i] - M) * kLog2e;
        e[i] = __builtin_amdgcn_exp2f(y);
        z[i] = e[i] * fmaxf(y, -200.f);   // 0 for a logit of -inf
    }
    a.t = (f == 0.f ? 0.f * a.s : f * fmaf(a.s, d, a.t)) + pair_sum(z);
    a.s = a.s * f + pair_sum(e);
    a.m = mx;
}

template <bool kHalf>
__device__ __forceinline__ float logit_at(const void* row, int i) {
    if constexpr (kHalf)
        return h2f(static_cast<const uint16_t*>(row)[i]);
    else
        return static_cast<const float*>(row)[i];
}

// What one row comes to, from the joined sums.
struct RowEnd {
    float M, log_s;
    __device__ RowEnd(Sums v) : M(v.m), log_s(v.s == 0.f ? NAN : logf(v.s)) {}
    __device__ float logprob(float x) const { return x - M - log_s; }
};
__device__ __forceinline__ void write_row(const Logprobs& a, int r, Sums v, int rank, uint64_t top, int lane, float mine,
                                          bool given) {
    const RowEnd end(v);
    if (lane == 0) {
        if (a.entropies) a.entropies[r] = end.log_s - v.t * kLn2 / v.s;
        if (a.logprobs) a.logprobs[r] = given ? end.logprob(mine) : 0.f;
        if (a.ranks) a.ranks[r] = given ? rank : -1;
    }
    if (lane < a.top_k) {
        a.top_ids[(size_t)r * a.top_k + lane] = top ? (int32_t)~(uint32_t)top : -1;
        a.top_logprobs[(size_t)r * a.top_k + lane] = top ? end.logprob(key_logit(top)) : -INFINITY;
    }
}

// Workspace of a cut row: [rows][splits] of these, then their keys [k].
struct alignas(16) Part {
    float m, s, t;
    int rank;
};

// Workgroup (row, piece); its four waves take `per_wave` steps of 1024 logits
// each, 16-byte loads from the row's first aligned logit on, the next step's in
// flight.  The logits before it go to the row's first wave, those behind the
// last whole 16 bytes to its last.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void logprobs_kernel(Logprobs a, int splits, int per_wave) {
    constexpr int kVec = kHalf ? 8 : 4, kLoads = kPer / kVec;
    __shared__ uint64_t room[kWaves][kWave];
    __shared__ Part parts[kWaves];
    const int r = blockIdx.x / splits, split = blockIdx.x - r * splits;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.row_stride * (kHalf ? 2 : 4);
    const int lead = (int)((16 - ((uintptr_t)row & 15)) & 15) / (kHalf ? 2 : 4);
    const int head = min(lead, a.vocab);                   // logits before the aligned ones
    const int vecs = (a.vocab - head) / kVec, behind = head + vecs * kVec;
    const u32x4* body = reinterpret_cast<const u32x4*>(row + (size_t)head * (kHalf ? 2 : 4));
    const int steps = (vecs + kWave * kLoads - 1) / (kWave * kLoads);
    const int piece = split * kWaves + wave;
    const int first = min(steps, piece * per_wave), last = min(steps, first + per_wave);

    const int token = a.tokens ? a.tokens[r] : -1;
    const bool given = token >= 0 && token < a.vocab;
    const float mine = given ? logit_at<kHalf>(row, token) : NAN;
    // before the token an equal logit counts too: x > the float below
    const uint64_t my_key = logit_key(mine, 0);
    const bool nan_token = given && mine != mine;          // every other logit is before a NaN

    Sums sums{-INFINITY, 0.f, 0.f};
    int rank = 0;
    TopKeys top;
    top.room = room[wave];
    top.lane = lane;
    top.k = max(1, a.top_k);

    // one logit a lane (id >= vocab: none)
    auto add_one = [&](int id) {
        const bool real = id < a.vocab;
        const float x = real ? logit_at<kHalf>(row, id) : -INFINITY;
        sums = join(sums, Sums{x, x == -INFINITY ? 0.f : x == INFINITY ? NAN : x - x + 1.f, x - x == 0.f || x == -INFINITY ? 0.f : NAN});
        const uint64_t key = real ? logit_key(x, id) : 0ull;
        if (given) rank += nan_token ? key != 0 : key > ((my_key & ~0xffffffffull) | (uint32_t)~(uint32_t)token);
        if (a.top_k) top.add(key);
    };

    u32x4 raw[kLoads];
    auto load = [&](int step) {   // steps past the last one read it again
        const int at = min(step, steps - 1) * (kWave * kLoads) + lane;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) raw[i] = __builtin_nontemporal_load(body + min(at + i * kWave, vecs - 1));
    };
    if (piece == 0 && head > 0) add_one(lane < head ? lane : INT_MAX);
    if (first < last) {
        load(first);
        for (int step = first; step < last; ++step) {
            float x[kPer];
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (kHalf) {
                        const f16x2 h = as_h2(raw[i][j]);
                        x[i * kVec + 2 * j] = (float)h.x;
                        x[i * kVec + 2 * j + 1] = (float)h.y;
                    } else {
                        x[i * kVec + j] = __uint_as_float(raw[i][j]);
                    }
                }
            load(step + 1);
            const int vec0 = step * (kWave * kLoads) + lane;   // the lane's first; then every 64th
            const bool whole = (step + 1) * (kWave * kLoads) <= vecs;
            if (!whole) {
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (vec0 + i / kVec * kWave >= vecs) x[i] = -INFINITY;
            }
            auto id_of = [&](int i) {
                const int v = vec0 + i / kVec * kWave;
                return whole || v < vecs ? head + v * kVec + i % kVec : INT_MAX;
            };
            add_logits(sums, x);
            if (given) {
                const int id0 = head + step * kStep;
                if (nan_token) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) rank += x[i] == x[i] && id_of(i) != INT_MAX;
                } else if (whole && token >= id0 + kStep) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) rank += x[i] >= mine;
                } else if (token < id0) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) rank += x[i] > mine;
                } else {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) rank += x[i] > mine || (x[i] == mine && id_of(i) < token);
                }
            }
            if (a.top_k) {
                float mx = x[0];
#pragma unroll
                for (int i = 1; i < kPer; ++i) mx = fmaxf(mx, x[i]);
                // ids only grow, so a later logit equal to the k-th is not above it
                const uint64_t over = __builtin_amdgcn_ballot_w64(top.floor == 0 || mx > key_logit(top.floor));
                if (over != 0) {
                    if (__popcll(over) > 16) {
                        uint64_t best = 0;
#pragma unroll
                        for (int i = 0; i < kPer; ++i) {
                            const uint64_t key = id_of(i) == INT_MAX ? 0ull : logit_key(x[i], id_of(i));
                            best = key > best ? key : best;
                        }
                        top.raise(best);
                    }
                    // registers i with a candidate, each added in turn
                    const float least = top.floor == 0 ? -INFINITY : key_logit(top.floor);
                    uint32_t todo = 0;
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        todo |= (__builtin_amdgcn_ballot_w64(x[i] >= least) != 0 ? 1u : 0u) << i;
                    while (todo != 0) {
                        const int i = __builtin_ctz(todo);
                        todo &= todo - 1;
                        float xi = x[0];
#pragma unroll
                        for (int j = 1; j < kPer; ++j) xi = i == j ? x[j] : xi;
                        top.add(id_of(i) == INT_MAX ? 0ull : logit_key(xi, id_of(i)));
                    }
                }
            }
        }
    }
    if (piece == splits * kWaves - 1 && behind < a.vocab) add_one(lane < a.vocab - behind ? behind + lane : INT_MAX);

    // the waves of the workgroup, then the piece or the row
    sums = wave_join(sums);
    for (int o = 1; o < kWave; o <<= 1) rank += __shfl_xor(rank, o, kWave);
    if (a.top_k) top.flush();
    if (lane == 0) parts[wave] = Part{sums.m, sums.s, sums.t, rank};
    room[wave][lane] = top.mine;
    __syncthreads();
    if (wave != 0) return;
    for (int w = 1; w < kWaves; ++w) {
        sums = join(sums, Sums{parts[w].m, parts[w].s, parts[w].t});
        rank += parts[w].rank;
        if (a.top_k) top.mine = merge_descending(top.mine, room[w][lane], lane);
    }
    if (splits == 1) {
        write_row(a, r, sums, rank, top.mine, lane, mine, given);
        return;
    }
    Part* out = static_cast<Part*>(a.workspace) + blockIdx.x;
    if (lane == 0) *out = Part{sums.m, sums.s, sums.t, rank};
    uint64_t* keys = reinterpret_cast<uint64_t*>(static_cast<Part*>(a.workspace) + (size_t)a.rows * splits);
    if (lane < a.top_k) keys[(size_t)blockIdx.x * a.top_k + lane] = top.mine;
}

// One wave joins the pieces of a row.
template <bool kHalf>
__global__ __launch_bounds__(kWave) void logprobs_join_kernel(Logprobs a, int splits) {
    __shared__ uint64_t room[kWave];
    const int r = blockIdx.x, lane = threadIdx.x;
    const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.row_stride * (kHalf ? 2 : 4);
    const int token = a.tokens ? a.tokens[r] : -1;
    const bool given = token >= 0 && token < a.vocab;
    const float mine = given ? logit_at<kHalf>(row, token) : NAN;
    const Part* parts = static_cast<const Part*>(a.workspace) + (size_t)r * splits;
    Sums sums{-INFINITY, 0.f, 0.f};
    int rank = 0;
    for (int j = lane; j < splits; j += kWave) {
        const Part p = parts[j];
        sums = join(sums, Sums{p.m, p.s, p.t});
        rank += p.rank;
    }
    sums = wave_join(sums);
    for (int o = 1; o < kWave; o <<= 1) rank += __shfl_xor(rank, o, kWave);
    TopKeys top;
    top.room = room;
    top.lane = lane;
    top.k = max(1, a.top_k);
    if (a.top_k) {
        const uint64_t* keys =
            reinterpret_cast<const uint64_t*>(static_cast<const Part*>(a.workspace) + (size_t)a.rows * splits) +
            (size_t)r * splits * a.top_k;
        const int n = splits * a.top_k;
        for (int j0 = 0; j0 < n; j0 += kStep) {
            uint64_t key[kPer], best = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int j = j0 + i * kWave + lane;
                key[i] = j < n ? keys[j] : 0ull;
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) best = key[i] > best ? key[i] : best;
            top.raise(best);
#pragma unroll
            for (int i = 0; i < kPer; ++i) top.add(key[i]);
        }
        top.flush();
    }
    write_row(a, r, sums, rank, top.mine, lane, mine, given);
}

// Pieces of a row: about four workgroups per CU over all rows, each wave with a
// whole step at least.
constexpr int kTargetBlocks = 1024;
struct Cut {
    int splits, per_wave;
};
Cut cut_row(int rows, int vocab) {
    const int steps = std::max(1, (vocab + kStep - 1) / kStep);
    const int want = std::max(1, std::min((steps + kWaves - 1) / kWaves, kTargetBlocks / std::min(rows, kTargetBlocks)));
    Cut c;
    c.per_wave = (steps + want * kWaves - 1) / (want * kWaves);
    c.splits = (steps + c.per_wave * kWaves - 1) / (c.per_wave * kWaves);
    return c;
}

}  // namespace

size_t logprobs_workspace(int rows, int vocab, int top_k) {
    const Cut c = cut_row(rows, vocab);
    return c.splits == 1 ? 0 : (size_t)rows * c.splits * (sizeof(Part) + sizeof(uint64_t) * top_k);
}

namespace {
template <bool kHalf>
void launch_for(const Logprobs& a, hipStream_t s) {
    const Cut c = cut_row(a.rows, a.vocab);
    launch_kernel_in_call(c.splits == 1, logprobs_kernel<kHalf>, dim3((unsigned)a.rows * c.splits), dim3(kBlk), 0, s, a,
                          c.splits, c.per_wave);
    if (c.splits > 1) launch_kernel(logprobs_join_kernel<kHalf>, dim3(a.rows), dim3(kWave), 0, s, a, c.splits);
}
}  // namespace

hipError_t launch_token_logprobs(const Logprobs& a, hipStream_t s) {
    if (a.half)
        launch_for<true>(a, s);
    else
        launch_for<false>(a, s);
    return hipGetLastError();
}

}  // namespace citlali::hip
