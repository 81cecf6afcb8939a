// logprobs.hip -- log probability and rank of a given token, entropy and the
// most likely tokens of each row of logits, in one pass over them.
//
// With m a row's maximum, s = sum 2^y and t = sum 2^y y over y = (x - m) log2 e,
//   log p(x) = x - m - log s        H = log s - ln 2 t / s.
// Every lane keeps (m, s, t) of its own logits, 16 at a time: their maximum
// first, then one rescaling, then their exponentials.  A row is cut into pieces
// of whole waves; lanes, waves and workgroups join by
//   (m, s, t) + (m', s', t'):  s f + s' f',  f (t + s d) + ...,  f = 2^d.
//
// The most likely tokens are kept as 64-bit keys (ordered bits of the logit,
// then the complement of the id, so that equal logits go by the lower id):
// lane i of a wave has the wave's i-th largest.  Logits below the k-th, the
// wave's own or another's of the workgroup, cost one comparison per 16; those
// above it are gathered in LDS, and 64 of them are sorted across the lanes and
// merged at a time.  Where many lanes have one (a row's first steps), a sort of
// the lanes' largest raises the threshold first.  The order is total, so the
// result does not depend on the cut.
//
// Bound by reading the logits where there are many rows: 2048 rows of 151936
// fp16 logits, 622 MB, in 122 us (5.1 TB/s); beside them a wave issues about 8
// vector instructions per 64 logits, one of them the exponential.  A few rows
// are a chain of latencies, the sorts its longest part: 8 rows 7.8 us and the
// join of their pieces 4.6.
#include "device_common.hpp"
#include "launch.hpp"

#include <float.h>
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

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
// Both of a lane's and its partner's (lane ^ kStride) values, in either order.
template <int kStride>
__device__ __forceinline__ void both(uint32_t v, uint32_t& a, uint32_t& b) {
    a = b = v;
    if constexpr (kStride >= 16) {
        float x = __uint_as_float(v), y = x;
        if constexpr (kStride == 16)
            swap16(x, y);
        else
            swap32(x, y);
        a = __float_as_uint(x);
        b = __float_as_uint(y);
    } else if constexpr (kStride == 4) {   // i ^ 7, then i ^ 3
        const int t = __builtin_amdgcn_update_dpp(0, (int)v, kDppHalfMirror, 0xF, 0xF, false);
        b = __builtin_amdgcn_update_dpp(0, t, 0x1B, 0xF, 0xF, false);
    } else {
        constexpr int kCtrl = kStride == 1 ? kDppXor1 : kStride == 2 ? kDppXor2 : DppRor<8>::value;
        b = __builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, false);
    }
}
// Larger of a lane's and its partner's key where `up`, else the smaller.
template <int kStride>
__device__ __forceinline__ uint32_t exchange(uint32_t v, bool up) {
    uint32_t a, b;
    both<kStride>(v, a, b);
    return (a > b) == up ? a : b;
}
template <int kStride>
__device__ __forceinline__ uint64_t exchange(uint64_t v, bool up) {
    uint32_t a0, a1, b0, b1;
    both<kStride>((uint32_t)v, a0, b0);
    both<kStride>((uint32_t)(v >> 32), a1, b1);
    const uint64_t a = ((uint64_t)a1 << 32) | a0, b = ((uint64_t)b1 << 32) | b0;
    return (a > b) == up ? a : b;
}
// The steps kStride, kStride / 2, .. 1 of a bitonic merge; each run of kSize
// lanes descends where `down`.
template <int kStride, typename T>
__device__ __forceinline__ T merge_steps(T v, int lane, bool down) {
    v = exchange<kStride>(v, ((lane & kStride) == 0) == down);
    if constexpr (kStride > 1) v = merge_steps<kStride / 2>(v, lane, down);
    return v;
}
template <typename T>
__device__ __forceinline__ T sort_descending(T v, int lane) {
    v = merge_steps<1>(v, lane, (lane & 2) == 0);
    v = merge_steps<2>(v, lane, (lane & 4) == 0);
    v = merge_steps<4>(v, lane, (lane & 8) == 0);
    v = merge_steps<8>(v, lane, (lane & 16) == 0);
    v = merge_steps<16>(v, lane, (lane & 32) == 0);
    return merge_steps<32>(v, lane, true);
}
// The 64 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t merge_descending(uint64_t a, uint64_t b, int lane) {
    const uint64_t w = __shfl((unsigned long long)b, kWave - 1 - lane, kWave);
    return merge_steps<32>(a > w ? a : w, lane, true);
}
__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return ((uint64_t)hi << 32) | lo;
}

// `lane`, of which the compiler keeps no comparisons from one sort to the next
// (they would fill the scalar registers of the whole kernel).
__device__ __forceinline__ int hidden(int lane) {
    asm("" : "+v"(lane));
    return lane;
}

// v[i] for an i of the lane's own.
template <typename T>
__device__ __forceinline__ T pick(const T (&v)[kPer], int i) {
    T a[kPer / 2];
    auto half = [](bool second, T x, T y) { return second ? y : x; };   // of values: the array stays in registers
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = half(i & 1, v[2 * j], v[2 * j + 1]);
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = half(i & 2, a[2 * j], a[2 * j + 1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) a[j] = half(i & 4, a[2 * j], a[2 * j + 1]);
    return half(i & 8, a[0], a[1]);
}

struct TopKeys {
    uint64_t mine = 0;    // lane i: the i-th largest
    uint64_t floor = 0;   // only keys above it can be among the k largest (uniform)
    uint64_t theirs = 0;  // likewise, from the workgroup's other waves
    int waiting = 0;      // keys in `room` (uniform)
    uint64_t* room;       // 64 of LDS, the wave's own
    int lane, k;

    __device__ uint64_t least() const { return floor > theirs ? floor : theirs; }
    __device__ void flush() {
        wave_lds_sync();
        const uint64_t v = lane < waiting ? room[lane] : 0ull;
        wave_lds_sync();
        const int at = hidden(lane);
        const uint64_t sorted = sort_descending(v, at);
        mine = lane_key(mine, 0) == 0 ? sorted : merge_descending(mine, sorted, at);
        const uint64_t kth = lane_key(mine, k - 1);
        floor = kth > floor ? kth : floor;
        waiting = 0;
    }
    __device__ void add(uint64_t key) {
        const uint64_t low = least();
        uint64_t who = __builtin_amdgcn_ballot_w64(key > low);
        if (who == 0) return;
        if (waiting + __popcll(who) > kWave) {
            flush();
            who = __builtin_amdgcn_ballot_w64(key > least());
        }
        if (key > least()) room[waiting + below(who)] = key;
        waiting += __popcll(who);
    }
    // The keys key_of(i) of the lane's marks (one not above least() does no harm).
    template <typename F>
    __device__ void add_marked(uint32_t marks, F key_of) {
        const int count = __builtin_popcount(marks);
        int before = 0, total = 0;   // over the lanes, the counts' bits in turn
#pragma unroll
        for (int b = 0; 1 << b <= kPer; ++b) {
            const uint64_t who = __builtin_amdgcn_ballot_w64((count >> b & 1) != 0);
            before += below(who) << b;
            total += __popcll(who) << b;
        }
        const bool fits = waiting + total <= kWave;
        int at = waiting + before;
        waiting += fits ? total : 0;
        while (__builtin_amdgcn_ballot_w64(marks != 0) != 0) {   // a key of each lane
            const uint64_t key = marks != 0 ? key_of(__builtin_ctz(marks)) : 0ull;
            if (!fits)
                add(key);
            else if (marks != 0)
                room[at++] = key;
            marks &= marks - 1;
        }
    }
    // Before many keys at once, of which `best` are the lanes' largest (their
    // upper halves): at least k of them reach the k-th largest of those.
    __device__ void raise(uint32_t best) {
        const uint32_t reach = __builtin_amdgcn_readlane((int)sort_descending(best, hidden(lane)), k - 1);
        const uint64_t kth = (uint64_t)reach << 32;
        floor = kth > floor ? kth : floor;
    }

private:
    // lanes of `who` below this one
    __device__ static int below(uint64_t who) {
        return __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
    }
};

// ---- sums --------------------------------------------------------------------
struct Sums {
    float m, s, t;
};
// Sums rescaled to maximum m.
__device__ __forceinline__ Sums rescaled(Sums a, float m) {
    // without a logit above -inf s and t are 0 (or NaN, which stays)
    const float d = a.m == -INFINITY ? 0.f : (a.m - m) * kLog2e, f = __builtin_amdgcn_exp2f(d);
    // a factor of 0 takes t with it (d may be infinite), but for a NaN
    return {m, a.s * f, f == 0.f ? 0.f * a.s : f * fmaf(a.s, d, a.t)};
}
__device__ __forceinline__ Sums join(Sums a, Sums b) {
    const float m = fmaxf(a.m, b.m);
    a = rescaled(a, m);
    b = rescaled(b, m);
    return {m, a.s + b.s, a.t + b.t};
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

// 16 logits of a lane as they were loaded: fp32, or pairs of fp16.
template <bool kHalf>
struct Logits {
    static constexpr int kVec = kHalf ? 8 : 4, kLoads = kPer / kVec;
    u32x4 w[kLoads];
    __device__ uint32_t word(int i) const { return w[i / kVec][kHalf ? i % kVec / 2 : i % kVec]; }
    __device__ auto at(int i) const {
        if constexpr (kHalf)
            return __builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? word(i) >> 16 : word(i)));
        else
            return __uint_as_float(word(i));
    }
    __device__ float largest() const {
        if constexpr (kHalf) {
            uint32_t m = word(0);
#pragma unroll
            for (int i = 2; i < kPer; i += 2) asm("v_pk_max_f16 %0, %1, %2" : "=v"(m) : "v"(m), "v"(word(i)));
            return fmaxf((float)as_h2(m).x, (float)as_h2(m).y);
        } else {
            float m = at(0);
#pragma unroll
            for (int i = 1; i < kPer; ++i) m = fmaxf(m, at(i));
            return m;
        }
    }
    // y of logit i
    __device__ float reach(int i, float m) const {
        float d;
        if constexpr (!kHalf)
            d = at(i) - m;
        else if (i & 1)
            asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(word(i)), "v"(m));
        else
            asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(d) : "v"(word(i)), "v"(m));
        return d * kLog2e;
    }
};
template <bool kHalf>
__device__ __forceinline__ void add_logits(Sums& a, const Logits<kHalf>& x, float largest) {
    const float m = fmaxf(a.m, largest), from = m == -INFINITY ? 0.f : m;
    float e[kPer], z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const float y = x.reach(i, from);
        e[i] = __builtin_amdgcn_exp2f(y);
        z[i % 4] = fmaf(e[i], fmaxf(y, -FLT_MAX), z[i % 4]);   // 0 for a logit of -inf
    }
    a = rescaled(a, m);
    a.t += (z[0] + z[1]) + (z[2] + z[3]);
    a.s += pair_sum(e);
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
    float m, log_s;
    __device__ RowEnd(Sums v) : m(v.m), log_s(v.s == 0.f ? NAN : logf(v.s)) {}
    __device__ float logprob(float x) const { return x - m - log_s; }
};
__device__ __forceinline__ void write_row(const Logprobs& a, int r, Sums v, int rank, uint64_t top, int lane,
                                          float mine, bool given) {
    const RowEnd end(v);
    if (lane == 0) {
        if (a.entropies) a.entropies[r] = end.log_s - kLn2 * (v.t / v.s);
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
// flight.  What is left of the row, before that logit and behind the last whole
// step, goes to the waves one logit a lane.
template <bool kHalf>
__global__ __launch_bounds__(kBlk) void logprobs_kernel(Logprobs a, int splits, int per_wave) {
    using L = Logits<kHalf>;
    using Logit = std::conditional_t<kHalf, _Float16, float>;
    constexpr int kVecs = kWave * L::kLoads;   // vectors of a step
    __shared__ uint64_t room[kWaves][kWave];
    __shared__ Part parts[kWaves];
    __shared__ uint64_t floors[kWaves];   // the waves' own, read without waiting for one another
    const int r = blockIdx.x / splits, split = blockIdx.x - r * splits;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const char* row = static_cast<const char*>(a.logits) + (size_t)r * a.row_stride * (kHalf ? 2 : 4);
    const int head = min(a.vocab, (int)((16 - ((uintptr_t)row & 15)) & 15) / (kHalf ? 2 : 4));
    const int steps = (a.vocab - head) / kStep;
    const u32x4* body = reinterpret_cast<const u32x4*>(row + (size_t)head * (kHalf ? 2 : 4)) + lane;
    const int piece = split * kWaves + wave;
    // the workgroup's steps in turn over its waves: 8 or 16 KB of the row at a time
    const int first = min(steps, split * kWaves * per_wave + wave), last = min(steps, (split + 1) * kWaves * per_wave);

    const int token = a.tokens ? a.tokens[r] : -1;
    const bool given = token >= 0 && token < a.vocab;
    const float mine = given ? logit_at<kHalf>(row, token) : NAN;
    const Logit given_x = (Logit)mine;
    const bool nan_token = given && mine != mine;   // every other logit is before a NaN

    Sums sums{-INFINITY, 0.f, 0.f};
    int rank = 0;   // logits of the lane before the given one
    TopKeys top;
    top.room = room[wave];
    top.lane = lane;
    top.k = max(1, a.top_k);

    if (lane == 0) floors[wave] = 0;
    __syncthreads();
    L next;
    auto load = [&](int step) {
#pragma unroll
        for (int i = 0; i < L::kLoads; ++i)
            next.w[i] = __builtin_nontemporal_load(body + (size_t)step * kVecs + i * kWave);
    };
    if (first < last) load(first);
    for (int step = first; step < last; step += kWaves) {
        const L x = next;
        load(min(step + kWaves, last - 1));
        const int id0 = head + step * kStep;
        auto id_of = [&](int i) { return id0 + (i / L::kVec * kWave + lane) * L::kVec + i % L::kVec; };
        uint64_t others[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
            others[w] = __hip_atomic_load(&floors[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        const float largest = x.largest();
        add_logits(sums, x, largest);
        if (given) {
            if (nan_token) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) rank += x.at(i) == x.at(i);
            } else if (token >= id0 + kStep) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) rank += x.at(i) >= given_x;
            } else if (token < id0) {
#pragma unroll
                for (int i = 0; i < kPer; ++i) rank += x.at(i) > given_x;
            } else {
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    rank += x.at(i) > given_x || (x.at(i) == given_x && id_of(i) < token);
            }
        }
        if (a.top_k) {
            uint64_t theirs = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) theirs = others[w] > theirs ? others[w] : theirs;
            top.theirs = lane_key(theirs, 0);
            // the least logit of a key above least(); an equal one only where its id may be lower
            auto limit = [&] {
                const uint64_t least = top.least();
                const uint64_t next = (uint64_t)((uint32_t)id0 >= ~(uint32_t)least) << 32;
                return least == 0 ? -INFINITY : key_logit(least + next);
            };
            float low = limit();
            // (beside a NaN `largest` may miss a logit: a signalling one makes the
            // maximum a NaN, whatever came before)
            const uint64_t over = __builtin_amdgcn_ballot_w64(largest >= low || sums.s != sums.s);
            if (over != 0) {
                if (__popcll(over) > 16) {
                    top.raise((uint32_t)(logit_key(largest, 0) >> 32));
                    low = limit();
                }
                float v[kPer];
                uint32_t marks = 0;
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    v[i] = (float)x.at(i);
                    marks |= (v[i] >= low ? 1u : 0u) << i;
                }
                top.add_marked(marks, [&](int i) { return logit_key(pick(v, i), id_of(i)); });
                if (lane == 0)
                    __hip_atomic_store(&floors[wave], top.floor, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
        }
    }

    const int rest = a.vocab - steps * kStep;   // the first `head` of them at the row's start
    for (int j = piece * kWave; j < rest; j += splits * kWaves * kWave) {
        const int n = j + lane, id = n < head ? n : n + steps * kStep;
        const bool real = n < rest;
        const float x = real ? logit_at<kHalf>(row, id) : -INFINITY;
        const bool any = x > -INFINITY || x != x;
        sums = join(sums, Sums{x, !any ? 0.f : x - x == 0.f ? 1.f : NAN, !any || x - x == 0.f ? 0.f : NAN});
        const uint64_t key = real ? logit_key(x, id) : 0ull;
        if (given) rank += key > logit_key(mine, token);
        if (a.top_k) top.add(key);
    }

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
            top.raise((uint32_t)(best >> 32));
            uint32_t marks = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) marks |= (key[i] > top.least() ? 1u : 0u) << i;
            top.add_marked(marks, [&](int i) { return pick(key, i); });
        }
        top.flush();
    }
    write_row(a, r, sums, rank, top.mine, lane, mine, given);
}

// Pieces of a row: about four workgroups per CU over all rows, each wave with a
// whole step at least; rows as many as CUs stay whole.  us for 151936 fp32 logits,
// 20 listed: 8 rows 12.9 with one step a wave, 14.3 with two, 18.5 with four; 100
// rows 27.4 (half or twice as many workgroups 27.6, 28.9), 200 rows of fp16 34.1
// (40.9); 300 rows whole 45.8, in three pieces 48.6, 500 rows 52.2, in two 64.6.
constexpr int kTargetBlocks = 1024, kWholeRows = 256;
struct Cut {
    int splits, per_wave;
};
Cut cut_row(int rows, int vocab) {
    const int steps = std::max(1, (vocab + kStep - 1) / kStep);
    const int want = rows > kWholeRows ? 1 : std::min((steps + kWaves - 1) / kWaves, kTargetBlocks / rows);
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
