// lx_logprobs.hip -- TokenLogProbs on gfx950: for each row of logits the log-probability of one given token, the
// entropy of the distribution and the most probable tokens, from one pass over the logits.
//
// With m the row's maximum, n how often it occurs, r the sum of exp(x - m) over the other logits and t the sum of
// exp(x - m) (m - x):
//   log S = log1p((n - 1) + r),  log p(i) = (x[i] - m) - log S,  entropy = log S + t / (n + r).
// Every sum is of terms of one sign and none holds the maximum's own 1, so a distribution that is all but certain
// keeps its digits.  (m, r, t, n) of two parts of a row merge into those of both (stat_merge), so a row may be
// split over threads and workgroups; the merges run in a fixed order and a row's result does not change from run
// to run.  A NaN or +inf logit makes r NaN, and with it every value of the row; a row of -inf has n = 0: NaN too.
//
// The most probable tokens come from the same pass: each thread keeps the largest of the four-logit units it reads,
// and the k-th largest over 64 groups of threads bounds the k-th largest logit from below (k distinct units reach
// it).  Only the logits of threads whose own largest reaches the bound are read again, and only logits that reach it
// are ranked, by counting; equal logits rank by index.
//
// Many rows are bound by memory: [4096, 30522] 91 us, 5.5 TB/s (with the top 5 about 105).  Few rows are bound by
// launches and the waits of the ranking: [1, 131072] 7 us in two launches, 11.4 with the top 20.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lx_device.h"
#include "lx_kernels.h"

namespace lx {

constexpr int kLpBlock = 256, kLpSplit = 64;

struct LpStat {
    float m, r, t, n;
};

__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504f); }

// brings a part's sums to the maximum of the whole: its own maximum joins the others where it is smaller
__device__ __forceinline__ void stat_scale(LpStat &s, float m) {
    const float d = fminf(m - s.m, 1e30f), e = s.m == m ? 1.0f : lp_exp(-d);
    const float q = s.r + s.n;
    s.t = s.m == m ? s.t : e * (s.t + d * q);
    s.r = s.m == m ? s.r : e * q;
    s.n = s.m == m ? s.n : 0.0f;
    s.m = m;
}

__device__ __forceinline__ LpStat stat_merge(LpStat a, LpStat b) {
    const float m = fmaxf(a.m, b.m);
    stat_scale(a, m);
    stat_scale(b, m);
    return {m, a.r + b.r, a.t + b.t, a.n + b.n};
}

__device__ __forceinline__ LpStat stat_xor(const LpStat &s, int o) {
    return {__shfl_xor(s.m, o), __shfl_xor(s.r, o), __shfl_xor(s.t, o), __shfl_xor(s.n, o)};
}
__device__ __forceinline__ LpStat stat_wave(LpStat s) {
    for (int o = 1; o < 64; o <<= 1) s = stat_merge(s, stat_xor(s, o));
    return s;
}

// A logit's rank as a number: larger logits are larger, NaN is below all, zero means none; equal logits by index.
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);  // -0 counts as 0
    return x != x ? 0u : (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) {
    return o == 0 ? __builtin_nanf("") : __builtin_bit_cast(float, (o >> 31) ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t index) { return (uint64_t)lp_order(x) << 32 | (uint32_t)~index; }

// A row in units of four logits, each 16-byte aligned: unit u holds logits 4 u - off .. 4 u - off + 3, those outside
// the row read as -inf.
struct LpRow {
    const float *base;  // the first unit
    int off, v;
    uint32_t units;
    __device__ __forceinline__ LpRow(const float *x, int64_t v_) : v((int)v_) {
        off = (int)(((uintptr_t)x >> 2) & 3);
        base = x - off;
        units = (uint32_t)((v_ + off + 3) / 4);
    }
    __device__ __forceinline__ float4 load(uint32_t u) const {
        const int e = (int)(4 * u) - off;
        if (e >= 0 && e + 4 <= v) return *(const float4 *)(base + 4 * (int64_t)u);
        float4 f;
        float *p = &f.x;
        for (int i = 0; i < 4; i++) p[i] = e + i >= 0 && e + i < v ? base[4 * (int64_t)u + i] : -__builtin_inff();
        return f;
    }
    __device__ __forceinline__ bool inside(uint32_t u, int i) const {
        const int e = (int)(4 * u) - off + i;
        return e >= 0 && e < v;
    }
};

__device__ __forceinline__ float max4(float4 f) { return fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w)); }

__device__ __forceinline__ void stat_add(LpStat &s, const float4 *f, int units) {
    float m = s.m;
#pragma unroll
    for (int c = 0; c < units; c++) m = fmaxf(m, max4(f[c]));
    stat_scale(s, m);
    const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int c = 0; c < units; c++) {
        const float *p = &f[c].x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float d = p[i] - base;
            const bool top = d == 0.0f;
            const float e = top ? 0.0f : lp_exp(d);
            s.n += top ? 1.0f : 0.0f;
            s.r += e;
            s.t = __builtin_fmaf(e, fminf(-d, 1e30f), s.t);
        }
    }
}

// A row is a team's work: one wave's (TEAM 64, four rows a workgroup) or a whole workgroup's (TEAM 256 or 1024).
template <int TEAM> __device__ __forceinline__ void team_sync() {
    if constexpr (TEAM == 64) {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    } else {
        __syncthreads();
    }
}

template <int TEAM> struct LpShared {
    static constexpr int kCap = 4 * TEAM + 2 * TEAM + 512;  // a round's keys, and those kept or waiting
    uint64_t buf[kCap + 8];
    uint64_t group[TEAM];
    uint64_t top[kLogProbsTop];
    uint32_t winner[TEAM];
    LpStat wave[TEAM / 64];
    uint64_t bound;
    int count, winners;
};

// The k largest of `count` distinct keys into out, largest first (buf has room for eight more; the team's writes to it
// are done).
template <int TEAM> __device__ __forceinline__ void rank_keys(uint64_t *buf, int count, int k, uint64_t *out, int lane) {
    if (lane < 8) buf[count + lane] = 0;
    team_sync<TEAM>();
    for (int c = lane; c < count; c += TEAM) {
        const uint64_t mine = buf[c];
        int rank = 0;
        for (int j = 0; j < count; j += 8) {
#pragma unroll
            for (int i = 0; i < 8; i++) rank += buf[j + i] > mine;
        }
        if (rank < k) out[rank] = mine;
    }
}

__device__ __forceinline__ uint64_t lane_key(uint64_t g, int j) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)g, j), hi = __builtin_amdgcn_readlane((int)(g >> 32), j);
    return (uint64_t)hi << 32 | lo;
}

// the k-th largest of the wave's keys, distinct but for zeros (none): zero if fewer than k are there
__device__ __forceinline__ uint64_t wave_kth(uint64_t g, int k) {
    const uint32_t hi = (uint32_t)(g >> 32);
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 64; j++) rank += (uint32_t)__builtin_amdgcn_readlane((int)hi, j) > hi;
    uint64_t at = __ballot(hi != 0 && rank == k - 1);
    if (__popcll(__ballot(rank < k)) != k || __popcll(at) != 1) {  // equal values around the k-th: by unit
        rank = 0;
        for (int j = 0; j < 64; j++) rank += lane_key(g, j) > g;
        at = __ballot(g != 0 && rank == k - 1);
    }
    return at ? lane_key(g, __builtin_ctzll(at)) : 0;
}
// the same of two keys a lane
__device__ __forceinline__ uint64_t wave_kth2(uint64_t g0, uint64_t g1, int k) {
    int r0 = 0, r1 = 0;
#pragma unroll 8
    for (int j = 0; j < 64; j++) {
        const uint64_t a = lane_key(g0, j), b = lane_key(g1, j);
        r0 += (a > g0) + (b > g0);
        r1 += (a > g1) + (b > g1);
    }
    const uint64_t at0 = __ballot(g0 != 0 && r0 == k - 1), at1 = __ballot(g1 != 0 && r1 == k - 1);
    return at0 ? lane_key(g0, __builtin_ctzll(at0)) : at1 ? lane_key(g1, __builtin_ctzll(at1)) : 0;
}

// sh.top[0 .. k) = the k largest keys of units [u0, u1) of the row, zeros where there are fewer; `best` is this
// thread's largest unit (value, unit) of those u0 + lane + TEAM i, zero if none.
template <int TEAM>
__device__ void team_top(const LpRow &row, uint32_t u0, uint32_t u1, int k, uint64_t best, LpShared<TEAM> &sh, int lane) {
    using Sh = LpShared<TEAM>;
    sh.group[lane] = best;
    if (lane < kLogProbsTop) sh.top[lane] = 0;
    if (lane == 0) sh.count = sh.winners = 0;
    team_sync<TEAM>();
    if (lane < 64) {
        uint64_t g = best;
        if constexpr (TEAM == 64) {
            g = wave_kth(g, k);
        } else {
            uint64_t g2 = 0;
#pragma unroll
            for (int w = 0; w < TEAM / 64; w++) {
                const uint64_t y = sh.group[64 * w + lane];
                if (w < TEAM / 128) g = std::max(g, y);
                else g2 = std::max(g2, y);
            }
            // over half of the 64 groups would let many logits past the bound: then 128 of them
            g = k > 32 ? wave_kth2(g, g2, k) : wave_kth(std::max(g, g2), k);
        }
        if (lane == 0) sh.bound = g;
    }
    team_sync<TEAM>();
    const uint64_t bound = sh.bound;
    if (best >= bound) sh.winner[atomicAdd(&sh.winners, 1)] = lane;
    team_sync<TEAM>();
    // the winners' units, shared out over the team
    const uint32_t winners = sh.winners, total = winners * ((u1 - u0 + TEAM - 1) / TEAM);
    auto unit = [&](uint32_t i) { return u0 + sh.winner[i % winners] + TEAM * (i / winners); };
    auto offer = [&](const float4 &f, uint32_t u, auto &&take) {
        const float *p = &f.x;
        for (int i = 0; i < 4; i++)
            if (lp_key(p[i], u) >= bound && row.inside(u, i)) take(lp_key(p[i], 4 * u - row.off + i));
    };
    for (uint32_t i = lane; i < total; i += 4 * TEAM) {
        float4 f[4];
        uint32_t u[4];
#pragma unroll
        for (int c = 0; c < 4; c++) {
            u[c] = i + c * TEAM < total ? unit(i + c * TEAM) : u1;
            if (u[c] < u1) f[c] = row.load(u[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (u[c] < u1)
                offer(f[c], u[c], [&](uint64_t key) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < Sh::kCap) sh.buf[at] = key;
                });
    }
    team_sync<TEAM>();
    int count = sh.count;
    if (count <= Sh::kCap) {
        rank_keys<TEAM>(sh.buf, count, k, sh.top, lane);
        team_sync<TEAM>();
        return;
    }
    // more than the buffer holds (few distinct logits, or sorted ones): by rounds, the k largest so far kept
    team_sync<TEAM>();
    if (lane == 0) sh.count = 0;
    team_sync<TEAM>();
    for (uint32_t i = 0; i < total; i += TEAM) {
        const uint32_t u = i + lane < total ? unit(i + lane) : u1;
        if (u < u1) {
            const uint64_t least = sh.top[k - 1];
            offer(row.load(u), u, [&](uint64_t key) {
                if (key > least) sh.buf[atomicAdd(&sh.count, 1)] = key;
            });
        }
        team_sync<TEAM>();
        count = sh.count;
        // room for the next round's 4 TEAM keys, or the last round
        if (count > Sh::kCap - 4 * TEAM - kLogProbsTop || i + TEAM >= total) {
            int kept = 0;
            while (kept < k && sh.top[kept]) kept++;
            if (lane < kept) sh.buf[count + lane] = sh.top[lane];
            team_sync<TEAM>();
            rank_keys<TEAM>(sh.buf, count + kept, k, sh.top, lane);
            if (lane == 0) sh.count = 0;
        }
        team_sync<TEAM>();
    }
}

// The given token's logit, read by the team's first lane before the row's pass, behind which its latency hides.
struct LpAsked {
    int64_t id;
    float x;
    __device__ __forceinline__ LpAsked(const LogProbsArgs &a, int64_t row, bool mine) : id(-1), x(0.0f) {
        if (!a.ids || !mine) return;
        id = a.ids_dtype == kInt64 ? ((const int64_t *)a.ids)[row] : (int64_t)((const int32_t *)a.ids)[row];
        if (id >= 0 && id < a.v) x = a.x[row * a.v + id];
    }
};

// a row's outputs from its sums and sorted keys
template <int TEAM>
__device__ __forceinline__ void lp_finish(const LogProbsArgs &a, int64_t row, const LpStat &s, const LpAsked &q,
                                          const uint64_t *top, int lane) {
    const float ls = s.n > 0.0f ? log1pf((s.n - 1.0f) + s.r) : __builtin_nanf("");
    if (lane == 0) {
        if (a.ids) a.lp[row] = q.id < 0 ? 0.0f : q.id >= a.v ? __builtin_nanf("") : (q.x - s.m) - ls;
        if (a.h) a.h[row] = ls + s.t / (s.n + s.r);
    }
    if (lane < a.top) {
        const uint64_t key = top[lane];
        a.top_ids[row * a.top + lane] = (int64_t)(uint32_t)~(uint32_t)key;
        a.top_lp[row * a.top + lane] = (lp_value((uint32_t)(key >> 32)) - s.m) - ls;
    }
}

// A part of a row (SPLIT: kLpSplit parts at most, their sums and keys to a.part) or a whole row for each team.
template <int TEAM, bool TOP, bool SPLIT>
__global__ __launch_bounds__(TEAM > kLpBlock ? TEAM : kLpBlock) void k_logprobs(LogProbsArgs a, int split) {
    constexpr int TEAMS = TEAM > kLpBlock ? 1 : kLpBlock / TEAM;
    __shared__ LpShared<TEAM> shared[TEAMS];
    const int lane = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    LpShared<TEAM> &sh = shared[team];
    const int64_t total = a.t * split;
    for (int64_t b = (int64_t)blockIdx.x * TEAMS + team; b < total; b += (int64_t)gridDim.x * TEAMS) {
        const int64_t r = SPLIT ? b / split : b;
        const int part = SPLIT ? (int)(b - r * split) : 0;
        const LpAsked asked(a, r, !SPLIT && lane == 0);
        const LpRow row(a.x + r * a.v, a.v);
        const uint32_t per = SPLIT ? (uint32_t)(((a.v + 6) / 4 + split - 1) / split) : row.units;
        const uint32_t u0 = std::min(row.units, part * per), u1 = std::min(row.units, u0 + per);
        const float4 none = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
        LpStat s = {-__builtin_inff(), 0.0f, 0.0f, 0.0f};
        float best = -__builtin_inff();
        uint32_t best_u = 0;
        for (uint32_t u = u0 + lane; u < u1; u += 4 * TEAM) {
            float4 f[4];
#pragma unroll
            for (int c = 0; c < 4; c++) f[c] = u + c * TEAM < u1 ? row.load(u + c * TEAM) : none;
            if constexpr (TOP) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float m = max4(f[c]);
                    best_u = m > best ? u + c * TEAM : best_u;
                    best = fmaxf(best, m);
                }
            }
            stat_add(s, f, 4);
        }
        s = stat_wave(s);
        if constexpr (TEAM > 64) {
            __syncthreads();  // the previous row's use of sh
            if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = s;
            __syncthreads();
            if constexpr (TEAM == 256) {
                s = stat_merge(stat_merge(sh.wave[0], sh.wave[1]), stat_merge(sh.wave[2], sh.wave[3]));
            } else {
                s = sh.wave[threadIdx.x & (TEAM / 64 - 1)];
                for (int o = 1; o < TEAM / 64; o <<= 1) s = stat_merge(s, stat_xor(s, o));
            }
        }
        if constexpr (TOP)
            team_top<TEAM>(row, u0, u1, a.top, best > -__builtin_inff() ? lp_key(best, best_u) : 0, sh, lane);
        if constexpr (SPLIT) {
            if (lane == 0) ((LpStat *)a.part)[b] = s;
            if (TOP && lane < a.top) ((uint64_t *)((LpStat *)a.part + total))[b * a.top + lane] = sh.top[lane];
        } else {
            lp_finish<TEAM>(a, r, s, asked, sh.top, lane);
        }
        if constexpr (TOP) team_sync<TEAM>();  // the next row's use of sh.top
    }
}

// Joins a row's parts.
template <bool TOP>
__global__ __launch_bounds__(kLpBlock) void k_logprobs_join(LogProbsArgs a, int split) {
    __shared__ uint64_t buf[TOP ? kLpSplit * kLogProbsTop + 8 : 1];
    __shared__ uint64_t top[kLogProbsTop];
    __shared__ uint64_t bound;
    __shared__ int count;
    for (int64_t r = blockIdx.x; r < a.t; r += gridDim.x) {
        const int lane = threadIdx.x & 63;
        const LpAsked asked(a, r, threadIdx.x == 0);
        LpStat s = {-__builtin_inff(), 0.0f, 0.0f, 0.0f};
        if (lane < split) s = ((const LpStat *)a.part)[r * split + lane];
        constexpr int kKeys = 4;  // read before the bound is known; there are seldom more than 4 a thread
        uint64_t key[kKeys], first = 0;
        const int j = TOP ? (a.top + split - 1) / split : 1;
        const uint64_t *keys = (const uint64_t *)((const LpStat *)a.part + a.t * split) + r * split * a.top;
        if constexpr (TOP) {
            first = lane < split ? keys[lane * a.top + j - 1] : j == 1 ? 0 : ~0ull;
#pragma unroll
            for (int i = 0; i < kKeys; i++)
                key[i] = threadIdx.x + i * kLpBlock < split * a.top ? keys[threadIdx.x + i * kLpBlock] : 0;
        }
        s = stat_wave(s);
        if constexpr (TOP) {
            __syncthreads();  // the previous row's use of the shared arrays
            if (threadIdx.x == 0) count = 0;
            if (threadIdx.x < 64) {
                // k keys of the parts' sorted lists reach the bound: the k-th of the first ones, or every list's j-th
                if (j == 1) {
                    first = wave_kth(first, a.top);
                } else {
                    for (int o = 1; o < 64; o <<= 1) {
                        const uint64_t y = __shfl_xor((unsigned long long)first, o);
                        first = std::min(first, y);
                    }
                }
                if (threadIdx.x == 0) bound = first;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kKeys; i++)
                if (key[i] && key[i] >= bound) buf[atomicAdd(&count, 1)] = key[i];
            for (int c = threadIdx.x + kKeys * kLpBlock; c < split * a.top; c += kLpBlock)
                if (keys[c] && keys[c] >= bound) buf[atomicAdd(&count, 1)] = keys[c];
            __syncthreads();
            rank_keys<kLpBlock>(buf, count, a.top, top, threadIdx.x);
            __syncthreads();
        }
        lp_finish<kLpBlock>(a, r, s, asked, top, threadIdx.x);
        if constexpr (TOP) __syncthreads();
    }
}

// How rows are read, by the time of a call (us, top 5 unless said):
//   up to 1024 logits, or from 512 rows on up to 4096, a wave each (4000x1000 9.9 against 25.2 with a workgroup of 256
//     each, 1000x4000 9.6 against 10.4, but 64x4000 8.7 against 6.8);
//   up to 24576, or from 384 rows on, a workgroup of 256 each (64x10000 7.9 against 9.3 with 1024 threads and 10.5 in
//     parts, 384x30522 16.4 against 22.6 and 20.7, 700x131072 75.6 against 85.0 and 89.1);
//   few rows of more than 32768 in parts, joined by a second launch: about four workgroups a CU over all rows, parts of at
//     least 2048 logits (1x131072 top 20 11.5 against 22.8 with 1024 threads, 64x50001 13.6 against 14.2);
//   the others a workgroup of 1024 each (192x65536 16.6 against 23.3 with 256 and 21.0 in parts, 64x30522 11.3, 12.2, 13.1).
static int lp_team(const LogProbsArgs &a) {
    if (a.v <= 1024 || (a.v <= 4096 && a.t >= 512)) return 64;
    return a.v <= 24576 || a.t >= 384 ? 256 : 1024;
}
static int lp_split(const LogProbsArgs &a) {
    if (a.v <= 32768 || a.t >= 96) return 1;
    return (int)std::min<int64_t>({(1024 + a.t - 1) / a.t, a.v / 2048, kLpSplit});
}

int64_t logprobs_part_bytes(const LogProbsArgs &a) {
    const int split = lp_split(a);
    return split == 1 ? 0 : a.t * split * (int64_t)(sizeof(LpStat) + 8 * a.top);
}

template <int TEAM, bool SPLIT> static void logprobs(const LogProbsArgs &a, int split, hipStream_t s) {
    constexpr int block = std::max(TEAM, kLpBlock), teams = block / TEAM;
    const unsigned grid = (unsigned)std::min<int64_t>((a.t * split + teams - 1) / teams, 1 << 20);
    if (a.top) k_logprobs<TEAM, true, SPLIT><<<grid, block, 0, s>>>(a, split);
    else k_logprobs<TEAM, false, SPLIT><<<grid, block, 0, s>>>(a, split);
}

hipError_t launch_logprobs(const LogProbsArgs &a, hipStream_t s) {
    const int split = lp_split(a);
    if (split > 1) {
        logprobs<256, true>(a, split, s);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        const unsigned rows = (unsigned)std::min<int64_t>(a.t, 1 << 20);
        if (a.top) k_logprobs_join<true><<<rows, kLpBlock, 0, s>>>(a, split);
        else k_logprobs_join<false><<<rows, kLpBlock, 0, s>>>(a, split);
        return hipGetLastError();
    }
    switch (lp_team(a)) {
    case 64: logprobs<64, false>(a, 1, s); break;
    case 256: logprobs<256, false>(a, 1, s); break;
    default: logprobs<1024, false>(a, 1, s); break;
    }
    return hipGetLastError();
}

}  // namespace lx
