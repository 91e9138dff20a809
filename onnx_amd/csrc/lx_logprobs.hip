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
// it).  Only threads whose own largest reaches the bound read their logits again, and only logits that reach it
// are ranked, by counting; equal logits rank by index.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lx_device.h"
#include "lx_kernels.h"

namespace lx {

constexpr int kLpBlock = 256, kLpCap = 2048, kLpSplit = 64;

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

__device__ __forceinline__ LpStat stat_wave(LpStat s) {
    for (int o = 1; o < 64; o <<= 1) {
        const LpStat b = {__shfl_xor(s.m, o), __shfl_xor(s.r, o), __shfl_xor(s.t, o), __shfl_xor(s.n, o)};
        s = stat_merge(s, b);
    }
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

// The k largest of `count` distinct keys into out, largest first (all threads of the block; count <= what buf holds).
__device__ __forceinline__ void rank_keys(const uint64_t *buf, int count, int k, uint64_t *out) {
    for (int c = threadIdx.x; c < count; c += kLpBlock) {
        const uint64_t mine = buf[c];
        int rank = 0;
        for (int j = 0; j < count && rank < k; j++) rank += buf[j] > mine;
        if (rank < k) out[rank] = mine;
    }
}

struct LpShared {
    uint64_t buf[kLpCap];
    uint64_t group[kLpBlock];
    uint64_t top[kLogProbsTop];
    LpStat wave[4];
    uint64_t bound;
    int count;
};

// the k-th largest of the wave's 64 keys, distinct but for zeros (none): zero if fewer than k are there
__device__ __forceinline__ uint64_t wave_kth(uint64_t g, int k) {
    int rank = 0;
    for (int j = 0; j < 64; j++) {
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)g, j), hi = __builtin_amdgcn_readlane((int)(g >> 32), j);
        rank += ((uint64_t)hi << 32 | lo) > g;
    }
    const uint64_t at = __ballot(g != 0 && rank == k - 1);
    if (!at) return 0;
    const int j = __builtin_ctzll(at);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)g, j), hi = __builtin_amdgcn_readlane((int)(g >> 32), j);
    return (uint64_t)hi << 32 | lo;
}

// sh.top[0 .. k) = the k largest keys of units [u0, u1) of the row, zeros where there are fewer; `best` is this
// thread's largest unit (value, unit), zero if none.
__device__ void block_top(const LpRow &row, uint32_t u0, uint32_t u1, int k, uint64_t best, LpShared &sh) {
    sh.group[threadIdx.x] = best;
    if (threadIdx.x < kLogProbsTop) sh.top[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    if (threadIdx.x < 64) {
        uint64_t g = 0;
        for (int w = 0; w < kLpBlock / 64; w++) g = std::max(g, sh.group[64 * w + threadIdx.x]);
        g = wave_kth(g, k);
        if (threadIdx.x == 0) sh.bound = g;
    }
    __syncthreads();
    const uint64_t bound = sh.bound;
    const bool search = best >= bound;
    if (search) {
        for (uint32_t u = u0 + threadIdx.x; u < u1; u += kLpBlock) {
            const float4 f = row.load(u);
            const float *p = &f.x;
            for (int i = 0; i < 4; i++)
                if (lp_key(p[i], u) >= bound && row.inside(u, i)) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < kLpCap) sh.buf[at] = lp_key(p[i], 4 * u - row.off + i);
                }
        }
    }
    __syncthreads();
    int count = sh.count;
    if (count <= kLpCap) {
        rank_keys(sh.buf, count, k, sh.top);
        __syncthreads();
        return;
    }
    // more than the buffer holds (few distinct logits, or sorted ones): by rounds, the k largest so far kept
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    for (uint32_t u = u0; u < u1; u += kLpBlock) {
        if (search && u + threadIdx.x < u1) {
            const float4 f = row.load(u + threadIdx.x);
            const float *p = &f.x;
            const uint64_t least = sh.top[k - 1];
            for (int i = 0; i < 4; i++) {
                const uint64_t key = lp_key(p[i], 4 * (u + threadIdx.x) - row.off + i);
                if (lp_key(p[i], u + threadIdx.x) >= bound && row.inside(u + threadIdx.x, i) && key > least)
                    sh.buf[atomicAdd(&sh.count, 1)] = key;
            }
        }
        __syncthreads();
        count = sh.count;
        // room for the next round's 4 * kLpBlock keys, or the last round
        if (count > kLpCap - 4 * kLpBlock - kLogProbsTop || u + kLpBlock >= u1) {
            if (threadIdx.x < k && sh.top[threadIdx.x]) sh.buf[count + threadIdx.x] = sh.top[threadIdx.x];
            __syncthreads();
            int kept = 0;
            while (kept < k && sh.top[kept]) kept++;
            __syncthreads();
            rank_keys(sh.buf, count + kept, k, sh.top);
            if (threadIdx.x == 0) sh.count = 0;
        }
        __syncthreads();
    }
}

// a row's outputs from its sums and sorted keys
__device__ __forceinline__ void lp_finish(const LogProbsArgs &a, int64_t row, const LpStat &s, const uint64_t *top) {
    const float ls = s.n > 0.0f ? log1pf((s.n - 1.0f) + s.r) : __builtin_nanf("");
    if (threadIdx.x == 0) {
        if (a.ids) {
            const int64_t id = a.ids_dtype == kInt64 ? ((const int64_t *)a.ids)[row] : (int64_t)((const int32_t *)a.ids)[row];
            float lp = 0.0f;
            if (id >= a.v) lp = __builtin_nanf("");
            else if (id >= 0) lp = (a.x[row * a.v + id] - s.m) - ls;
            a.lp[row] = lp;
        }
        if (a.h) a.h[row] = ls + s.t / (s.n + s.r);
    }
    if (threadIdx.x < a.top) {
        const uint64_t key = top[threadIdx.x];
        a.top_ids[row * a.top + threadIdx.x] = (int64_t)(uint32_t)~(uint32_t)key;
        a.top_lp[row * a.top + threadIdx.x] = (lp_value((uint32_t)(key >> 32)) - s.m) - ls;
    }
}

// One workgroup a part of a row (SPLIT: kLpSplit parts at most, their sums and keys to a.part) or a whole row.
template <bool TOP, bool SPLIT>
__global__ __launch_bounds__(kLpBlock) void k_logprobs(LogProbsArgs a, int split) {
    __shared__ LpShared sh;
    const int64_t total = a.t * split;
    for (int64_t b = blockIdx.x; b < total; b += gridDim.x) {
        const int64_t r = SPLIT ? b / split : b;
        const int part = SPLIT ? (int)(b - r * split) : 0;
        const LpRow row(a.x + r * a.v, a.v);
        const uint32_t per = SPLIT ? (uint32_t)(((a.v + 6) / 4 + split - 1) / split) : row.units;
        const uint32_t u0 = std::min(row.units, part * per), u1 = std::min(row.units, u0 + per);
        const float4 none = {-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff()};
        LpStat s = {-__builtin_inff(), 0.0f, 0.0f, 0.0f};
        float best = -__builtin_inff();
        uint32_t best_u = 0;
        for (uint32_t u = u0 + threadIdx.x; u < u1; u += 4 * kLpBlock) {
            float4 f[4];
#pragma unroll
            for (int c = 0; c < 4; c++) f[c] = u + c * kLpBlock < u1 ? row.load(u + c * kLpBlock) : none;
            if constexpr (TOP) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float m = max4(f[c]);
                    best_u = m > best ? u + c * kLpBlock : best_u;
                    best = fmaxf(best, m);
                }
            }
            stat_add(s, f, 4);
        }
        s = stat_wave(s);
        __syncthreads();  // the previous row's use of sh
        if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = s;
        __syncthreads();
        s = stat_merge(stat_merge(sh.wave[0], sh.wave[1]), stat_merge(sh.wave[2], sh.wave[3]));
        if constexpr (TOP)
            block_top(row, u0, u1, a.top, best > -__builtin_inff() ? lp_key(best, best_u) : 0, sh);
        if constexpr (SPLIT) {
            if (threadIdx.x == 0) ((LpStat *)a.part)[b] = s;
            if (TOP && threadIdx.x < a.top) ((uint64_t *)((LpStat *)a.part + total))[b * a.top + threadIdx.x] = sh.top[threadIdx.x];
        } else {
            lp_finish(a, r, s, sh.top);
        }
    }
}

// Joins a row's parts.
template <bool TOP>
__global__ __launch_bounds__(kLpBlock) void k_logprobs_join(LogProbsArgs a, int split) {
    __shared__ uint64_t buf[TOP ? kLpSplit * kLogProbsTop : 1];
    __shared__ uint64_t top[kLogProbsTop];
    __shared__ uint64_t bound;
    __shared__ int count;
    for (int64_t r = blockIdx.x; r < a.t; r += gridDim.x) {
        const int lane = threadIdx.x & 63;
        LpStat s = {-__builtin_inff(), 0.0f, 0.0f, 0.0f};
        if (lane < split) s = ((const LpStat *)a.part)[r * split + lane];
        s = stat_wave(s);
        if constexpr (TOP) {
            const uint64_t *keys = (const uint64_t *)((const LpStat *)a.part + a.t * split) + r * split * a.top;
            __syncthreads();  // the previous row's use of the shared arrays
            if (threadIdx.x == 0) count = 0;
            if (threadIdx.x < 64) {
                // k keys of the parts' sorted lists reach the bound: the k-th of the first ones, or every list's j-th
                const int j = (a.top + split - 1) / split;
                uint64_t g = lane < split ? keys[lane * a.top + j - 1] : j == 1 ? 0 : ~0ull;
                if (j == 1) {
                    g = wave_kth(g, a.top);
                } else {
                    for (int o = 1; o < 64; o <<= 1) {
                        const uint64_t y = __shfl_xor((unsigned long long)g, o);
                        g = std::min(g, y);
                    }
                }
                if (threadIdx.x == 0) bound = g;
            }
            __syncthreads();
            for (int c = threadIdx.x; c < split * a.top; c += kLpBlock) {
                const uint64_t key = keys[c];
                if (key && key >= bound) buf[atomicAdd(&count, 1)] = key;
            }
            __syncthreads();
            rank_keys(buf, count, a.top, top);
            __syncthreads();
        }
        lp_finish(a, r, s, top);
    }
}

// Parts of a row: about four workgroups a CU over all rows, parts of at least 2048 logits, at most kLpSplit.
static int lp_split(const LogProbsArgs &a) {
    const int64_t want = (1024 + a.t - 1) / a.t, most = a.v / 2048;
    return (int)std::max<int64_t>(1, std::min<int64_t>({want, most, kLpSplit}));
}

int64_t logprobs_part_bytes(const LogProbsArgs &a) {
    const int split = lp_split(a);
    return split == 1 ? 0 : a.t * split * (int64_t)(sizeof(LpStat) + 8 * a.top);
}

hipError_t launch_logprobs(const LogProbsArgs &a, hipStream_t s) {
    const int split = lp_split(a);
    const unsigned grid = (unsigned)std::min<int64_t>(a.t * split, 1 << 20);
    if (split == 1) {
        if (a.top) k_logprobs<true, false><<<grid, kLpBlock, 0, s>>>(a, 1);
        else k_logprobs<false, false><<<grid, kLpBlock, 0, s>>>(a, 1);
        return hipGetLastError();
    }
    if (a.top) k_logprobs<true, true><<<grid, kLpBlock, 0, s>>>(a, split);
    else k_logprobs<false, true><<<grid, kLpBlock, 0, s>>>(a, split);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const unsigned rows = (unsigned)std::min<int64_t>(a.t, 1 << 20);
    if (a.top) k_logprobs_join<true><<<rows, kLpBlock, 0, s>>>(a, split);
    else k_logprobs_join<false><<<rows, kLpBlock, 0, s>>>(a, split);
    return hipGetLastError();
}

}  // namespace lx
