// lx_f8.hip -- block-scaled 8-bit floating point on gfx950: QuantizeBlocks (Float to Float8E4M3FN or Float8E5M2
// codes with one Float scale for each block of 128 values) and MatMulBlocks (the product of two such operands).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "lx_device.h"
#include "lx_kernels.h"

namespace lx {

typedef float f8_v4f __attribute__((ext_vector_type(4)));
typedef float f8_v16f __attribute__((ext_vector_type(16)));
typedef __bf16 f8_v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 f8_v8bf __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------
// QuantizeBlocks
// ---------------------------------------------------------------------------
// Block scale s = amax / MAX over the block's finite values (1 where they are all zero, never below the smallest
// normal float), code = the 8-bit value nearest to the exact quotient x / s, ties to even.  v_cvt_pk_fp8_f32 /
// v_cvt_pk_bf8_f32 round a float to nearest even (every value, middle and neighbour of one checked on the device),
// so the float they get has to stand for the exact quotient: a float quotient that was rounded onto the middle of
// two codes would then go to the even one whichever side it came from.  The quotient is therefore rounded to odd:
// a faithful quotient t by one Newton step, the exact sign of x - t s by an fma, t moved toward zero where it is
// above, and its last bit set unless it is exact.  A middle has at most 5 significant bits, far fewer than 24, so
// the value given to the conversion lies on the exact quotient's side of every middle.
template <int FMT> struct F8;
template <> struct F8<kFloat8E4M3FN> {
    static constexpr float kMax = 448.0f;
};
template <> struct F8<kFloat8E5M2> {
    static constexpr float kMax = 57344.0f;
};

struct F8Scale {
    float s;      // the block's scale
    float up;     // 2^64 for tiny scales: x up and s up keep the fma's remainder above the subnormals
    float su, r;  // s up and 1 / (s up)
    float lim;    // |x| beyond this saturates
};

template <int FMT> __device__ __forceinline__ F8Scale f8_scale(float amax) {
    F8Scale c;
    c.s = amax > 0.0f ? fmaxf(amax / F8<FMT>::kMax, 0x1p-126f) : 1.0f;
    c.up = c.s < 0x1p-60f ? 0x1p64f : 1.0f;
    c.su = c.s * c.up;
    c.r = 1.0f / c.su;
    c.lim = amax > 0.0f ? amax : F8<FMT>::kMax;
    return c;
}

// the float whose conversion to FMT is the nearest code to x / s
__device__ __forceinline__ float f8_quotient(float x, const F8Scale &c) {
    const float a = fminf(fabsf(x), c.lim) * c.up;  // NaN: replaced below
    float t = a * c.r;
    t = __builtin_fmaf(__builtin_fmaf(-t, c.su, a), c.r, t);
    const float e = __builtin_fmaf(-t, c.su, a);
    int b = __builtin_bit_cast(int, t);
    b -= e < 0.0f ? 1 : 0;  // t > a / s >= 0, so t is not zero
    b |= e != 0.0f ? 1 : 0;
    const float q = __builtin_copysignf(__builtin_bit_cast(float, b), x);
    return x != x ? x : q;
}

template <int FMT> __device__ __forceinline__ int f8_pack2(float a, float b, int old, bool hi) {
    if constexpr (FMT == kFloat8E4M3FN)
        return hi ? __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, true) : __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, false);
    else
        return hi ? __builtin_amdgcn_cvt_pk_bf8_f32(a, b, old, true) : __builtin_amdgcn_cvt_pk_bf8_f32(a, b, old, false);
}

__device__ __forceinline__ float f8_finite_abs(float x) {
    const float a = fabsf(x);
    return a < __builtin_inff() ? a : 0.0f;  // NaN compares false
}

// Blocks of one row: 32 lanes a block, four values a lane.
template <int FMT, bool VEC>
__global__ __launch_bounds__(256) void k_quantize_rows(const float *__restrict__ x, uint8_t *__restrict__ q,
                                                       float *__restrict__ s, int64_t k, int64_t kb, int64_t blocks) {
    const int lane = threadIdx.x & 31;
    const int64_t step = (int64_t)gridDim.x * 8;
    for (int64_t b = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); b < blocks; b += step) {
        const int64_t row = b / kb, j = b - row * kb;
        const int64_t base = row * k + j * 128;
        const int n = (int)std::min<int64_t>(128, k - j * 128);
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (VEC) {
            if (4 * lane < n) {
                const f8_v4f t = *(const f8_v4f *)(x + base + 4 * lane);
                for (int i = 0; i < 4; i++) v[i] = t[i];
            }
        } else {
            for (int i = 0; i < 4; i++)
                if (lane + 32 * i < n) v[i] = x[base + lane + 32 * i];
        }
        float m = 0.0f;
        for (int i = 0; i < 4; i++) m = fmaxf(m, f8_finite_abs(v[i]));
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 32));
        const F8Scale c = f8_scale<FMT>(m);
        int w = f8_pack2<FMT>(f8_quotient(v[0], c), f8_quotient(v[1], c), 0, false);
        w = f8_pack2<FMT>(f8_quotient(v[2], c), f8_quotient(v[3], c), w, true);
        if constexpr (VEC) {
            if (4 * lane < n) *(int *)(q + base + 4 * lane) = w;
        } else {
            for (int i = 0; i < 4; i++)
                if (lane + 32 * i < n) q[base + lane + 32 * i] = (uint8_t)(w >> (8 * i));
        }
        if (lane == 0) s[b] = c.s;
    }
}

// Blocks of 128 rows: one workgroup a block, the values in registers between the maximum and the codes.
template <int FMT, bool VEC>
__global__ __launch_bounds__(256) void k_quantize_tiles(const float *__restrict__ x, uint8_t *__restrict__ q,
                                                        float *__restrict__ s, int64_t rows, int64_t k, int64_t rb,
                                                        int64_t kb, int64_t blocks) {
    __shared__ float part[4];
    const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
    for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int64_t mat = b / (rb * kb), in = b - mat * rb * kb, i0 = in / kb, j = in - i0 * kb;
        const int64_t base = (mat * rows + i0 * 128) * k + j * 128;
        const int nr = (int)std::min<int64_t>(128, rows - i0 * 128), n = (int)std::min<int64_t>(128, k - j * 128);
        float v[16][4];
        float m = 0.0f;
#pragma unroll
        for (int p = 0; p < 16; p++) {
            const int r = sub + 8 * p;
            for (int i = 0; i < 4; i++) v[p][i] = 0.0f;
            if (r < nr) {
                if constexpr (VEC) {
                    if (4 * lane < n) {
                        const f8_v4f t = *(const f8_v4f *)(x + base + r * k + 4 * lane);
                        for (int i = 0; i < 4; i++) v[p][i] = t[i];
                    }
                } else {
                    for (int i = 0; i < 4; i++)
                        if (lane + 32 * i < n) v[p][i] = x[base + r * k + lane + 32 * i];
                }
            }
            for (int i = 0; i < 4; i++) m = fmaxf(m, f8_finite_abs(v[p][i]));
        }
        for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        __syncthreads();  // the previous block's reads of part
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
        const F8Scale c = f8_scale<FMT>(m);
#pragma unroll
        for (int p = 0; p < 16; p++) {
            const int r = sub + 8 * p;
            if (r >= nr) continue;
            int w = f8_pack2<FMT>(f8_quotient(v[p][0], c), f8_quotient(v[p][1], c), 0, false);
            w = f8_pack2<FMT>(f8_quotient(v[p][2], c), f8_quotient(v[p][3], c), w, true);
            if constexpr (VEC) {
                if (4 * lane < n) *(int *)(q + base + r * k + 4 * lane) = w;
            } else {
                for (int i = 0; i < 4; i++)
                    if (lane + 32 * i < n) q[base + r * k + lane + 32 * i] = (uint8_t)(w >> (8 * i));
            }
        }
        if (threadIdx.x == 0) s[b] = c.s;
    }
}

template <int FMT> static hipError_t quantize(const QuantizeArgs &a, hipStream_t st) {
    const int64_t kb = (a.k + 127) / 128;
    // four values a lane need rows of whole float4s; others go value by value, 32 neighbours at a time
    const bool vec = a.k % 4 == 0 && ((uintptr_t)a.x & 15) == 0 && ((uintptr_t)a.q & 3) == 0;
    if (a.block_rows == 1) {
        const int64_t blocks = a.mats * a.rows * kb;
        const int64_t grid = std::min<int64_t>((blocks + 7) / 8, 1 << 20);
        if (vec) k_quantize_rows<FMT, true><<<(unsigned)grid, 256, 0, st>>>(a.x, a.q, a.s, a.k, kb, blocks);
        else k_quantize_rows<FMT, false><<<(unsigned)grid, 256, 0, st>>>(a.x, a.q, a.s, a.k, kb, blocks);
    } else {
        const int64_t rb = (a.rows + 127) / 128, blocks = a.mats * rb * kb;
        const int64_t grid = std::min<int64_t>(blocks, 1 << 20);
        if (vec) k_quantize_tiles<FMT, true><<<(unsigned)grid, 256, 0, st>>>(a.x, a.q, a.s, a.rows, a.k, rb, kb, blocks);
        else k_quantize_tiles<FMT, false><<<(unsigned)grid, 256, 0, st>>>(a.x, a.q, a.s, a.rows, a.k, rb, kb, blocks);
    }
    return hipGetLastError();
}

hipError_t launch_quantize_blocks(const QuantizeArgs &a, hipStream_t s) {
    return a.fmt == kFloat8E4M3FN ? quantize<kFloat8E4M3FN>(a, s) : quantize<kFloat8E5M2>(a, s);
}

// ---------------------------------------------------------------------------
// MatMulBlocks
// ---------------------------------------------------------------------------
// Y[m][n] = sum over the blocks j of K of sa[m][j] sb[n][j] (sum over k in block j of A[m][k] B[n][k]) + bias[n].
// The codes' products run on the bf16 matrix unit: both 8-bit types convert exactly to bf16 and the products are
// exact in float, so only the float sums round.  (The 8-bit matrix instructions of gfx950 keep fewer bits of the
// products they add: 1.5e-5 of the result's norm over 128 products of normal values, against 1e-7.)
template <int FMT> __device__ __forceinline__ f8_v2bf f8_bf16x2(unsigned v, bool hi) {
    if constexpr (FMT == kFloat8E4M3FN)
        return hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v, 1.0f, false);
    else
        return hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v, 1.0f, true)
                  : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(v, 1.0f, false);
}

// eight codes to eight bf16
template <int FMT> __device__ __forceinline__ f8_v8bf f8_bf16x8(unsigned lo, unsigned hi) {
    f8_v8bf r;
    const f8_v2bf a = f8_bf16x2<FMT>(lo, false), b = f8_bf16x2<FMT>(lo, true);
    const f8_v2bf c = f8_bf16x2<FMT>(hi, false), d = f8_bf16x2<FMT>(hi, true);
    r[0] = a[0]; r[1] = a[1]; r[2] = b[0]; r[3] = b[1];
    r[4] = c[0]; r[5] = c[1]; r[6] = d[0]; r[7] = d[1];
    return r;
}

// 16 codes of a row from column c on, zeros (a code of value zero) past the row's end
__device__ __forceinline__ uint4 f8_load16(const uint8_t *row, int64_t c, int64_t k) {
    uint4 v = {0, 0, 0, 0};
    if (c + 16 <= k) {
        __builtin_memcpy(&v, row + c, 16);
    } else {
        unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (c + i < k) w[i / 4] |= (unsigned)row[c + i] << (8 * (i % 4));
        v = {w[0], w[1], w[2], w[3]};
    }
    return v;
}

// One 32x32 tile of Y a workgroup, its four waves over every fourth block of K, their sums added in order.
template <int FA, int FB, bool BROWS>
__global__ __launch_bounds__(256) void k_matmul_blocks_small(MatMulBlocksArgs p) {
    __shared__ f8_v16f part[3][64];
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;
    const int64_t tiles_n = (p.n + 31) / 32;
    const int64_t m0 = blockIdx.x / tiles_n * 32, n0 = blockIdx.x % tiles_n * 32;
    const int64_t kb = (p.k + 127) / 128;
    const int64_t m = std::min<int64_t>(m0 + (l & 31), p.m - 1), n = std::min<int64_t>(n0 + (l & 31), p.n - 1);
    const uint8_t *ar = p.a + m * p.k, *br = p.b + n * p.k;
    f8_v16f acc = {};
    for (int64_t j = w; j < kb; j += 4) {
        f8_v16f t = {};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t c = j * 128 + i * 32 + h * 16;
            const uint4 va = f8_load16(ar, c, p.k), vb = f8_load16(br, c, p.k);
            t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f8_bf16x8<FB>(vb.x, vb.y), f8_bf16x8<FA>(va.x, va.y), t, 0, 0, 0);
            t = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f8_bf16x8<FB>(vb.z, vb.w), f8_bf16x8<FA>(va.z, va.w), t, 0, 0, 0);
        }
        const float sa = p.sa[m * kb + j];
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const int64_t nr = std::min<int64_t>(n0 + 8 * (r / 4) + 4 * h + r % 4, p.n - 1);
            const float sb = p.sb[(BROWS ? nr : nr / 128) * kb + j];
            acc[r] = __builtin_fmaf(t[r], sa * sb, acc[r]);
        }
    }
    if (w) part[w - 1][l] = acc;
    __syncthreads();
    if (w || m0 + (l & 31) >= p.m) return;
    for (int i = 0; i < 3; i++) acc += part[i][l];
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int64_t nr = n0 + 8 * (r / 4) + 4 * h + r % 4;
        if (nr < p.n) p.y[m * p.n + nr] = p.bias ? acc[r] + p.bias[nr] : acc[r];
    }
}

// ---- tiles of Y through LDS -------------------------------------------------------------------------------------
// A workgroup computes BM x BN of Y (BM = 32 TM WM rows, BN = 32 TN WN columns); each of its WM x WN waves TM x TN
// tiles of 32x32.  A stage of LDS holds one block of K: BM rows of A and BN rows of B, 128 codes each, and their
// scales; S stages are filled by direct-to-LDS loads S - 1 blocks ahead, with one barrier a block.  The codes stay 8
// bits in LDS (half the traffic of bf16) and are converted as a wave reads them.  Row r's 16-byte chunk c lies at
// slot c ^ ((r >> 1) & 7): the 32 rows a fragment read touches then spread over all banks.
// Operands need rows of whole 16-byte chunks (k a multiple of 16, aligned storage) and tiles within 2^31 bytes.
__device__ __forceinline__ uint32_t f8_lds(const void *p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p;
}
// The lane's 16 (4) bytes at base + off land in LDS at lds + 16 (4) * lane; lds is uniform over the wave.  Inline asm
// so that the compiler does not make LDS reads of other stages wait for them; the kernel waits itself.
__device__ __forceinline__ void f8_load_lds16(const void *base, uint32_t off, void *lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(f8_lds(lds)), "v"(off), "s"(base) : "memory");
#endif
}
__device__ __forceinline__ void f8_load_lds4(const void *base, uint32_t off, void *lds) {
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("s_nop 0\n\tglobal_load_lds_dword %1, %2" ::"{m0}"(f8_lds(lds)), "v"(off), "s"(base) : "memory");
#endif
}
// All but this wave's last N direct loads have landed and its LDS operations are done, then the workgroup's barrier.
template <int N> __device__ __forceinline__ void f8_wait_barrier() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("s_barrier" ::: "memory");
#endif
}

template <int FA, int FB, bool BROWS, int TM, int TN, int WM, int WN, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_matmul_blocks(MatMulBlocksArgs p, int tm, int tn) {
    constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, R = BM + BN;
    constexpr int L = R / 8 / NW;               // 16-byte loads a wave and stage, of eight rows each
    constexpr int LS = (R / 64 + NW - 1) / NW;  // 4-byte loads of the rows' scales
    static_assert(R % (8 * NW) == 0 && R % 64 == 0 && BM % 8 == 0 && BN <= 128, "whole wave loads");
    constexpr int STAGE = R * 128 + LS * NW * 256;
    __shared__ __attribute__((aligned(1024))) char sm[S][STAGE];
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;

    // tiles in groups of eight rows of tiles, contiguous ranges of them to each XCD (workgroups go round the 8 XCDs)
    const int tiles = tm * tn, per = (tiles + 7) / 8;
    const int t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || t >= tiles) return;
    const int group = t / (8 * tn), first = 8 * group, gs = min(tm - first, 8), in = t - group * 8 * tn;
    const int m0 = (first + in % gs) * BM, n0 = in / gs * BN;

    const int64_t kb = (p.k + 127) / 128;
    const uint8_t *abase = p.a + m0 * p.k, *bbase = p.b + n0 * p.k;
    const int row_n = BROWS ? 1 : 128;
    const float *sabase = p.sa + m0 * kb, *sbbase = p.sb + n0 / row_n * kb;
    uint32_t off[L], soff[LS];
#pragma unroll
    for (int i = 0; i < L; i++) {
        const int r = 8 * (w + NW * i) + (l >> 3), c = (l & 7) ^ ((r >> 1) & 7);
        const int row = r < BM ? min(r, (int)p.m - 1 - m0) : min(r - BM, (int)p.n - 1 - n0);
        off[i] = (uint32_t)(row * (int)p.k + 16 * c);
    }
#pragma unroll
    for (int i = 0; i < LS; i++) {
        const int r = min(64 * (w + NW * i) + l, R - 1);
        const int row = r < BM ? min(r, (int)p.m - 1 - m0) : min(r - BM, (int)p.n - 1 - n0) / row_n;
        soff[i] = (uint32_t)(row * (int)kb * 4);
    }
    const int tail = (int)(p.k & 127);  // codes of a last block that is not whole
    auto load = [&](int64_t j, char *st) {
        const bool cut = tail && j == kb - 1;
#pragma unroll
        for (int i = 0; i < L; i++) {
            const bool is_a = 8 * (w + NW * i) < BM;  // uniform: eight rows are all A's or all B's
            const uint8_t *base = (is_a ? abase : bbase) + 128 * j;
            char *lds = st + 1024 * (w + NW * i);
            if (!cut) {
                f8_load_lds16(base, off[i], lds);
            } else {
                const int r = 8 * (w + NW * i) + (l >> 3), c = (l & 7) ^ ((r >> 1) & 7);
                if (16 * c < tail) f8_load_lds16(base, off[i], lds);
                else *(uint4 *)(lds + 16 * l) = uint4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int i = 0; i < LS; i++) {
            const bool is_a = 64 * (w + NW * i) < BM;
            f8_load_lds4((is_a ? sabase : sbbase) + j, soff[i], st + R * 128 + 256 * (w + NW * i));
        }
    };

    f8_v16f acc[TN][TM] = {};
    const int wm = w % WM, wn = w / WM;
    const int swz = ((l & 31) >> 1) & 7;
    for (int s = 0; s < S - 1; s++)
        if (s < kb) load(s, sm[s]);
    int cur = 0;
    for (int64_t j = 0; j < kb; j++) {
        // the last S - 2 stages ahead may still be landing; near the end there are fewer
        if (S > 2 && j + S - 2 < kb) f8_wait_barrier<(S - 2) * (L + LS)>();
        else f8_wait_barrier<0>();
        const char *st = sm[cur];
        if (j + S - 1 < kb) load(j + S - 1, sm[cur == 0 ? S - 1 : cur - 1]);
        cur = cur + 1 == S ? 0 : cur + 1;
        const char *ap = st + (wm * TM * 32 + (l & 31)) * 128, *bp = st + (BM + wn * TN * 32 + (l & 31)) * 128;
        f8_v16f part[TN][TM] = {};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint4 va[TM], vb[TN];
            const int slot = 16 * ((2 * c + h) ^ swz);
#pragma unroll
            for (int i = 0; i < TM; i++) va[i] = *(const uint4 *)(ap + i * 32 * 128 + slot);
#pragma unroll
            for (int i = 0; i < TN; i++) vb[i] = *(const uint4 *)(bp + i * 32 * 128 + slot);
#pragma unroll
            for (int z = 0; z < 2; z++) {
                f8_v8bf a[TM], b[TN];
#pragma unroll
                for (int i = 0; i < TM; i++) a[i] = z ? f8_bf16x8<FA>(va[i].z, va[i].w) : f8_bf16x8<FA>(va[i].x, va[i].y);
#pragma unroll
                for (int i = 0; i < TN; i++) b[i] = z ? f8_bf16x8<FB>(vb[i].z, vb[i].w) : f8_bf16x8<FB>(vb[i].x, vb[i].y);
#pragma unroll
                for (int in_ = 0; in_ < TN; in_++)
#pragma unroll
                    for (int im = 0; im < TM; im++)
                        part[in_][im] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[in_], a[im], part[in_][im], 0, 0, 0);
            }
        }
        const float *sc = (const float *)(st + R * 128);
        float sa[TM];
#pragma unroll
        for (int i = 0; i < TM; i++) sa[i] = sc[(wm * TM + i) * 32 + (l & 31)];
#pragma unroll
        for (int in_ = 0; in_ < TN; in_++) {
            const float *sb = sc + BM + (wn * TN + in_) * 32 + 4 * h;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                f8_v4f b4;
                if constexpr (BROWS) b4 = *(const f8_v4f *)(sb + 8 * q);
#pragma unroll
                for (int im = 0; im < TM; im++) {
                    const float one = sa[im] * sc[BM + wn * TN * 32];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float f = BROWS ? sa[im] * b4[e] : one;
                        acc[in_][im][4 * q + e] = __builtin_fmaf(part[in_][im][4 * q + e], f, acc[in_][im][4 * q + e]);
                    }
                }
            }
        }
    }
    const bool vec = p.n % 4 == 0 && ((uintptr_t)p.y & 15) == 0;
#pragma unroll
    for (int im = 0; im < TM; im++) {
        const int64_t m = m0 + (wm * TM + im) * 32 + (l & 31);
        if (m >= p.m) continue;
#pragma unroll
        for (int in_ = 0; in_ < TN; in_++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int64_t n = n0 + (wn * TN + in_) * 32 + 8 * q + 4 * h;
                f8_v4f v;
                for (int e = 0; e < 4; e++) v[e] = acc[in_][im][4 * q + e];
                if (vec) {
                    if (n < p.n) {
                        if (p.bias)
                            for (int e = 0; e < 4; e++) v[e] += p.bias[n + e];
                        *(f8_v4f *)(p.y + m * p.n + n) = v;
                    }
                } else {
                    for (int e = 0; e < 4; e++)
                        if (n + e < p.n) p.y[m * p.n + n + e] = p.bias ? v[e] + p.bias[n + e] : v[e];
                }
            }
    }
}

template <int FA, int FB, bool BROWS> static hipError_t matmul_blocks(const MatMulBlocksArgs &p, hipStream_t s) {
    const bool chunks = p.k % 16 == 0 && p.k > 0 && (((uintptr_t)p.a | (uintptr_t)p.b) & 15) == 0 && p.k < (1 << 23);
    const int64_t t128 = (p.m + 127) / 128 * ((p.n + 127) / 128), t64 = (p.m + 63) / 64 * ((p.n + 63) / 64);
    if (chunks && t128 >= 256 && t128 < (1 << 26)) {
        k_matmul_blocks<FA, FB, BROWS, 2, 2, 2, 2, 2, 2>
            <<<(unsigned)((t128 + 7) / 8 * 8), 256, 0, s>>>(p, (int)((p.m + 127) / 128), (int)((p.n + 127) / 128));
    } else if (chunks && p.m > 32 && t64 >= 256 && t64 < (1 << 26)) {
        k_matmul_blocks<FA, FB, BROWS, 1, 1, 2, 2, 3, 3>
            <<<(unsigned)((t64 + 7) / 8 * 8), 256, 0, s>>>(p, (int)((p.m + 63) / 64), (int)((p.n + 63) / 64));
    } else {
        const int64_t tiles = (p.m + 31) / 32 * ((p.n + 31) / 32);
        k_matmul_blocks_small<FA, FB, BROWS><<<(unsigned)tiles, 256, 0, s>>>(p);
    }
    return hipGetLastError();
}

template <int FA, int FB> static hipError_t matmul_blocks(const MatMulBlocksArgs &p, hipStream_t s) {
    return p.b_rows == 1 ? matmul_blocks<FA, FB, true>(p, s) : matmul_blocks<FA, FB, false>(p, s);
}

hipError_t launch_matmul_blocks(const MatMulBlocksArgs &p, hipStream_t s) {
    if (p.fmt_a == kFloat8E4M3FN)
        return p.fmt_b == kFloat8E4M3FN ? matmul_blocks<kFloat8E4M3FN, kFloat8E4M3FN>(p, s)
                                        : matmul_blocks<kFloat8E4M3FN, kFloat8E5M2>(p, s);
    return p.fmt_b == kFloat8E4M3FN ? matmul_blocks<kFloat8E5M2, kFloat8E4M3FN>(p, s)
                                    : matmul_blocks<kFloat8E5M2, kFloat8E5M2>(p, s);
}

}  // namespace lx
