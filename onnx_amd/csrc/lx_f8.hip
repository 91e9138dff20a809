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

template <int FA, int FB> static hipError_t matmul_blocks(const MatMulBlocksArgs &p, hipStream_t s) {
    const int64_t tiles = (p.m + 31) / 32 * ((p.n + 31) / 32);
    if (p.b_rows == 1) k_matmul_blocks_small<FA, FB, true><<<(unsigned)tiles, 256, 0, s>>>(p);
    else k_matmul_blocks_small<FA, FB, false><<<(unsigned)tiles, 256, 0, s>>>(p);
    return hipGetLastError();
}

hipError_t launch_matmul_blocks(const MatMulBlocksArgs &p, hipStream_t s) {
    if (p.fmt_a == kFloat8E4M3FN)
        return p.fmt_b == kFloat8E4M3FN ? matmul_blocks<kFloat8E4M3FN, kFloat8E4M3FN>(p, s)
                                        : matmul_blocks<kFloat8E4M3FN, kFloat8E5M2>(p, s);
    return p.fmt_b == kFloat8E4M3FN ? matmul_blocks<kFloat8E5M2, kFloat8E4M3FN>(p, s)
                                    : matmul_blocks<kFloat8E5M2, kFloat8E5M2>(p, s);
}

}  // namespace lx
