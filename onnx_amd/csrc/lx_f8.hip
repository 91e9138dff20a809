// lx_f8.hip -- block-scaled 8-bit floating point on gfx950: QuantizeBlocks (Float to Float8E4M3FN or Float8E5M2
// codes with one Float scale for each block of 128 values) and MatMulBlocks (the product of two such operands).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

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

// Blocks of one row: 32 lanes a block, four values a lane, U blocks at once (their loads and reductions overlap).
// Bound by memory: [16384, 2048] 33.4 us, 5.0 TB/s, the rate of a large copy (one block at once: 42.7).
template <int FMT, bool VEC, int U>
__global__ __launch_bounds__(256) void k_quantize_rows(const float *__restrict__ x, uint8_t *__restrict__ q,
                                                       float *__restrict__ s, int64_t k, FastDiv kb, uint32_t blocks) {
    const int lane = threadIdx.x & 31;
    const uint32_t b0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * U;
    int64_t base[U];
    int n[U];
    float v[U][4];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t row = fdiv(b0 + u, kb), j = b0 + u - row * kb.d;
        base[u] = row * k + j * 128;
        n[u] = b0 + u < blocks ? (int)std::min<int64_t>(128, k - (int64_t)j * 128) : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) v[u][i] = 0.0f;
        if constexpr (VEC) {
            if (4 * lane < n[u]) {
                const f8_v4f t = *(const f8_v4f *)(x + base[u] + 4 * lane);
                for (int i = 0; i < 4; i++) v[u][i] = t[i];
            }
        } else {
            for (int i = 0; i < 4; i++)
                if (lane + 32 * i < n[u]) v[u][i] = x[base[u] + lane + 32 * i];
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        float m = 0.0f;
        for (int i = 0; i < 4; i++) m = fmaxf(m, f8_finite_abs(v[u][i]));
        m = group_reduce<32>(m, [](float a, float b) { return fmaxf(a, b); });
        const F8Scale c = f8_scale<FMT>(m);
        int w = f8_pack2<FMT>(f8_quotient(v[u][0], c), f8_quotient(v[u][1], c), 0, false);
        w = f8_pack2<FMT>(f8_quotient(v[u][2], c), f8_quotient(v[u][3], c), w, true);
        if constexpr (VEC) {
            if (4 * lane < n[u]) *(int *)(q + base[u] + 4 * lane) = w;
        } else {
            for (int i = 0; i < 4; i++)
                if (lane + 32 * i < n[u]) q[base[u] + lane + 32 * i] = (uint8_t)(w >> (8 * i));
        }
        if (lane == 0 && n[u]) s[b0 + u] = c.s;
    }
}

// Blocks of 128 rows: one workgroup a block, the values in registers between the maximum and the codes.  512 threads
// ([30522, 768] 26.6 us, 4.4 TB/s, and [512, 768] 5.2) keep more of a CU's loads in flight than 1024 (33.7, 5.3) and
// reach the maximum sooner than 256 (28.5, 6.8).
constexpr int kTileThreads = 512;
template <int FMT, bool VEC>
__global__ __launch_bounds__(kTileThreads) void k_quantize_tiles(const float *__restrict__ x, uint8_t *__restrict__ q,
                                                        float *__restrict__ s, int64_t rows, int64_t k, int64_t rb,
                                                        int64_t kb, int64_t blocks) {
    constexpr int P = 4096 / kTileThreads, ROWS = kTileThreads / 32;
    __shared__ float part[kTileThreads / 64];
    const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
    for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x) {
        const int64_t mat = b / (rb * kb), in = b - mat * rb * kb, i0 = in / kb, j = in - i0 * kb;
        const int64_t base = (mat * rows + i0 * 128) * k + j * 128;
        const int nr = (int)std::min<int64_t>(128, rows - i0 * 128), n = (int)std::min<int64_t>(128, k - j * 128);
        float v[P][4];
        float m = 0.0f;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const int r = sub + ROWS * p;
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
        m = wave_reduce_dpp(m, [](float a, float b) { return fmaxf(a, b); });
        __syncthreads();  // the previous block's reads of part
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
        __syncthreads();
        m = part[0];
#pragma unroll
        for (int w = 1; w < kTileThreads / 64; w++) m = fmaxf(m, part[w]);
        const F8Scale c = f8_scale<FMT>(m);
#pragma unroll
        for (int p = 0; p < P; p++) {
            const int r = sub + ROWS * p;
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
        // in row ranges of at most 2^28 blocks (a launch takes fewer than 2^32 threads)
        const int64_t rows = a.mats * a.rows, most = std::max<int64_t>(1, ((int64_t)1 << 28) / kb);
        for (int64_t r = 0; r < rows; r += most) {
            const uint32_t blocks = (uint32_t)(std::min(most, rows - r) * kb);
            const float *x = a.x + r * a.k;
            uint8_t *q = a.q + r * a.k;
            float *s = a.s + r * kb;
            const FastDiv d = make_fastdiv((uint32_t)kb);
            const unsigned g4 = (blocks + 31) / 32, g1 = (blocks + 7) / 8;
            // four blocks at once where that still gives every CU a workgroup
            if (g4 >= 256) {
                if (vec) k_quantize_rows<FMT, true, 4><<<g4, 256, 0, st>>>(x, q, s, a.k, d, blocks);
                else k_quantize_rows<FMT, false, 4><<<g4, 256, 0, st>>>(x, q, s, a.k, d, blocks);
            } else {
                if (vec) k_quantize_rows<FMT, true, 1><<<g1, 256, 0, st>>>(x, q, s, a.k, d, blocks);
                else k_quantize_rows<FMT, false, 1><<<g1, 256, 0, st>>>(x, q, s, a.k, d, blocks);
            }
        }
    } else {
        const int64_t rb = (a.rows + 127) / 128, blocks = a.mats * rb * kb;
        const int64_t grid = std::min<int64_t>(blocks, 1 << 20);
        if (vec) k_quantize_tiles<FMT, true><<<(unsigned)grid, kTileThreads, 0, st>>>(a.x, a.q, a.s, a.rows, a.k, rb, kb, blocks);
        else k_quantize_tiles<FMT, false><<<(unsigned)grid, kTileThreads, 0, st>>>(a.x, a.q, a.s, a.rows, a.k, rb, kb, blocks);
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

// 16 codes of a row of k from column c on, as they lie in memory: the 16 that end with the row where fewer are left
// (f8_tail16 moves them down), none from a column past it.  No byte outside the row is read.
__device__ __forceinline__ uint4 f8_load16(const uint8_t *row, int c, int k) {
    uint4 v = {0, 0, 0, 0};
    if (k < 16) {
        uint64_t b[2] = {0, 0};
        for (int i = c; i < k; i++) b[(i - c) / 8] |= (uint64_t)row[i] << (8 * ((i - c) & 7));
        v = uint4{(unsigned)b[0], (unsigned)(b[0] >> 32), (unsigned)b[1], (unsigned)(b[1] >> 32)};
    } else if (c < k) {
        __builtin_memcpy(&v, row + min(c, k - 16), 16);
    }
    return v;
}
// what f8_load16 read for column c with the codes before c dropped and zeros (codes of value zero) past the row's end
__device__ __forceinline__ uint4 f8_tail16(uint4 v, int c, int k) {
    const int sh = c - (k - 16);
    if (k < 16 || sh <= 0 || sh >= 16) return v;
    uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
    if (sh >= 8) {
        lo = hi;
        hi = 0;
    }
    const int bits = 8 * (sh & 7);
    if (bits) lo = lo >> bits | hi << (64 - bits);
    hi >>= bits;
    return uint4{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
}

// ---- tiles of Y through LDS -------------------------------------------------------------------------------------
// A workgroup computes BM x BN of Y (BM = 32 TM WM rows, BN = 32 TN WN columns); each of its WM x WN waves TM x TN
// tiles of 32x32.  A stage of LDS holds one block of K: BM rows of A and BN rows of B, 128 codes each, and their
// scales; S stages are filled by direct-to-LDS loads S - 1 blocks ahead, with one barrier a block.  The codes stay 8
// bits in LDS (half the traffic of bf16) and are converted as a wave reads them.  Row r's 16-byte chunk c lies at
// slot c ^ ((r >> 1) & 7): the 32 rows a fragment read touches then spread over all banks.
// Operands need rows of whole 16-byte chunks (k a multiple of 16, aligned storage) and tiles within 2^31 bytes.
// 8192x4096x8192: 474 us, 1.16 PFLOP/s, where the library's bf16 product of 8192^3 reaches 1.25.  The matrix unit is busy
// in 57% of the cycles; each of its instructions (32 cycles) comes with four conversions and two scalings (24), and
// under this load the clock falls to 1.6 to 1.9 GHz: fewer cycles no longer mean as much less time.
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

// A wave's own waits: all but its last N direct loads, and its LDS operations, are done; nothing that touches memory
// moves across.
template <int N> __device__ __forceinline__ void f8_wait() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
#endif
}
__device__ __forceinline__ void f8_wait_lds() {
#if defined(__HIP_DEVICE_COMPILE__)
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#endif
}

// A block of K for a wave's TM x TN tiles of 32x32 is read in four chunks of 32 codes a row (the lane's 16 bytes of
// chunk c are k = 32 c + 16 h .. + 15 of its row: the same permutation of k on both sides), and multiplied in eight
// steps of half a chunk.
template <int TM, int TN> struct F8Raw {
    uint4 a[TM], b[TN];
    // ap, bp: the lane's row of the wave's first tile of A's and of B's rows
    __device__ __forceinline__ void read(const char *ap, const char *bp, int c, int h, int swz) {
        const int slot = 16 * ((2 * c + h) ^ swz);
#pragma unroll
        for (int i = 0; i < TM; i++) a[i] = *(const uint4 *)(ap + i * 32 * 128 + slot);
#pragma unroll
        for (int i = 0; i < TN; i++) b[i] = *(const uint4 *)(bp + i * 32 * 128 + slot);
    }
};
template <int TM, int TN> struct F8Step {
    f8_v8bf a[TM], b[TN];
    // operand i of step z of a chunk: A's tiles, then B's
    template <int FA, int FB> __device__ __forceinline__ void convert(const F8Raw<TM, TN> &r, int z, int i) {
        if (i < TM) a[i] = z ? f8_bf16x8<FA>(r.a[i].z, r.a[i].w) : f8_bf16x8<FA>(r.a[i].x, r.a[i].y);
        else b[i - TM] = z ? f8_bf16x8<FB>(r.b[i - TM].z, r.b[i - TM].w) : f8_bf16x8<FB>(r.b[i - TM].x, r.b[i - TM].y);
    }
};
// no instruction is scheduled across
__device__ __forceinline__ void f8_pin() {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_sched_barrier(0);
#endif
}

// The scales of a block for a wave's tiles: sa_ at the lane's row of A, sb_ at the wave's first row of B.
template <bool BROWS, int TM, int TN> struct F8Scales {
    float a[TM], b;
    f8_v4f rows[BROWS ? 4 * TN : 1];
    __device__ __forceinline__ void read(const float *sa_, const float *sb_, int h) {
#pragma unroll
        for (int i = 0; i < TM; i++) a[i] = sa_[i * 32];
        if constexpr (BROWS) {
#pragma unroll
            for (int q = 0; q < 4 * TN; q++) rows[q] = *(const f8_v4f *)(sb_ + 4 * h + 8 * q);
        } else {
            b = sb_[0];
        }
    }
    // acc += part times the scales, for tile (im, in)
    __device__ __forceinline__ void add(const f8_v16f &part, f8_v16f &acc, int im, int in) const {
        const float one = a[im] * b;
#pragma unroll
        for (int i = 0; i < 16; i++)
            acc[i] = __builtin_fmaf(part[i], BROWS ? a[im] * rows[BROWS ? 4 * in + i / 4 : 0][i % 4] : one, acc[i]);
    }
};

// One block: the block before's products (part) are scaled into acc with the scales at sa, sb, then this block's are
// computed.  The order keeps the matrix unit fed and is pinned, since the compiler's own puts the LDS reads next to
// their use: a chunk is read a chunk ahead, and between one matrix instruction and the next stand the conversions of
// an operand of the next step and, in the first step, the scaling of the tile that is overwritten next.  So do the
// direct loads of a later block, feed(slot, slots) after each matrix instruction: issued together they hold the wave
// up for as long as the CU takes to address them (16 cycles each).  LATE false: this block's own products are scaled,
// after them, and the loads go into the stage just read, in the second half; else into another, in the first.
template <int FA, int FB, bool BROWS, int TM, int TN, bool LATE, typename F>
__device__ __forceinline__ void f8_block(const char *ap, const char *bp, const float *sa, const float *sb, int h, int swz,
                                         f8_v16f (&part)[TN][TM], f8_v16f (&acc)[TN][TM], F &&feed) {
    constexpr int T = TM * TN, P = TM + TN;
    F8Raw<TM, TN> r[2];
    F8Step<TM, TN> s[2];
    F8Scales<BROWS, TM, TN> sc;
    r[0].read(ap, bp, 0, h, swz);
    sc.read(sa, sb, h);
    r[1].read(ap, bp, 1, h, swz);
    f8_pin();
#pragma unroll
    for (int i = 0; i < P; i++) s[0].template convert<FA, FB>(r[0], 0, i);
    if constexpr (LATE) sc.add(part[0][0], acc[0][0], 0, 0);
#pragma unroll
    for (int t = 0; t < 8; t++) {
        if (!LATE && t == 4) f8_wait_lds();
#pragma unroll
        for (int i = 0; i < T; i++) {
            const int in = i / TM, im = i % TM;
            f8_pin();
            part[in][im] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(s[t & 1].b[in], s[t & 1].a[im], t ? part[in][im] : f8_v16f{}, 0, 0, 0);
            f8_pin();
            if (LATE ? t < 4 : t >= 4) feed((t & 3) * T + i, 4 * T);
            f8_pin();
            if (i == 0 && (t == 1 || t == 3)) {
                r[t == 3].read(ap, bp, t == 1 ? 2 : 3, h, swz);
                f8_pin();
            }
            if (t < 7) {
#pragma unroll
                for (int o = i * P / T; o < (i + 1) * P / T; o++)
                    s[(t + 1) & 1].template convert<FA, FB>(r[((t + 1) / 2) & 1], (t + 1) & 1, o);
            }
            if (LATE && t == 0 && i + 1 < T) sc.add(part[(i + 1) / TM][(i + 1) % TM], acc[(i + 1) / TM][(i + 1) % TM], (i + 1) % TM, (i + 1) / TM);
        }
    }
    f8_pin();
    if constexpr (!LATE) {
#pragma unroll
        for (int i = 0; i < T; i++) sc.add(part[i / TM][i % TM], acc[i / TM][i % TM], i % TM, i / TM);
    }
}
// the last block's products into acc
template <bool BROWS, int TM, int TN>
__device__ __forceinline__ void f8_scale_add(const f8_v16f (&part)[TN][TM], const float *sa, const float *sb, int h,
                                             f8_v16f (&acc)[TN][TM]) {
    F8Scales<BROWS, TM, TN> sc;
    sc.read(sa, sb, h);
#pragma unroll
    for (int in = 0; in < TN; in++)
#pragma unroll
        for (int im = 0; im < TM; im++) sc.add(part[in][im], acc[in][im], im, in);
}

// A wave's tiles as rows of 32 TN floats in LDS, in slots of four floats, slot s of row m at s ^ f8_turn(m): a column
// of the accumulators' four-float pieces and a row both spread over the banks.
template <int TN> __device__ __forceinline__ int f8_turn(int m) { return TN == 1 ? (m >> 1) & 7 : m & 15; }

template <int TM, int TN>
__device__ __forceinline__ void f8_put(float *t, const f8_v16f (&acc)[TN][TM], int l) {
    static_assert(TN == 1 || TN == 2, "8 or 16 slots a row");
    const int h = l >> 5;
#pragma unroll
    for (int im = 0; im < TM; im++) {
        const int m = im * 32 + (l & 31);
#pragma unroll
        for (int in = 0; in < TN; in++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                f8_v4f v;
                for (int e = 0; e < 4; e++) v[e] = acc[in][im][4 * q + e];
                *(f8_v4f *)(t + m * 32 * TN + 4 * ((8 * in + 2 * q + h) ^ f8_turn<TN>(m))) = v;
            }
    }
}

// Writes rows [0, rows) of such a tile, summed over `parts` of them `stride` floats apart in order, to y's rows from
// (m0, n0) on, plus the bias: whole rows of neighbouring floats by neighbouring threads.  PAST: past the caches.
template <int TM, int TN, bool PAST>
__device__ __forceinline__ void f8_store_rows(const MatMulBlocksArgs &p, const float *t, int parts, int stride, int64_t m0, int64_t n0,
                                         int thread, int threads) {
    constexpr int W = 32 * TN;
    const int rows = (int)std::min<int64_t>(32 * TM, p.m - m0), cols = (int)std::min<int64_t>(W, p.n - n0);
    float *y = p.y + m0 * p.n + n0;
    const float *bias = p.bias ? p.bias + n0 : nullptr;
    if (p.n % 4 == 0 && ((uintptr_t)p.y & 15) == 0) {
        for (int i = thread; i < rows * (W / 4); i += threads) {
            const int m = i / (W / 4), s = i % (W / 4);
            if (4 * s >= cols) continue;
            const float *f = t + m * W + 4 * (s ^ f8_turn<TN>(m));
            f8_v4f v = *(const f8_v4f *)f;
            for (int k = 1; k < parts; k++) v += *(const f8_v4f *)(f + k * stride);
            if (bias)
                for (int e = 0; e < 4; e++) v[e] += bias[4 * s + e];
            if constexpr (PAST) __builtin_nontemporal_store(v, (f8_v4f *)(y + m * p.n + 4 * s));
            else *(f8_v4f *)(y + m * p.n + 4 * s) = v;
        }
    } else {
        for (int i = thread; i < rows * W; i += threads) {
            const int m = i / W, n = i % W;
            if (n >= cols) continue;
            const float *f = t + m * W + 4 * ((n / 4) ^ f8_turn<TN>(m)) + n % 4;
            float v = *f;
            for (int k = 1; k < parts; k++) v += f[k * stride];
            if (bias) v += bias[n];
            if constexpr (PAST) __builtin_nontemporal_store(v, y + m * p.n + n);
            else y[m * p.n + n] = v;
        }
    }
}

__device__ __forceinline__ void f8_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Results of more than the L2s hold (32 MB) go past them: 8192x4096x8192 495 us against 479, and a vocabulary's logits,
// [512, 30522], leave the inputs of the next call there (the product alone 38.0 against 39.1, with the quantisation
// before it and the log-probabilities after it 66.5 against 64.5).
template <int TM, int TN>
__device__ __forceinline__ void f8_store(const MatMulBlocksArgs &p, const float *t, int parts, int stride, int64_t m0, int64_t n0,
                                         int thread, int threads) {
    if (p.m * p.n > (8 << 20)) f8_store_rows<TM, TN, true>(p, t, parts, stride, m0, n0, thread, threads);
    else f8_store_rows<TM, TN, false>(p, t, parts, stride, m0, n0, thread, threads);
}

// The tile of a workgroup, false if it has none: tiles in groups of eight rows of them, down a group's columns one after
// the other, and a contiguous range of that order for each XCD (workgroups go round the 8 XCDs), so that an XCD's cache
// is asked for few rows of A and of B (64x4096x4096 in tiles of 32x32 8.0 us against 9.8 in the grid's order).
__device__ __forceinline__ bool f8_tile(int tm, int tn, int *im, int *in) {
    const int tiles = tm * tn, per = (tiles + 7) / 8, t = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || t >= tiles) return false;
    const int group = t / (8 * tn), first = 8 * group, rows = min(tm - first, 8), at = t - group * 8 * tn;
    *im = first + at % rows;
    *in = at / rows;
    return true;
}

template <int FA, int FB, bool BROWS, int TM, int TN, int WM, int WN, int S, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void k_matmul_blocks(MatMulBlocksArgs p, int tm, int tn) {
    constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, R = BM + BN;
    constexpr int L = R / 8 / NW;               // 16-byte loads a wave and stage, of eight rows each
    constexpr int LS = (R / 64 + NW - 1) / NW;  // 4-byte loads of the rows' scales
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM % 64 == 0 && BN % 64 == 0 && BN <= 128, "whole wave loads");
    constexpr int STAGE = R * 128, SCALES = LS * NW * 64;
    __shared__ __attribute__((aligned(1024))) char sm[S][STAGE];
    __shared__ __attribute__((aligned(256))) float sc[S + 1][SCALES];  // a block's scales are read one block later
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = l >> 5;

    int im0, in0;
    if (!f8_tile(tm, tn, &im0, &in0)) return;
    const int m0 = im0 * BM, n0 = in0 * BN;

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
    // direct load i of the wave's L + LS of a stage (none of a cut last block's)
    auto load_one = [&](int i, int64_t j, char *st, float *scl) {
        if (i < L) f8_load_lds16((NW * i < BM / 8 ? abase : bbase) + 128 * j, off[i], st + 1024 * (w + NW * i));
        else f8_load_lds4((64 * (w + NW * (i - L)) < BM ? sabase : sbbase) + j, soff[i - L], scl + 64 * (w + NW * (i - L)));
    };
    auto load_cut = [&](int64_t j, char *st, float *scl) {
#pragma unroll
        for (int i = 0; i < L; i++) {
            const int r = 8 * (w + NW * i) + (l >> 3), c = (l & 7) ^ ((r >> 1) & 7);
            char *lds = st + 1024 * (w + NW * i);
            if (16 * c < tail) load_one(i, j, st, scl);
            else *(uint4 *)(lds + 16 * l) = uint4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = L; i < L + LS; i++) load_one(i, j, st, scl);
    };
    auto load = [&](int64_t j, char *st, float *scl) {
        if (tail && j == kb - 1) {
            load_cut(j, st, scl);
        } else {
#pragma unroll
            for (int i = 0; i < L + LS; i++) load_one(i, j, st, scl);
        }
    };

    f8_v16f acc[TN][TM] = {}, part[TN][TM] = {};
    const int wm = w % WM, wn = w / WM;
    const int swz = ((l & 31) >> 1) & 7;
    for (int i = threadIdx.x; i < SCALES; i += 64 * NW) sc[S][i] = 0.0f;  // before the first block: nothing times zero
    for (int s = 0; s < S - 1; s++)
        if (s < kb) load(s, sm[s], sc[s]);
    int cur = 0, scur = 0;
    // block j; FEED: block j + S - 1 is there and whole
    auto step = [&](int64_t j, auto feed_) {
        constexpr bool FEED = decltype(feed_)::value;
        // the last S - 2 stages ahead may still be landing; near the end there are fewer
        if (S > 2 && (FEED || j + S - 2 < kb)) f8_wait_barrier<(S - 2) * (L + LS)>();
        else f8_wait_barrier<0>();
        const char *st = sm[cur], *ap = st + (wm * TM * 32 + (l & 31)) * 128, *bp = st + (BM + wn * TN * 32 + (l & 31)) * 128;
        const int before = scur == 0 ? S : scur - 1;  // the block before's scales
        const int ahead = scur + S - 1;
        const int64_t jn = j + S - 1;
        char *stn = sm[cur == 0 ? S - 1 : cur - 1];
        float *scn = sc[ahead > S ? ahead - S - 1 : ahead];
        if (!FEED && jn == kb - 1) load_cut(jn, stn, scn);
        cur = cur + 1 == S ? 0 : cur + 1;
        scur = scur == S ? 0 : scur + 1;
        const float *c = sc[before];
        f8_block<FA, FB, BROWS, TM, TN, true>(ap, bp, c + wm * TM * 32 + (l & 31), c + BM + wn * TN * 32, h, swz, part, acc,
                                              [&](int slot, int slots) {
            if constexpr (FEED) {
#pragma unroll
                for (int i = slot * (L + LS) / slots; i < (slot + 1) * (L + LS) / slots; i++) load_one(i, jn, stn, scn);
            }
        });
    };
    const int64_t fed = kb - (S - 1) - (tail ? 1 : 0);
    int64_t j = 0;
    for (; j < fed; j++) step(j, std::true_type());
    for (; j < kb; j++) step(j, std::false_type());
    if (kb) {
        const float *c = sc[scur == 0 ? S : scur - 1];
        f8_scale_add<BROWS>(part, c + wm * TM * 32 + (l & 31), c + BM + wn * TN * 32, h, acc);
    }
    // the stages are done with: each wave's tiles go out through its part of them
    f8_wait_barrier<0>();
    float *t_ = (float *)&sm[0][0] + w * TM * TN * 1024;
    static_assert(NW * TM * TN * 4096 <= S * STAGE, "room for the waves' tiles");
    f8_put<TM, TN>(t_, acc, l);
    f8_wave_sync();
    f8_store<TM, TN>(p, t_, 1, 0, m0 + wm * TM * 32, n0 + wn * TN * 32, l, 64);
}

// ---- few tiles: waves over K ------------------------------------------------------------------------------------
// Where a launch has too few tiles for the chip's workgroups, a workgroup takes one wave's tiles (TM x TN of 32x32) and
// its W waves share the blocks of K (block j to wave j mod W), each with two stages of its own in LDS, so that no wave
// waits for another until their sums are joined in order at the end.  LA: eight-row groups of A that are loaded (rows
// from p.m on only reach results that are not stored).  CHUNKS: rows of whole aligned 16-byte chunks, loaded straight to
// LDS; other rows go through registers, a block ahead too.
template <int FA, int FB, bool BROWS, int TM, int TN, int LA, int MAXW, bool CHUNKS>
__global__ __launch_bounds__(64 * MAXW) void k_matmul_blocks_thin(MatMulBlocksArgs p, int tm, int tn) {
    constexpr int BM = 32 * TM, BN = 32 * TN, LB = BN / 8, L = LA + LB, LS = (BM + BN) / 64;
    constexpr int STAGE = (BM + BN) * 128 + LS * 256;
    __shared__ __attribute__((aligned(1024))) char sm[MAXW * 2 * STAGE];
    const int l = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = blockDim.x >> 6, h = l >> 5;
    char *mine = sm + w * 2 * STAGE;
    int im0, in0;
    if (!f8_tile(tm, tn, &im0, &in0)) return;
    const int64_t m0 = (int64_t)im0 * BM, n0 = (int64_t)in0 * BN;
    const int64_t kb = (p.k + 127) / 128;
    const int row_n = BROWS ? 1 : 128;
    const uint8_t *abase = p.a + m0 * p.k, *bbase = p.b + n0 * p.k;
    const float *sabase = p.sa + m0 * kb, *sbbase = p.sb + n0 / row_n * kb;
    const int rows_a = (int)std::min<int64_t>(p.m - m0, BM) - 1, rows_b = (int)std::min<int64_t>(p.n - n0, BN) - 1;
    const int tail = (int)(p.k & 127);

    uint32_t off[L], soff[LS];
#pragma unroll
    for (int i = 0; i < L; i++) {
        const int r = 8 * (i < LA ? i : i - LA + BM / 8) + (l >> 3), c = (l & 7) ^ ((r >> 1) & 7);
        off[i] = (uint32_t)((i < LA ? min(r, rows_a) : min(r - BM, rows_b)) * (int)p.k + 16 * c);
    }
#pragma unroll
    for (int i = 0; i < LS; i++) {
        const int r = 64 * i + l;
        soff[i] = (uint32_t)((r < BM ? min(r, rows_a) : min(r - BM, rows_b) / row_n) * (int)kb * 4);
    }
    auto scales = [&](int64_t j, char *st, int i) {
        if constexpr (BM % 64 == 0) {
            f8_load_lds4((64 * i < BM ? sabase : sbbase) + j, soff[i], st + (BM + BN) * 128 + 256 * i);
        } else {  // the first half of the lanes A's rows, the second B's
            if (l < BM) f8_load_lds4(sabase + j, soff[i], st + (BM + BN) * 128);
            else f8_load_lds4(sbbase + j, soff[i], st + (BM + BN) * 128);
        }
    };
    constexpr int NL = L + (BM % 64 == 0 ? LS : 2);  // direct loads a stage
    auto load_one = [&](int i, int64_t j, char *st) {  // i-th of L + LS (none of a cut last block's)
        if (i < L) f8_load_lds16((i < LA ? abase : bbase) + 128 * j, off[i], st + 1024 * (i < LA ? i : i - LA + BM / 8));
        else scales(j, st, i - L);
    };
    auto load_cut = [&](int64_t j, char *st) {
#pragma unroll
        for (int i = 0; i < L; i++) {
            const int g = i < LA ? i : i - LA + BM / 8, r = 8 * g + (l >> 3), c = (l & 7) ^ ((r >> 1) & 7);
            if (16 * c < tail) load_one(i, j, st);
            else *(uint4 *)(st + 1024 * g + 16 * l) = uint4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = L; i < L + LS; i++) load_one(i, j, st);
    };
    auto load = [&](int64_t j, char *st) {
        if (tail && j == kb - 1) {
            load_cut(j, st);
        } else {
#pragma unroll
            for (int i = 0; i < L + LS; i++) load_one(i, j, st);
        }
    };
    uint4 reg[CHUNKS ? 1 : L];
    auto fetch = [&](int64_t j) {
#pragma unroll
        for (int i = 0; i < (CHUNKS ? 0 : L); i++) {
            const int g = i < LA ? i : i - LA + BM / 8, r = 8 * g + (l >> 3), c = (l & 7) ^ ((r >> 1) & 7);
            const uint8_t *row = (i < LA ? abase : bbase) + (int64_t)off[i] - 16 * c;
            reg[i] = f8_load16(row, 128 * (int)j + 16 * c, (int)p.k);
        }
    };
    auto drop = [&](int64_t j, char *st) {
#pragma unroll
        for (int i = 0; i < (CHUNKS ? 0 : L); i++) {
            const int g = i < LA ? i : i - LA + BM / 8, r = 8 * g + (l >> 3), c = (l & 7) ^ ((r >> 1) & 7);
            *(uint4 *)(st + 1024 * g + 16 * l) = j == kb - 1 ? f8_tail16(reg[i], 128 * (int)j + 16 * c, (int)p.k) : reg[i];
        }
    };

    f8_v16f acc[TN][TM] = {}, part[TN][TM];
    const int swz = ((l & 31) >> 1) & 7;
    auto block = [&](const char *st, auto &&feed) {
        const float *sc = (const float *)(st + (BM + BN) * 128);
        f8_block<FA, FB, BROWS, TM, TN, false>(st + (l & 31) * 128, st + (BM + (l & 31)) * 128, sc + (l & 31), sc + BM, h, swz, part, acc,
                                                 feed);
    };
    if constexpr (CHUNKS) {
        if (w < kb) load(w, mine);
        if (w + W < kb) load(w + W, mine + STAGE);
        int cur = 0;
        auto step = [&](int64_t j, auto feed_) {
            constexpr bool FEED = decltype(feed_)::value;  // block j + 2 W is there and whole
            char *st = mine + cur * STAGE;
            if (FEED || j + W < kb) f8_wait<NL>();
            else f8_wait<0>();
            block(st, [&](int slot, int slots) {
                if constexpr (FEED) {
#pragma unroll
                    for (int i = slot * (L + LS) / slots; i < (slot + 1) * (L + LS) / slots; i++) load_one(i, j + 2 * W, st);
                }
            });
            if (!FEED && j + 2 * W == kb - 1) load_cut(j + 2 * W, st);
            cur ^= 1;
        };
        const int64_t fed = kb - 2 * W - (tail ? 1 : 0);
        int64_t j = w;
        for (; j < fed; j += W) step(j, std::true_type());
        for (; j < kb; j += W) step(j, std::false_type());
    } else {
        if (w < kb) fetch(w);
        for (int64_t j = w; j < kb; j += W) {
            f8_wait_lds();
            drop(j, mine);
#pragma unroll
            for (int i = 0; i < LS; i++) scales(j, mine, i);
            if (j + W < kb) fetch(j + W);
            f8_wait<0>();
            block(mine, [](int, int) {});
        }
    }
    // every wave's sums in its own stage, joined in the waves' order
    f8_wait_lds();
    f8_put<TM, TN>((float *)mine, acc, l);
    __syncthreads();
    f8_store<TM, TN>(p, (const float *)sm, W, 2 * STAGE / 4, m0, n0, threadIdx.x, blockDim.x);
}

template <int FA, int FB, bool BROWS, int TM, int TN, int LA, int MAXW>
static void thin(const MatMulBlocksArgs &p, bool chunks, hipStream_t s) {
    const int64_t tm = (p.m + 32 * TM - 1) / (32 * TM), tn = (p.n + 32 * TN - 1) / (32 * TN);
    const unsigned threads = 64 * (unsigned)std::max<int64_t>(1, std::min<int64_t>(MAXW, (p.k + 127) / 128));
    const unsigned grid = (unsigned)((tm * tn + 7) / 8 * 8);
    if (chunks) k_matmul_blocks_thin<FA, FB, BROWS, TM, TN, LA, MAXW, true><<<grid, threads, 0, s>>>(p, (int)tm, (int)tn);
    else k_matmul_blocks_thin<FA, FB, BROWS, TM, TN, LA, MAXW, false><<<grid, threads, 0, s>>>(p, (int)tm, (int)tn);
}

// Rows of whole aligned 16-byte chunks: what the direct-to-LDS loads take.
static bool whole_chunks(const MatMulBlocksArgs &p) { return p.k % 16 == 0 && (((uintptr_t)p.a | (uintptr_t)p.b) & 15) == 0; }
static int64_t tiles(const MatMulBlocksArgs &p, int64_t b) { return (p.m + b - 1) / b * ((p.n + b - 1) / b); }

// Other rows copied to such, zeros behind them: 16 bytes a thread, A's rows and then B's.
__global__ __launch_bounds__(256) void k_matmul_blocks_rows(MatMulBlocksArgs p, uint4 *out, FastDiv chunks, uint32_t total) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const uint32_t r = fdiv(i, chunks), c = 16 * (i - r * chunks.d);
    const uint8_t *row = r < p.m ? p.a + (int64_t)r * p.k : p.b + (int64_t)(r - p.m) * p.k;
    out[i] = f8_tail16(f8_load16(row, (int)c, (int)p.k), (int)c, (int)p.k);
}

// Products of many tiles are worth that copy: (m + n) k bytes read and written against kernels that wait for
// their loads.
int64_t matmul_blocks_part_bytes(const MatMulBlocksArgs &p) {
    const int64_t bytes = (p.m + p.n) * ((p.k + 15) / 16 * 16);
    return !whole_chunks(p) && p.k > 0 && p.m > 32 && tiles(p, 64) > 256 && bytes / 16 < ((int64_t)1 << 31) ? bytes : 0;
}

// The kernel of a product by its tiles of Y, one workgroup each, against the chip's 256 CUs (us on one device, e4m3):
//   128x128 from 256 of them on: [512,768]x[30522,768] 39 against 48 in tiles of 64x64, 8192x4096x8192 469 against 640;
//     4096x768x768, 192 of them, 13.0 against 12.5
//   64x64 from 257 on: 2048x1024x1024 11.4 against 12.9 with waves over K; 1024x1024x1024, 256 of them, 8.6 against 7.5
//   64x64 with waves over K from 129 on, and for rows that are not whole chunks: 788x768x768 6.7 against 7.2 in tiles
//     of 32x32; 128x4096x4096, 128 of them, 13.1 against 11.5
//   32x32 with waves over K: eight waves up to 256 of them (64x4096x4096 9.6 against 10.0), more with four, two
//     workgroups a CU (788x768x768 7.4 against 8.9); of at most eight rows only those of A are read.
template <int FA, int FB, bool BROWS> static hipError_t matmul_blocks(const MatMulBlocksArgs &p, hipStream_t s) {
    const bool chunks = whole_chunks(p);
    if (chunks && tiles(p, 128) >= 256) {
        k_matmul_blocks<FA, FB, BROWS, 2, 2, 2, 2, 2, 2>
            <<<(unsigned)((tiles(p, 128) + 7) / 8 * 8), 256, 0, s>>>(p, (int)((p.m + 127) / 128), (int)((p.n + 127) / 128));
    } else if (chunks && p.m > 32 && tiles(p, 64) > 256) {
        k_matmul_blocks<FA, FB, BROWS, 1, 1, 2, 2, 3, 3>
            <<<(unsigned)((tiles(p, 64) + 7) / 8 * 8), 256, 0, s>>>(p, (int)((p.m + 63) / 64), (int)((p.n + 63) / 64));
    } else if (p.m > 32 && tiles(p, 64) > 128) {
        thin<FA, FB, BROWS, 2, 2, 8, 4>(p, chunks, s);
    } else if (tiles(p, 32) <= 256) {
        if (p.m <= 8) thin<FA, FB, BROWS, 1, 1, 1, 8>(p, chunks, s);
        else thin<FA, FB, BROWS, 1, 1, 4, 8>(p, chunks, s);
    } else {
        if (p.m <= 8) thin<FA, FB, BROWS, 1, 1, 1, 4>(p, chunks, s);
        else thin<FA, FB, BROWS, 1, 1, 4, 4>(p, chunks, s);
    }
    return hipGetLastError();
}

template <int FA, int FB> static hipError_t matmul_blocks(const MatMulBlocksArgs &p, hipStream_t s) {
    return p.b_rows == 1 ? matmul_blocks<FA, FB, true>(p, s) : matmul_blocks<FA, FB, false>(p, s);
}

hipError_t launch_matmul_blocks(const MatMulBlocksArgs &given, hipStream_t s) {
    MatMulBlocksArgs p = given;
    if (const int64_t bytes = matmul_blocks_part_bytes(given)) {
        const uint32_t row = (uint32_t)((p.k + 15) / 16), total = (uint32_t)(bytes / 16);
        k_matmul_blocks_rows<<<(total + 255) / 256, 256, 0, s>>>(given, (uint4 *)p.part, make_fastdiv(row), total);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        p.k = 16 * (int64_t)row;
        p.a = (const uint8_t *)p.part;
        p.b = p.a + p.m * p.k;
    }
    if (p.fmt_a == kFloat8E4M3FN)
        return p.fmt_b == kFloat8E4M3FN ? matmul_blocks<kFloat8E4M3FN, kFloat8E4M3FN>(p, s)
                                        : matmul_blocks<kFloat8E4M3FN, kFloat8E5M2>(p, s);
    return p.fmt_b == kFloat8E4M3FN ? matmul_blocks<kFloat8E5M2, kFloat8E4M3FN>(p, s)
                                    : matmul_blocks<kFloat8E5M2, kFloat8E5M2>(p, s);
}

}  // namespace lx
