// mp_fp8.hip -- e4m3 weights with a scale for each block of 128 x 128: the
// quantizer (moe_fp8_quantize), products (moe_fp8_product) and a layer of experts
// (moe_fp8_layer).
//
// y[m][n] = sum over the blocks b of K of  sx[m][b] sw[n/128][b] (xq[m] . wq[n])_b:  a block's
// dot runs on the matrix cores, and one fma adds it, scaled, to the f32 sum of the row.  The weight's 16 rows are the A
// operand, so that a lane holds four of them for one row of x: one scale a lane and block.
//
// The codes become fp16 for the matrix cores (exactly), whose fp16 products are exact and their sums f32.  The cores' own e4m3
// instructions (16x16x128 and 16x16x32 alike) add eight neighbouring products at 13 bits below the largest of them, what is below cut
// off (found by products of powers of two: 2^-13 of the largest stays, 2^-14 does not).  They take half the time, but that is 1.4e-5
// of a sum of normal numbers, where f32 sums have 1e-8, and all of a sum whose large products cancel.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

typedef int int4_v __attribute__((ext_vector_type(4)));
typedef int int4_u __attribute__((ext_vector_type(4), aligned(1)));       // wherever it begins
typedef int int8_v __attribute__((ext_vector_type(8)));
typedef float float4_v __attribute__((ext_vector_type(4)));
typedef _Float16 half2_v __attribute__((ext_vector_type(2)));
typedef _Float16 half8_v __attribute__((ext_vector_type(8)));

constexpr int FB = FP8_BLOCK;
#define FP8_INLINE __attribute__((always_inline))

// ---- the quantizer ---------------------------------------------------------------
// The scale of a block whose largest finite magnitude is amax: the least power of two s, from 2^-126 on, with amax <= 448 s.
// 448 = 1.75 * 2^8, so the exponent is amax's less 8, or less 7 above 1.75.
__device__ inline int scale_exp(float amax) {
    const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return e < -126 ? -126 : e;
}
__device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }      // e from -126 to 127

// eight values -> their codes; inv: 1 / the scale.  |v * inv| <= 448, so no code overflows; the conversion rounds to the nearest,
// ties to even, and a NaN stays one.
__device__ inline uint2 codes8(const float *v, float inv) {
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Infinities become NaN, as e4m3 has none, and do not count for the scale.
__device__ inline float finite_or_nan(float v) { return v - v == 0.0f ? v : NAN; }

// maximum over 16 neighbouring lanes, on each of them
__device__ inline float max16(float v) {
    v = fmaxf(v, dpp_f<DPP_XOR1>(v));
    v = fmaxf(v, dpp_f<DPP_XOR2>(v));
    v = fmaxf(v, dpp_f<DPP_HALF_MIRROR>(v));
    return fmaxf(v, dpp_f<DPP_MIRROR>(v));
}

// n of eight elements of a row, the rest zeros
template <int T>
__device__ inline void load8(const typename Elem<T>::raw *p, int n, float *v) {
    if (n >= 8) {
        typename Elem<T>::raw q[8];
        __builtin_memcpy(q, p, sizeof q);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = Elem<T>::load(q[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? Elem<T>::load(p[i]) : 0.0f;
    }
}
__device__ inline void store8(uint8_t *p, int n, uint2 c) {
    if (n >= 8) __builtin_memcpy(p, &c, 8);
    else
        for (int i = 0; i < n; ++i) p[i] = (uint8_t)((i < 4 ? c.x : c.y) >> 8 * (i & 3));
}
__device__ inline float amax8(const float *v, float m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));        // passes over a NaN
    return m;
}
// the largest finite magnitude of a lane's values, if m, the largest of any lane's it is compared with, is infinite
__device__ inline float without_inf(float *v, float m) {
    if (!(m == INFINITY)) return m;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = finite_or_nan(v[i]);
    return amax8(v, 0.0f);
}

// Sixteen lanes a block of one row, eight neighbouring elements each in one load; NB blocks a lane, sixteen apart, whose loads are on their
// way together.  magic, shift: the division by the blocks of a row.  Memory bounds many rows (8,192 of 4,096 in bf16: 20.8 us, 4.9 TB/s, as a
// copy), the launch few (64 of 2,048: 2.5 us).
template <int T, int NB>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(Fp8QuantArgs a, uint32_t nb, uint32_t total, uint32_t magic, int shift) {
    const uint32_t g0 = blockIdx.x * (16 * NB) + threadIdx.x / 16;
    const int l = threadIdx.x % 16;
    float v[NB][8];
    uint32_t row[NB], b[NB];
    int n[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const uint32_t g = g0 + 16 * i;
        row[i] = (uint32_t)((uint64_t)g * magic >> shift);
        b[i] = g - row[i] * nb;
        n[i] = g < total ? a.K - (int)(b[i] * FB) - 8 * l : 0;
        load8<T>((const typename Elem<T>::raw *)a.x + row[i] * a.ldx + b[i] * FB + 8 * l, n[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float m = max16(amax8(v[i], 0.0f));
        if (__any(m == INFINITY)) m = max16(without_inf(v[i], m));
        const int e = scale_exp(m);
        if (n[i] > 0) store8(a.q + row[i] * a.ldq + b[i] * FB + 8 * l, n[i], codes8(v[i], pow2(-e)));
        if (l == 0 && n[i] > 0) a.s[row[i] * a.lds + b[i]] = pow2(e);
    }
}

// a workgroup a block of 128 rows: memory bounds it, too (98,304 of 2,048 in bf16: 123 us, 4.9 TB/s; 768 of 2,048 4.7 us)
template <int T>
__global__ __launch_bounds__(256) void fp8_quant_block_kernel(Fp8QuantArgs a) {
    __shared__ float s_max[4];
    const int64_t r0 = (int64_t)blockIdx.y * FB;
    const int b = blockIdx.x, l = threadIdx.x % 16, k = b * FB + 8 * l, n = a.K - k;
    float v[8][8];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = r0 + threadIdx.x / 16 + 16 * i;
        load8<T>((const typename Elem<T>::raw *)a.x + row * a.ldx + k, row < a.n_tok ? n : 0, v[i]);
        m = amax8(v[i], m);
    }
    auto largest = [&](float m) {
        m = wave_max(m);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
        __syncthreads();
        return fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    };
    m = largest(m);
    if (m == INFINITY) {                                  // (the same on every thread)
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, without_inf(v[i], INFINITY));
        m = largest(m);
    }
    const int e = scale_exp(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = r0 + threadIdx.x / 16 + 16 * i;
        if (n > 0 && row < a.n_tok) store8(a.q + row * a.ldq + k, n, codes8(v[i], pow2(-e)));
    }
    if (threadIdx.x == 0) a.s[blockIdx.y * a.lds + b] = pow2(e);
}

template <int T>
static hipError_t launch_quant_t(const Fp8QuantArgs &a, hipStream_t st) {
    const uint32_t nb = (uint32_t)((a.K + FB - 1) / FB);
    if (a.rows == 1) {
        const uint32_t total = (uint32_t)a.n_tok * nb;                // at most 2^31
        // g / nb = g * magic >> shift for every g below 2^31 + 2^12 (Granlund and Montgomery, Division by Invariant Integers, 1994)
        int bits = 0;
        while ((1u << bits) < nb) ++bits;
        const int shift = 31 + bits;
        const uint32_t magic = (uint32_t)(((1ull << shift) + nb - 1) / nb);
        // four blocks a lane where that leaves every compute unit four workgroups
        if (total >= 256 * 4 * 64)
            hipLaunchKernelGGL((fp8_quant_rows_kernel<T, 4>), dim3((total + 63) / 64), dim3(256), 0, st, a, nb, total, magic, shift);
        else
            hipLaunchKernelGGL((fp8_quant_rows_kernel<T, 1>), dim3((total + 15) / 16), dim3(256), 0, st, a, nb, total, magic, shift);
    } else {
        hipLaunchKernelGGL((fp8_quant_block_kernel<T>), dim3(nb, (unsigned)((a.n_tok + FB - 1) / FB)), dim3(256), 0, st, a);
    }
    return hipGetLastError();
}
hipError_t launch_fp8_quant(const Fp8QuantArgs &a, hipStream_t st) {
    return a.x_type == T_F32 ? launch_quant_t<T_F32>(a, st)
         : a.x_type == T_BF16 ? launch_quant_t<T_BF16>(a, st) : launch_quant_t<T_F16>(a, st);
}

// ---- products ------------------------------------------------------------------
// eight codes, as fp16
__device__ inline half8_v halves(uint32_t lo, uint32_t hi) {
    const half2_v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const half2_v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return half8_v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// a block's dot
__device__ inline float4_v mfma_block(int8_v w, int8_v x) {
    float4_v d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(w[i], w[i + 1]), halves(x[i], x[i + 1]), d, 0, 0, 0);
    return d;
}

// acc += s * (w . x over a block).  The sum is done here: without the empty statement the compiler moves it behind a branch that follows, and there
// it reads the product too early (it waits after the first of the four reads).
__device__ inline void add_block(float4_v &acc, int8_v w, int8_v x, float s) {
    const float4_v d = mfma_block(w, x);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = fmaf(d[k], s, acc[k]);
    asm volatile("" : "+v"(acc));
}

// A lane's 32 of the 128 codes of a row's block: bytes 16 g .. and 64 + 16 g .., g = lane / 16 (which codes meet which is the same
// for both operands).  n: bytes of the row from here on; codes past it are zeros.
__device__ inline int4_v load16(const uint8_t *p, int n) {
    if (n >= 16) return *(const int4_u *)p;
    uint64_t lo = 0, hi = 0;
    for (int i = min(n, 8) - 1; i >= 0; --i) lo = lo << 8 | p[i];
    for (int i = n - 1; i >= 8; --i) hi = hi << 8 | p[i];
    return int4_v{(int)lo, (int)(lo >> 32), (int)hi, (int)(hi >> 32)};
}
__device__ inline int8_v load_frag(const uint8_t *row, int b, int g) {              // of a whole block
    const uint8_t *p = row + b * FB + 16 * g;
    return __builtin_shufflevector(*(const int4_u *)p, *(const int4_u *)(p + 64), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ inline int8_v load_last(const uint8_t *row, int K, int g) {              // of the last one of K codes, which is not whole
    const int k = K / FB * FB;
    return __builtin_shufflevector(load16(row + k + 16 * g, K - k - 16 * g), load16(row + k + 64 + 16 * g, K - k - 64 - 16 * g), 0, 1, 2, 3, 4,
                                   5, 6, 7);
}

__device__ inline void store_elem(void *p, int64_t i, int type, float v) {
    if (type == T_F32) ((float *)p)[i] = v;
    else if (type == T_BF16) ((uint16_t *)p)[i] = Elem<T_BF16>::store(v);
    else ((uint16_t *)p)[i] = Elem<T_F16>::store(v);
}

// n of four neighbouring elements
__device__ inline void store4(void *p, int64_t i, int type, float4_v v, int n) {
    if (n >= 4) {
        if (type == T_F32) {
            __builtin_memcpy((float *)p + i, &v, 16);
        } else {
            uint16_t q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = type == T_BF16 ? Elem<T_BF16>::store(v[k]) : Elem<T_F16>::store(v[k]);
            __builtin_memcpy((uint16_t *)p + i, q, 8);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (k < n) store_elem(p, i + k, type, v[k]);
    }
}

__device__ inline float silu_times(float g, float u) { return u * (g / (1.0f + expf(-g))); }

// ---- products of few rows ----------------------------------------------------------
// Where a product's rows of x come from, and go to.
constexpr int OF_ALL = 0;         // rows 0 .. M - 1
constexpr int OF_DISPATCH = 1;    // an expert's pairs from a dispatch

// Sixteen rows of a weight (of gate and up: GATED) for sixteen rows of codes at a time: every weight is read once for them, and memory bounds the
// call.  KS waves share K, a block each in turn, and their sums are added in their order; with KS 1 each of the workgroup's four has
// sixteen rows of its own.  A wave's loads of DEEP blocks are on their way together.
template <int FROM, bool GATED, int KS>
__global__ __launch_bounds__(256) void fp8_stream_kernel(Fp8Args a) {
    // (one block of gate and up, two of down: 640 pairs of 128 experts 144 us for the layer, 960 158, 600 of 60 off 16 bytes 42.9; two and three
    // 145, 160 and 45.6; four and six 146, 162 and 46.5: waves count more)
    constexpr int DEEP = GATED ? 1 : 2, MATS = GATED ? 2 : 1;
    __shared__ float s_acc[KS > 1 ? MATS : 1][KS][KS > 1 ? 16 : 1][17];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int n0 = (KS > 1 ? blockIdx.x : blockIdx.x * 4 + wave) * 16, whole = a.K / FB, first = KS > 1 ? wave : 0;
    const int e = FROM == OF_ALL ? 0 : (int)blockIdx.y;
    const int begin = FROM == OF_ALL ? 0 : a.offsets[e], end = FROM == OF_ALL ? a.M : a.offsets[e + 1];
    if (KS == 1 && n0 >= a.N) return;
    const int64_t wrow = min(n0 + c, a.N - 1);
    const uint8_t *w[2] = {a.m[0].w + e * a.m[0].ex + wrow * a.m[0].ld, GATED ? a.m[1].w + e * a.m[1].ex + wrow * a.m[1].ld : nullptr};
    const float *ws[2] = {a.m[0].s + e * a.m[0].sex + (int64_t)(n0 / FB) * a.m[0].sld,
                          GATED ? a.m[1].s + e * a.m[1].sex + (int64_t)(n0 / FB) * a.m[1].sld : nullptr};
    for (int p0 = begin; p0 < end; p0 += 16) {
        const int p = min(p0 + c, end - 1);
        const int64_t xrow = FROM == OF_DISPATCH && a.top ? a.perm[p] / a.top : p;
        const uint8_t *x = a.x + xrow * a.ldx;
        const float *xs = a.xs + xrow * a.ldxs;
        float4_v acc[2] = {};
        for (int b0 = first; b0 < whole; b0 += KS * DEEP) {
            int8_v wf[DEEP][2], xf[DEEP];
            float f[DEEP][2], s[DEEP];
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                const int b = b0 + i * KS;
                if (b >= whole) break;
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    wf[i][m] = load_frag(w[m], b, g);
                    f[i][m] = ws[m][b];
                }
                xf[i] = load_frag(x, b, g);
                s[i] = xs[b];
            }
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                if (b0 + i * KS >= whole) break;
#pragma unroll
                for (int m = 0; m < MATS; ++m) add_block(acc[m], wf[i][m], xf[i], s[i] * f[i][m]);
            }
        }
        if (a.K % FB && whole % KS == first) {          // the last block
            const int8_v xt = load_last(x, a.K, g);
#pragma unroll
            for (int m = 0; m < MATS; ++m) add_block(acc[m], load_last(w[m], a.K, g), xt, xs[whole] * ws[m][whole]);
        }
        // (y, or h, of row p0 + col) -> where it goes, and its weight
        auto out_of = [&](int col, float &weight) FP8_INLINE {
            int64_t out = p0 + col;
            weight = 1.0f;
            if (FROM == OF_DISPATCH && a.pair_w) {
                out = a.perm[out];
                weight = a.pair_w[out];
            }
            return out;
        };
        if (KS == 1) {
            const int n = n0 + 4 * g;
            if (p0 + c >= end) continue;
            float weight;
            const int64_t out = out_of(c, weight);
            float4_v y = acc[0];
            if (GATED)
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = silu_times(y[k], acc[1][k]);
            store4(a.y, out * a.ldy + n, a.y_type, FROM == OF_DISPATCH && a.pair_w ? y * weight : y, a.N - n);
            continue;
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int k = 0; k < 4; ++k) s_acc[m][first][c][4 * g + k] = acc[m][k];
        __syncthreads();
        const int r = threadIdx.x & 15, col = threadIdx.x >> 4;
        if (n0 + r >= a.N || p0 + col >= end) continue;
        float y[2];
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
            y[m] = s_acc[m][0][col][r];
#pragma unroll
            for (int i = 1; i < KS; ++i) y[m] += s_acc[m][i][col][r];
        }
        float weight;
        const int64_t out = out_of(col, weight);
        const float v = GATED ? silu_times(y[0], y[1]) : y[0];
        store_elem(a.y, out * a.ldy + n0 + r, a.y_type, FROM == OF_DISPATCH && a.pair_w ? v * weight : v);
    }
}

// Rows quantized into LDS by a workgroup of THREADS, sixteen lanes a block: row i of n (from(i) gives its elements) at q + i * stride with nothing
// behind its K elements but zeros up to a whole block, its scales at s + i * blocks.
template <int T, int THREADS, class F>
__device__ inline void quant_to_lds(int n, int K, F from, uint8_t *q, int stride, float *s) {
    constexpr int NB = 4;
    const int nb = (K + FB - 1) / FB, l = threadIdx.x % 16;
    for (int g0 = threadIdx.x / 16; g0 < n * nb; g0 += THREADS / 16 * NB) {
        float v[NB][8];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int g = g0 + THREADS / 16 * i, row = g / nb, k = (g - row * nb) * FB + 8 * l;
            if (g < n * nb) load8<T>(from(row) + k, K - k, v[i]);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int g = g0 + THREADS / 16 * i, row = g / nb, k = (g - row * nb) * FB + 8 * l;
            if (g >= n * nb) break;                     // (the same for the sixteen lanes)
            float m = max16(amax8(v[i], 0.0f));
            if (m == INFINITY) m = max16(without_inf(v[i], m));
            const int e = scale_exp(m);
            *(uint2 *)(q + row * stride + k) = codes8(v[i], pow2(-e));
            if (l == 0) s[row * nb + (g - row * nb)] = pow2(e);
        }
    }
}
// a row's stride there: sixteen rows' chunks in banks of their own
__host__ __device__ inline int lds_stride(int K) { return (K + FB - 1) / FB * FB + 16; }
__device__ inline int8_v lds_frag(const uint8_t *q, int b, int g) {
    const int4_v *p = (const int4_v *)(q + b * FB + 16 * g);
    return __builtin_shufflevector(p[0], p[4], 0, 1, 2, 3, 4, 5, 6, 7);
}

// The places of the set bits of m, by one wave: list[i] of the i-th
__device__ inline void list_bits(uint64_t m, uint8_t *list) {
    const int lane = threadIdx.x & 63;
    if (m >> lane & 1) list[__popcll(m & ((1ull << lane) - 1))] = (uint8_t)lane;
}

// Sixteen rows of a weight (of gate and up: GATED) for few rows of x, which are quantized into LDS while the weight is on its way: one
// launch, and nothing between.  Four waves share K.
// GATED: workgroup y has the expert of pair y, where that is the expert's first pair, and all of its pairs among the ids
// (at most 64, a wave's lanes); h goes out in f32 in the order of pairs.  Else rows 0 .. M - 1 of x.
// One row through 2,048 x 2,048: 4.0 us, a launch and a trip to memory; gate and up of 768 x 2,048 of eight pairs' experts 10.9 us, 2.3 TB/s.
template <int T, bool GATED>
__global__ __launch_bounds__(256) void fp8_few_up_kernel(Fp8Args a) {
    constexpr int WAVES = 4, DEEP = 4, MATS = GATED ? 2 : 1;
    extern __shared__ __align__(16) uint8_t s_q[];      // [16][stride] codes, [16][nb] scales
    __shared__ float s_acc[MATS][WAVES][16][17];
    __shared__ uint8_t s_list[64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int n0 = blockIdx.x * 16, nb = (a.K + FB - 1) / FB, whole = a.K / FB, stride = lds_stride(a.K);
    float *s_s = (float *)(s_q + a.cols * stride);
    int e = 0, n = a.M;
    if (GATED) {
        const int mine = lane < a.M ? a.ids[lane] : -1;
        e = __builtin_amdgcn_readlane(mine, blockIdx.y);
        const uint64_t m = __ballot(mine == e);
        if ((uint32_t)e >= (uint32_t)a.E || __ffsll((unsigned long long)m) - 1 != (int)blockIdx.y) return;
        n = __popcll(m);
        if (wave == 0) list_bits(m, s_list);
    }
    const int64_t wrow = min(n0 + c, a.N - 1);
    const uint8_t *w[2] = {a.m[0].w + e * a.m[0].ex + wrow * a.m[0].ld, GATED ? a.m[1].w + e * a.m[1].ex + wrow * a.m[1].ld : nullptr};
    const float *ws[2] = {a.m[0].s + e * a.m[0].sex + (int64_t)(n0 / FB) * a.m[0].sld,
                          GATED ? a.m[1].s + e * a.m[1].sex + (int64_t)(n0 / FB) * a.m[1].sld : nullptr};
    int8_v wf[DEEP][2];
    float f[DEEP][2];
    auto load_w = [&](int b0) FP8_INLINE {
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (b0 + i * WAVES < whole)
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    wf[i][m] = load_frag(w[m], b0 + i * WAVES, g);
                    f[i][m] = ws[m][b0 + i * WAVES];
                }
    };
    load_w(wave);
    bool loaded = true;
    if (GATED) __syncthreads();
    for (int p0 = 0; p0 < n; p0 += a.cols) {
        const int cols = min(n - p0, a.cols);
        quant_to_lds<T, 256>(cols, a.K, [&](int i) {
            return (const typename Elem<T>::raw *)a.x + (int64_t)(GATED ? s_list[p0 + i] / a.top : p0 + i) * a.ldx;
        }, s_q, stride, s_s);
        __syncthreads();
        const uint8_t *q = s_q + min(c, cols - 1) * stride;
        const float *s = s_s + min(c, cols - 1) * nb;
        float4_v acc[2] = {};
        auto add = [&](int8_v w, float f, int b, int m) FP8_INLINE { add_block(acc[m], w, lds_frag(q, b, g), s[b] * f); };
        for (int b0 = wave; b0 < whole; b0 += WAVES * DEEP) {
            if (!loaded) load_w(b0);
            loaded = false;
#pragma unroll
            for (int i = 0; i < DEEP; ++i) {
                if (b0 + i * WAVES >= whole) break;
#pragma unroll
                for (int m = 0; m < MATS; ++m) add(wf[i][m], f[i][m], b0 + i * WAVES, m);
            }
        }
        if (whole < nb && whole % WAVES == wave)        // the last block
#pragma unroll
            for (int m = 0; m < MATS; ++m) add(load_last(w[m], a.K, g), ws[m][whole], whole, m);
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int k = 0; k < 4; ++k) s_acc[m][wave][c][4 * g + k] = acc[m][k];
        __syncthreads();
        const int r = threadIdx.x & 15, col = threadIdx.x >> 4;
        if (n0 + r < a.N && col < cols) {
            float y[2];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                y[m] = s_acc[m][0][col][r];
#pragma unroll
                for (int i = 1; i < WAVES; ++i) y[m] += s_acc[m][i][col][r];
            }
            const int64_t out = GATED ? s_list[p0 + col] : p0 + col;
            store_elem(a.y, out * a.ldy + n0 + r, a.y_type, GATED ? silu_times(y[0], y[1]) : y[0]);
        }
    }
}

constexpr int MID_PAIRS = FP8_MID_PAIRS;
// The same for up to MID_PAIRS pairs: workgroup y has expert y (where experts are more than pairs: the expert of pair y, if that is its first one),
// whose pairs every wave finds among the ids, and each of its four waves sixteen rows of the weights.  The expert's rows of x (GATED; else of h: in f32 and in the order of pairs, as GATED leaves them) are quantized into LDS
// by the workgroup, a wave's weights of DEEP blocks on their way while those before are multiplied (one of gate and up, two of down: 10 tokens of
// 256 experts 63.6 us for the layer, 37 of 60 27.9, 64 of 128 134; two and three 69.5, 30.9 and 140, four and six 74.0, 32.2 and 147: waves
// count more).  Memory bounds it: 64 tokens of 128 experts of 768 of 2,048 75 us (5.4 TB/s), down 44.3 (4.5).
template <int T, bool GATED>
__global__ __launch_bounds__(256) void fp8_mid_kernel(Fp8Args a) {
    constexpr int DEEP = GATED ? 1 : 2, MATS = GATED ? 2 : 1;
    extern __shared__ __align__(16) uint8_t s_q[];      // [cols][stride] codes, [cols][nb] scales
    __shared__ uint16_t s_list[MID_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int n0 = (blockIdx.x * 4 + wave) * 16, nb = (a.K + FB - 1) / FB, whole = a.K / FB, stride = lds_stride(a.K);
    const int e = a.E > a.M ? a.ids[blockIdx.y] : blockIdx.y;
    float *s_s = (float *)(s_q + a.cols * stride);
    int ids[MID_PAIRS / 64], n = 0, first = -1;
#pragma unroll
    for (int j = 0; j < MID_PAIRS / 64; ++j) ids[j] = 64 * j + lane < a.M ? a.ids[64 * j + lane] : -1;
#pragma unroll
    for (int j = 0; j < MID_PAIRS / 64; ++j) {
        const uint64_t m = __ballot(ids[j] == e);
        if (wave == 0 && ids[j] == e) s_list[n + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)(64 * j + lane);
        if (n == 0 && m) first = 64 * j + __ffsll((unsigned long long)m) - 1;
        n += __popcll(m);
    }
    if (n == 0 || (uint32_t)e >= (uint32_t)a.E || (a.E > a.M && first != (int)blockIdx.y)) return;
    const int64_t wrow = min(n0 + c, a.N - 1), srow = min(n0, a.N - 1) / FB;
    const uint8_t *w[2] = {a.m[0].w + e * a.m[0].ex + wrow * a.m[0].ld, GATED ? a.m[1].w + e * a.m[1].ex + wrow * a.m[1].ld : nullptr};
    const float *ws[2] = {a.m[0].s + e * a.m[0].sex + srow * a.m[0].sld, GATED ? a.m[1].s + e * a.m[1].sex + srow * a.m[1].sld : nullptr};
    struct Weights {
        int8_v w[DEEP][MATS];
        float s[DEEP][MATS];
    };
    Weights w0, w1;
    auto load_w = [&](Weights &t, int b0) FP8_INLINE {
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (b0 + i < whole)
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    t.w[i][m] = load_frag(w[m], b0 + i, g);
                    t.s[i][m] = ws[m][b0 + i];
                }
    };
    load_w(w0, 0);
    __syncthreads();                                    // the list
    for (int p0 = 0; p0 < n; p0 += a.cols) {
        const int cols = min(n - p0, a.cols);
        if (p0) {
            load_w(w0, 0);
            __syncthreads();                            // the rows before are read
        }
        quant_to_lds<T, 256>(cols, a.K, [&](int i) {
            return (const typename Elem<T>::raw *)a.x + (int64_t)(GATED ? s_list[p0 + i] / a.top : s_list[p0 + i]) * a.ldx;
        }, s_q, stride, s_s);
        __syncthreads();
        const uint8_t *q = s_q + min(c, cols - 1) * stride;
        const float *s = s_s + min(c, cols - 1) * nb;
        float4_v acc[2] = {};
        auto add = [&](const Weights &t, int b0) FP8_INLINE {
#pragma unroll
            for (int i = 0; i < DEEP; ++i)
                if (b0 + i < whole)
#pragma unroll
                    for (int m = 0; m < MATS; ++m) add_block(acc[m], t.w[i][m], lds_frag(q, b0 + i, g), s[b0 + i] * t.s[i][m]);
        };
        for (int b0 = 0; b0 < whole; b0 += 2 * DEEP) {
            load_w(w1, b0 + DEEP);
            add(w0, b0);
            load_w(w0, b0 + 2 * DEEP);
            add(w1, b0 + DEEP);
        }
        if (whole < nb)                                 // the last block
#pragma unroll
            for (int m = 0; m < MATS; ++m) add_block(acc[m], load_last(w[m], a.K, g), lds_frag(q, whole, g), s[whole] * ws[m][whole]);
        const int n1 = n0 + 4 * g;
        if (c < cols && n1 < a.N) {
            const int pair = s_list[p0 + c];
            float4_v y = acc[0];
            if (GATED)
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] = silu_times(y[k], acc[1][k]);
            else y *= a.pair_w[pair];
            store4(a.y, (int64_t)pair * a.ldy + n1, T_F32, y, a.N - n1);
        }
    }
}

// The down product of DOWN_PAIRS pairs at most and the sum over a token's experts: sixteen columns of out for all tokens.  h of all pairs is
// quantized into LDS while the weights are on their way; eight waves share the experts in use, and K.  The pairs' rows meet in LDS,
// where each token's are added in order.
constexpr int DOWN_PAIRS = 8;
__global__ __launch_bounds__(512) void fp8_few_down_kernel(Fp8FewArgs a) {
    constexpr int WAVES = 8, DEEP = 6;
    extern __shared__ __align__(16) uint8_t s_q[];      // [P][stride] codes, [P][nb] scales, [parts][P][17] rows
    __shared__ float s_w[DOWN_PAIRS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, c = lane & 15;
    const int n0 = blockIdx.x * 16, nb = (a.I + FB - 1) / FB, whole = a.I / FB, P = a.n_tok * a.K, stride = lds_stride(a.I);
    float *s_s = (float *)(s_q + P * stride), *s_rows = s_s + P * nb;
    // this wave's expert: the one of pair `mine`, if that is its first, and which of the parts of K
    const int per = WAVES / a.parts, part = wave / per, mine = wave % per;
    const int64_t wrow = min(n0 + c, a.H - 1);
    int ids[DOWN_PAIRS], e = -1, n = 0, pair = 0;       // pair: of this lane's column, the c-th of e's
#pragma unroll
    for (int j = 0; j < DOWN_PAIRS; ++j) {
        ids[j] = j < P ? a.ids[j] : -1;
        if (j == mine) e = ids[j];
    }
    bool live = (uint32_t)e < (uint32_t)a.E;
#pragma unroll
    for (int j = 0; j < DOWN_PAIRS; ++j) {
        if (j >= P || ids[j] != e) continue;
        if (j < mine) live = false;                     // another wave's
        if (n <= c) pair = j;
        ++n;
    }
    if (threadIdx.x < P) s_w[threadIdx.x] = a.w[threadIdx.x];
    const uint8_t *w = a.down.w + (live ? e : 0) * a.down.ex + wrow * a.down.ld;
    const float *ws = a.down.s + (live ? e : 0) * a.down.sex + (int64_t)(n0 / FB) * a.down.sld;
    int8_v wf[DEEP];
    float f[DEEP];
    if (live)
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (part + i * a.parts < whole) {
                wf[i] = load_frag(w, part + i * a.parts, g);
                f[i] = ws[part + i * a.parts];
            }
    quant_to_lds<T_F32, 512>(P, a.I, [&](int i) { return a.h + (int64_t)i * a.I; }, s_q, stride, s_s);
    __syncthreads();
    if (live) {
        const uint8_t *q = s_q + pair * stride;
        float4_v acc = {};
        auto add = [&](int8_v w, int b, float sw) FP8_INLINE { add_block(acc, w, lds_frag(q, b, g), s_s[pair * nb + b] * sw); };
#pragma unroll
        for (int i = 0; i < DEEP; ++i)
            if (part + i * a.parts < whole) add(wf[i], part + i * a.parts, f[i]);
        for (int b0 = part + DEEP * a.parts; b0 < whole; b0 += DEEP * a.parts) {
#pragma unroll
            for (int i = 0; i < DEEP; ++i)
                if (b0 + i * a.parts < whole) {
                    wf[i] = load_frag(w, b0 + i * a.parts, g);
                    f[i] = ws[b0 + i * a.parts];
                }
#pragma unroll
            for (int i = 0; i < DEEP; ++i)
                if (b0 + i * a.parts < whole) add(wf[i], b0 + i * a.parts, f[i]);
        }
        if (whole < nb && whole % a.parts == part) add(load_last(w, a.I, g), whole, ws[whole]);
        if (c < n)
#pragma unroll
            for (int k = 0; k < 4; ++k) s_rows[(part * P + pair) * 17 + 4 * g + k] = acc[k];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_tok * 16; i += 64 * WAVES) {
        const int t = i >> 4, r = i & 15;
        if (n0 + r >= a.H) continue;
        float sum = 0.0f;
        for (int k = 0; k < a.K; ++k) {
            const int pair = t * a.K + k;
            if ((uint32_t)a.ids[pair] >= (uint32_t)a.E) continue;      // of no expert: nothing stands there
            float v = s_rows[pair * 17 + r];
            for (int q = 1; q < a.parts; ++q) v += s_rows[(q * P + pair) * 17 + r];
            sum += s_w[pair] * v;
        }
        store_elem(a.out, (int64_t)t * a.ldo + n0 + r, a.out_type, sum);
    }
}

// Rows of K codes in LDS, at most sixteen, beside a kernel's own 9 KiB
static int lds_rows(int K) { return std::min(16, 54 * 1024 / (lds_stride(K) + 4 * ((K + FB - 1) / FB))); }
bool fp8_few_product(int M, int K) { return M <= lds_rows(K); }
// From how many rows an expert (on average) a layer's products run on tiles.  Weights on 16 bytes: 8 (128 experts of 768 of 2,048, 960 pairs:
// 160 us for the layer, from codes sixteen rows at a time 158; 640: 156 and 144; 1,536: 165 and 197).  Others: 16 (60 of 200 of 1,000, 960 pairs:
// 52 and 51; 600: 52 and 43; 1,920: 55 and 73).
int fp8_tile_rows(const Fp8Mat &gate, const Fp8Mat &up, const Fp8Mat &down) {
    auto on16 = [](const Fp8Mat &m) { return ((uintptr_t)m.w | m.ld | m.ex) % 16 == 0; };
    return on16(gate) && on16(up) && on16(down) ? 8 : 16;
}
// Which layers take the kernels above: few pairs, fewer than tiles have, and of an expert as many as LDS holds, for else its weights are read
// again (80 pairs of 8 experts of 2,048 of 1,024: 37 us, tiles 49; 512 of 128 of 768 of 2,048: 134 and 162; 256 of 32 57.5 and 58.2; 128 of 8 of
// 14,336 of 4,096: 910 and 363).
bool fp8_few_layer(int64_t P, int E, int H, int I, int tile_rows) {
    const int64_t fit = lds_rows(std::max(H, I));
    return P <= MID_PAIRS && (P <= 128 || P < (int64_t)tile_rows * E) && P <= fit * E && std::min(P, (int64_t)2) <= fit;
}

template <int T, bool GATED>
static hipError_t launch_few_t(Fp8Args a, hipStream_t st) {
    a.cols = std::min(a.M, lds_rows(a.K));
    const dim3 grid((unsigned)((a.N + 15) / 16), GATED ? (unsigned)a.M : 1);
    const size_t lds = (size_t)a.cols * (lds_stride(a.K) + 4 * ((a.K + FB - 1) / FB));
    hipLaunchKernelGGL((fp8_few_up_kernel<T, GATED>), grid, dim3(256), lds, st, a);
    return hipGetLastError();
}
template <bool GATED>
static hipError_t launch_few(const Fp8Args &a, int x_type, hipStream_t st) {
    return x_type == T_F32 ? launch_few_t<T_F32, GATED>(a, st) : x_type == T_BF16 ? launch_few_t<T_BF16, GATED>(a, st) : launch_few_t<T_F16, GATED>(a, st);
}
hipError_t launch_fp8_few_product(const Fp8Args &a, int x_type, hipStream_t st) { return launch_few<false>(a, x_type, st); }

static hipError_t launch_few_down(Fp8FewArgs a, hipStream_t st) {
    const int P = a.n_tok * a.K, nb = (a.I + FB - 1) / FB;
    a.parts = 1;
    while (2 * a.parts * P <= 8 && 2 * a.parts <= nb) a.parts *= 2;
    const dim3 grid((unsigned)((a.H + 15) / 16));
    const size_t lds = (size_t)P * (lds_stride(a.I) + 4 * nb) + (size_t)a.parts * P * 17 * 4;
    hipLaunchKernelGGL(fp8_few_down_kernel, grid, dim3(512), lds, st, a);
    return hipGetLastError();
}

template <int T, bool GATED>
static hipError_t launch_mid_t(Fp8Args a, hipStream_t st) {
    a.cols = std::min(a.M, lds_rows(a.K));
    const dim3 grid((unsigned)((a.N + 63) / 64), (unsigned)std::min(a.E, a.M));
    const size_t lds = (size_t)a.cols * (lds_stride(a.K) + 4 * ((a.K + FB - 1) / FB));
    hipLaunchKernelGGL((fp8_mid_kernel<T, GATED>), grid, dim3(256), lds, st, a);
    return hipGetLastError();
}
// Gate and up: up to 32 pairs with K shared by four waves, more with sixteen rows a wave (experts of 768 of 2,048, the layer: 8 pairs 22.7 us and
// 27.3, 16 29.6 and 31.4, 32 46.8 and 46.4; of 512, 24 pairs of 256 29.9 and 32.1, 64 55.9 and 54.7; 64 of 16 of 1,024 43.1 and 40.0).
constexpr int FEW_PAIRS = 32;
static_assert(FEW_PAIRS <= 64, "fp8_few_up_kernel finds pairs by the lanes of a wave");
static hipError_t launch_few_gated(const Fp8Args &a, int x_type, hipStream_t st) {
    if (a.M <= FEW_PAIRS) return launch_few<true>(a, x_type, st);
    return x_type == T_F32 ? launch_mid_t<T_F32, true>(a, st) : x_type == T_BF16 ? launch_mid_t<T_BF16, true>(a, st) : launch_mid_t<T_F16, true>(a, st);
}
// Down with the sum over a token's experts where pairs are DOWN_PAIRS at most, a wave each, else into pair rows (a layer of one token, two
// experts of 2,048 of 1,024: 15.1 us, through pair rows 19.2; one of 8,192 of 5,120: 41.1 and 55.4; four of 768 of 2,048 16.1 and 18.7, eight 21.5
// and 22.8, eight of 1,536 30.8 and 30.1, of 2,048 of 7,168 84.7 and 85.2).
hipError_t launch_fp8_few_layer(Fp8Args a, int x_type, Fp8FewArgs f, float *rows, hipStream_t st) {
    hipError_t err = launch_few_gated(a, x_type, st);
    if (err != hipSuccess) return err;
    if (a.M <= DOWN_PAIRS && a.M <= lds_rows(f.I)) return launch_few_down(f, st);
    a.m[0] = f.down; a.gated = 0;
    a.x = (const uint8_t *)f.h; a.ldx = f.I;
    a.N = f.H; a.K = f.I;
    a.pair_w = f.w;
    a.y = rows; a.ldy = f.H;
    err = launch_mid_t<T_F32, false>(a, st);
    if (err != hipSuccess) return err;
    return launch_fp8_combine({rows, f.ids, f.n_tok, f.K, f.E, f.H, f.out, f.ldo, f.out_type}, st);
}

template <int FROM, bool GATED, int KS>
static hipError_t launch_stream(const Fp8Args &a, hipStream_t st) {
    const int rows = KS > 1 ? 16 : 64;
    const dim3 grid((unsigned)((a.N + rows - 1) / rows), FROM == OF_ALL ? 1 : (unsigned)a.E);
    hipLaunchKernelGGL((fp8_stream_kernel<FROM, GATED, KS>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// ---- products of many rows: tiles through LDS --------------------------------------
// A workgroup computes BN rows of the weight (GATED: BN / 2 of gate and as many of up) for BM rows of x, a wave TN x TM tiles of
// 16 x 16 of it.  A block of K (128 bytes a row) of both operands is one stage of LDS; the next stage's loads, which go to LDS
// without registers, are on their way while this one is multiplied.
// The eight 16-byte chunks of a row lie in LDS at chunk ^ (row & 7): the lanes that read one chunk of eight rows then touch
// all banks once.
// 256 x 128 tiles, three stages, eight waves of 64 x 64: 4,096^3 of given codes 131 us (1.05 PFLOP/s; traced behind a quantizer 137 to 155), 1.65
// us a step of K and 9 a tile and launch beside them (2,048 rows through 4,096 rows of K 256 to 8,192: 12.8 to 118 us).  A step's products take 0.86
// us of the matrix cores at least, its reads of LDS and the loads into it 0.6, its conversions to fp16 are 128 a wave for 64 products.
// 128 x 128 or 256 x 64 tiles took 165 us for the call, not 145.  With the cores' e4m3 products 256 x 256 in two stages, waves of a higher
// priority, the weight loaded to registers past LDS and workgroups that walk over tiles gained nothing or lost.
// This form spills 20 bytes a lane, and that of gate and up of 128 rows 28, none of them within the loop over six steps.
// A dispatch's, 2,048 tokens of 128 experts of 768 of 2,048: gate and up 197 to 203 us, down 123 to 131.
// Workgroups go round the eight XCDs: each has a run of the tiles, so that those at work at once share what they read in its L2.
__device__ inline int xcd_tile(int id, int total) { return id < total / 8 * 8 ? (id % 8) * (total / 8) + id / 8 : id; }
// A workgroup's tile of a dispatch's products: its expert and first row (in the dispatch's order) of a run of bm, and its place among the
// run's n_tiles, which follow one another (2,048 tokens of 128 experts: 341 us for the layer, 363 round the XCDs); false: there is none
__device__ inline bool find_run(const int32_t *offsets, int E, int bm, int n_tiles, int &n_tile, int &e, int &p0, int &end, int *s_run) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int tiles[4], o[5], sum = 0;
#pragma unroll
        for (int j = 0; j < 5; ++j) o[j] = offsets[min(4 * lane + j, E)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            tiles[j] = (o[j + 1] - o[j] + bm - 1) / bm;
            sum += tiles[j];
        }
        int incl = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int t = __shfl_up(incl, d, 64);
            if (lane >= d) incl += t;
        }
        const int total = __builtin_amdgcn_readlane(incl, 63) * n_tiles;
        const int id = xcd_tile(blockIdx.x, total), slot = id / n_tiles;
        if (lane == 0) {
            s_run[3] = (int)blockIdx.x < total;
            s_run[4] = id - slot * n_tiles;
        }
        int at = incl - sum;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (slot >= at && slot < at + tiles[j]) {
                s_run[0] = 4 * lane + j;
                s_run[1] = o[j] + (slot - at) * bm;
                s_run[2] = o[j + 1];
            }
            at += tiles[j];
        }
    }
    __syncthreads();
    e = __builtin_amdgcn_readfirstlane(s_run[0]);
    p0 = __builtin_amdgcn_readfirstlane(s_run[1]);
    end = __builtin_amdgcn_readfirstlane(s_run[2]);
    n_tile = __builtin_amdgcn_readfirstlane(s_run[4]);
    return s_run[3] != 0;
}

// every load of the wave's but the last N is done
template <int N>
__device__ inline void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// a barrier that leaves loads from memory on their way
__device__ inline void barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// NS: stages of loads to LDS without registers (rows on 16 bytes, near one another); 1: through registers.  KG groups of waves share K, a block
// each in turn, and their sums are added in their order.
template <bool GATED, int NS, int KG, int WN, int WM, int TN, int TM>
__global__ __launch_bounds__(64 * WN * WM * KG) void fp8_tile_kernel(Fp8Args a, int n_tiles, int m_tiles) {
    constexpr int THREADS = 64 * WN * WM, BN = 16 * TN * WN, BM = 16 * TM * WM, CH = (BN + BM) * 8 / THREADS, SB = 6;
    static_assert(KG == 1 || (NS > 1 && !GATED && (KG - 1) * THREADS * TN * TM <= KG * (BN + BM) * 8), "sums fit a stage");
    static_assert((BN + BM) * 8 % THREADS == 0 && BN * 8 % THREADS == 0 && THREADS % BM == 0 && SB * 2 * WN <= THREADS, "whole loads");
    static_assert(NS == 1 || (NS == 3 && SB % NS == 0), "each step its own places");
    constexpr int CHUNKS = (BN + BM) * 8 * KG;
    __shared__ int4_v s_0[CHUNKS], s_1[NS > 1 ? CHUNKS : 1], s_2[NS > 1 ? CHUNKS : 1];
    __shared__ int s_run[5];
    __shared__ float s_max[WN][BM], s_sx[KG][2][SB][BM], s_sw[KG][2][SB][2 * WN];
    const int lane = threadIdx.x & 63, tid = threadIdx.x % THREADS, kg = __builtin_amdgcn_readfirstlane(threadIdx.x / THREADS);
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15;
    const int wn = wave % WN, wm = wave / WN;
    int e = 0, p0, end = a.M;
    int n_tile;
    if (a.offsets) {
        if (!find_run(a.offsets, a.E, BM, n_tiles, n_tile, e, p0, end, s_run)) return;
    } else {
        // (in strips of eight tiles of x)
        const int id = xcd_tile(blockIdx.x, n_tiles * m_tiles);
        const int strip = id / (8 * n_tiles), wide = min(8, m_tiles - 8 * strip), in = id - strip * 8 * n_tiles;
        n_tile = in / wide;
        p0 = (8 * strip + in % wide) * BM;
    }
    constexpr int ROWS = GATED ? BN / 2 : BN;           // rows of y's columns
    const int n0 = n_tile * ROWS, nb = (a.K + FB - 1) / FB, whole = a.K / FB;

    // The row of chunk q of a stage: of a weight, from n0 on (a wave's rows: TN / 2 tiles of gate and as many of up), or of x; and which of its
    // chunks it is
    auto weight_row = [&](int q) FP8_INLINE {
        const int r = q >> 3;
        return min(GATED ? r / (16 * TN) * 8 * TN + r % (8 * TN) : r, a.N - 1 - n0);
    };
    auto is_up = [](int q) FP8_INLINE { return GATED && (q >> 3) % (16 * TN) >= 8 * TN; };
    auto x_row = [&](int q) FP8_INLINE -> int64_t {
        const int p = min(p0 + (q >> 3) - BN, end - 1);
        return a.top ? a.perm[p] / a.top : p;
    };
    auto chunk_of = [](int q) FP8_INLINE { return (q & 7) ^ (q >> 3 & 7); };
    const uint8_t *const w0 = a.m[0].w + e * a.m[0].ex + n0 * a.m[0].ld, *const w1 = GATED ? a.m[1].w + e * a.m[1].ex + n0 * a.m[1].ld : w0;
    auto row_of = [&](int q) FP8_INLINE -> const uint8_t * {
        if (q >= BN * 8) return a.x + x_row(q) * a.ldx;
        return is_up(q) ? w1 + weight_row(q) * a.m[1].ld : w0 + weight_row(q) * a.m[0].ld;
    };
    // a whole block's loads, to LDS without registers: a place that is the same for all lanes, and a lane's 32 bits from there
    const uint8_t *const x0 = a.top ? a.x : a.x + p0 * a.ldx;
    uint32_t from[CH];
    const uint8_t *src[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int q = i * THREADS + tid;
        if (NS == 1) src[i] = row_of(q) + 16 * chunk_of(q);
        else if (i * THREADS < BN * 8) from[i] = (uint32_t)(weight_row(q) * (is_up(q) ? a.m[1].ld : a.m[0].ld)) + 16 * chunk_of(q);
        else from[i] = (uint32_t)((x_row(q) - (a.top ? 0 : p0)) * a.ldx) + 16 * chunk_of(q);
    }
    auto stage = [&](int4_v *s, int b, int first, int n) FP8_INLINE {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if (i < first || i >= first + n) continue;
            // (a wave's 64 chunks are eight rows, all of gate, of up or of x)
            const uint8_t *base = (i * THREADS >= BN * 8 ? x0 : is_up(i * THREADS + 64 * wave) ? w1 : w0) + (int64_t)min(b * KG + kg, whole - 1) * FB;
            uint32_t o = from[i];
            asm volatile("" : "+v"(o));                 // (not a pointer kept for every chunk)
            __builtin_amdgcn_global_load_lds((const void *)(base + o), (__attribute__((address_space(3))) void *)(s + i * THREADS + 64 * wave), 16, 0, 0);
        }
    };
    // The scales of SB blocks, by block: of the rows of x, and of each wave's rows of the weight (of gate and up).  Read one block at a
    // time, each row's would be a line of its own for every block.
    constexpr int PER = THREADS / BM, EACH = (SB + PER - 1) / PER;
    const float *from_x, *from_w;
    {
        const int p = min(p0 + tid % BM, end - 1);
        from_x = a.xs + (int64_t)(a.top ? a.perm[p] / a.top : p) * a.ldxs;
        const int w = tid % (2 * WN) / 2;
        const Fp8Mat &m = a.m[GATED && tid % 2];
        from_w = m.s + e * m.sex + (int64_t)min((n0 + w * (GATED ? 8 : 16) * TN) / FB, (a.N - 1) / FB) * m.sld;
    }
    float held_x[EACH], held_w = 0.0f;
    auto fetch_scales = [&](int b) FP8_INLINE {          // (a step past K's whole blocks, which another group may have, counts nothing)
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = (b + tid / BM + PER * i) * KG + kg;
            held_x[i] = KG > 1 && at >= whole ? 0.0f : from_x[min(at, nb - 1)];
        }
        if (tid < SB * 2 * WN) {
            const int at = (b + tid / (2 * WN)) * KG + kg;
            held_w = KG > 1 && at >= whole ? 0.0f : from_w[min(at, nb - 1)];
        }
    };
    auto put_scales = [&](int par) FP8_INLINE {
#pragma unroll
        for (int i = 0; i < EACH; ++i)
            if (SB % PER == 0 || tid / BM + PER * i < SB) s_sx[kg][par][tid / BM + PER * i][tid % BM] = held_x[i];
        if (tid < SB * 2 * WN) s_sw[kg][par][tid / (2 * WN)][tid % (2 * WN)] = held_w;
    };
    float4_v acc[TN][TM] = {};
    auto frag = [&](const int4_v *s, int r) FP8_INLINE {
        return __builtin_shufflevector(s[r * 8 + (g ^ (r & 7))], s[r * 8 + ((4 + g) ^ (r & 7))], 0, 1, 2, 3, 4, 5, 6, 7);
    };
    struct Operands {                                   // what a wave's first row of tiles of a stage needs
        int8_v x[TM], w;
        float f0, f1, fx[TM];
    };
    auto fetch = [&](Operands &o, const int4_v *s, int par, int u) FP8_INLINE {
        o.w = frag(s, wn * TN * 16 + c);
#pragma unroll
        for (int j = 0; j < TM; ++j) o.x[j] = frag(s, BN + (wm * TM + j) * 16 + c);
        o.f0 = s_sw[kg][par][u][2 * wn];
        o.f1 = GATED ? s_sw[kg][par][u][2 * wn + 1] : 0.0f;
#pragma unroll
        for (int j = 0; j < TM; ++j) o.fx[j] = s_sx[kg][par][u][(wm * TM + j) * 16 + c];
    };
    // A stage's products, a row of tiles' while the row before is scaled and added and the row after is read; before the last row, when every
    // read of the stage is done, then(); in each row, after its products, along(row).
    // (The fp16 operands take the registers that a row's sums would wait in: 4 x 2 tiles have room for both (2,048 tokens of 128 experts 341 us,
    // 343 without), 2 x 2 lose by it (500 rows through 2,500 x 2,000 20.6 us, 21.5 so), and so does one row of tiles (64 through 4,096 x 4,096 16.3,
    // 17.3).)
    auto multiply = [&](const int4_v *s, const Operands &o, auto then, auto along) FP8_INLINE {
        half8_v xh[TM][4];
        auto convert_x = [&]() FP8_INLINE {
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) xh[j][k] = halves(o.x[j][2 * k], o.x[j][2 * k + 1]);
        };
        if (TN > 1) convert_x();
        constexpr int LAG = TM > 2 || TN < 4 ? 0 : 1;
        int8_v wf = o.w;
        float4_v d[LAG + 1][TM];
#pragma unroll
        for (int i = 0; i < TN + LAG; ++i) {
            int8_v wnext;
            if (i + 1 < TN) wnext = frag(s, (wn * TN + i + 1) * 16 + c);
            if (i == TN - 1) then();
            if (i < TN) {
                half8_v wh[4];
                if (TN == 1) convert_x();               // (one row of tiles: the registers are the next stage's operands' until here)
#pragma unroll
                for (int k = 0; k < 4; ++k) wh[k] = halves(wf[2 * k], wf[2 * k + 1]);
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    float4_v t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int k = 0; k < 4; ++k) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[k], xh[j][k], t, 0, 0, 0);
                    d[i & LAG][j] = t;
                }
            }
            if (LAG) __builtin_amdgcn_sched_barrier(0);     // first the products
            if (i < TN) along(i);
            const int l = i - LAG;
            if (l >= 0) {
                const float sw = GATED && l >= TN / 2 ? o.f1 : o.f0;
#pragma unroll
                for (int j = 0; j < TM; ++j) {
                    const float f = o.fx[j] * sw;
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[l][j][k] = fmaf(d[l & LAG][j][k], f, acc[l][j][k]);
                    asm volatile("" : "+v"(acc[l][j]));     // here, not further on, where every product would wait in registers
                }
            }
            wf = wnext;
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto nothing = []() {};
    const int n_steps = (whole + KG - 1) / KG;
    int b = 0, par = 0;
    Operands o0, o1;
    if (NS > 1 && whole) {
        // Steps stand in the code one by one, each with its own places in LDS, so that reads wait for the loads to their own place alone; at
        // the loop's head they wait for all.  At the end of K the loads are of its last block again, so that every step is alike.
        // One stage is multiplied while the loads of the NS - 1 after it are on their way.  Before its last row of tiles, when every
        // wave has read all of it, the next stage's first operands are read.  The loads stand between the rows of tiles; all of
        // them after the first take the same time (4096^3 143 us, the layer of 2,048 tokens 338, 341 so).
        constexpr int ROWS_LOAD = TN > 1 ? TN - 1 : 1, EACH_ROW = (CH + ROWS_LOAD - 1) / ROWS_LOAD, BEHIND = NS - 2 - (TN == 1);
        auto run = [&](auto live) FP8_INLINE {
            constexpr bool LIVE = decltype(live)::value;
            auto place = [&](int u) FP8_INLINE {
                u %= NS;
                return (u == 0 ? s_0 : u == 1 ? s_1 : s_2) + kg * (CHUNKS / KG);
            };
            auto step = [&](Operands &o, Operands &on, int u) FP8_INLINE {
                auto along = [&](int i) FP8_INLINE {
                    if (i < ROWS_LOAD) stage(place(u + NS - 1), b + u + NS - 1, i * EACH_ROW, EACH_ROW);
                };
                auto then = [&]() FP8_INLINE {
                    if (u == SB - 1) put_scales(par ^= 1);
                    wait_loads<CH * BEHIND>();          // the next stage is there (with one row of tiles, its step's loads come later)
                    barrier();                          // and every wave's part of it; and all have read this one
                    if (LIVE) fetch(on, place(u + 1), par, (u + 1) % SB);
                };
                if (LIVE) {
                    multiply(place(u), o, then, along);
                } else {
#pragma unroll
                    for (int i = 0; i < TN - 1; ++i) along(i);
                    then();
                    if (TN == 1) along(0);
                }
            };
            auto steps = [&](int n) FP8_INLINE {
                step(o0, o1, 0);
                if (n > 1) step(o1, o0, 1);
                if (n > 2) step(o0, o1, 2);
                if (n > 3) step(o1, o0, 3);
                if (n > 4) step(o0, o1, 4);
                if (n > 5) step(o1, o0, 5);
            };
            fetch_scales(0);
#pragma unroll
            for (int i = 0; i < NS - 1; ++i) stage(place(i), i, 0, CH);
            put_scales(0);
            wait_loads<CH * (NS - 2)>();
            barrier();
            if (LIVE) fetch(o0, place(0), 0, 0);
            for (; b + SB <= n_steps; b += SB) {
                fetch_scales(b + SB);
                steps(SB);
            }
            if (b < n_steps) steps(n_steps - b);
            wait_loads<0>();
        };
        // a wave none of whose rows of x are there only loads
        if (p0 + 16 * TM * wm < end) run(std::true_type{});
        else run(std::false_type{});
    } else {
        fetch_scales(0);
        put_scales(0);
        for (; b < whole; b += SB) {
#pragma unroll 1
            for (int u = 0; u < SB && b + u < whole; ++u) {
                int4_v held[CH];
#pragma unroll
                for (int i = 0; i < CH; ++i) held[i] = *(const int4_u *)(src[i] + (int64_t)(b + u) * FB);
                __syncthreads();                        // the stage is free
#pragma unroll
                for (int i = 0; i < CH; ++i) s_0[i * THREADS + tid] = held[i];
                __syncthreads();
                fetch(o0, s_0, par, u);
                multiply(s_0, o0, nothing, [](int) {});
            }
            if (b + SB > whole) break;
            fetch_scales(b + SB);
            put_scales(par ^= 1);
        }
    }
    if (a.K % FB) {                                     // the last block, the first group's
        __syncthreads();
        if (kg == 0) {
#pragma unroll 1
            for (int q = tid; q < (BN + BM) * 8; q += THREADS) {
                const int k = whole * FB + 16 * chunk_of(q);
                s_0[q] = load16(row_of(q) + k, a.K - k);
            }
            if (KG > 1) {
                if (tid < BM) s_sx[0][0][0][tid] = from_x[whole];
                if (tid < 2 * WN) s_sw[0][0][0][tid] = from_w[whole];
            }
        }
        __syncthreads();
        if (kg == 0) {
            fetch(o0, s_0, KG > 1 ? 0 : par, KG > 1 ? 0 : whole - b);
            multiply(s_0, o0, nothing, [](int) {});
        }
    }
    if (KG > 1) {
        float4_v *sums = (float4_v *)s_0;
        __syncthreads();
        if (kg > 0)
#pragma unroll
            for (int i = 0; i < TN; ++i)
#pragma unroll
                for (int j = 0; j < TM; ++j) sums[((kg - 1) * TN * TM + i * TM + j) * THREADS + tid] = acc[i][j];
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int i = 0; i < TN; ++i)
#pragma unroll
            for (int j = 0; j < TM; ++j)
#pragma unroll
                for (int q = 0; q < KG - 1; ++q) acc[i][j] += sums[(q * TN * TM + i * TM + j) * THREADS + tid];
    }

    if (GATED) {
        // h, and its codes: a workgroup has whole blocks of 128 of I
        static_assert(!GATED || ROWS == FB, "a block");
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < TN / 2; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int n = n0 + wn * 8 * TN + 16 * i + 4 * g + k;
                    const float h = n < a.N ? finite_or_nan(silu_times(acc[i][j][k], acc[i + TN / 2][j][k])) : 0.0f;
                    acc[i][j][k] = h;
                    m = fmaxf(m, fabsf(h));
                }
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if (g == 0) s_max[wn][(wm * TM + j) * 16 + c] = m;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TM; ++j) {
            const int col = (wm * TM + j) * 16 + c;
            const int64_t p = p0 + col;
            float m = s_max[0][col];
#pragma unroll
            for (int w = 1; w < WN; ++w) m = fmaxf(m, s_max[w][col]);
            const int ex = scale_exp(m);
            const float inv = pow2(-ex);
            if (p >= end) continue;
            if (wn == 0 && g == 0) a.hs[p * a.ldhs + n_tile] = pow2(ex);
#pragma unroll
            for (int i = 0; i < TN / 2; ++i) {
                const int n = n0 + wn * 8 * TN + 16 * i + 4 * g;
                int q = __builtin_amdgcn_cvt_pk_fp8_f32(acc[i][j][0] * inv, acc[i][j][1] * inv, 0, false);
                q = __builtin_amdgcn_cvt_pk_fp8_f32(acc[i][j][2] * inv, acc[i][j][3] * inv, q, true);
                // (ldh is a multiple of 16: four codes stay inside the row)
                if (n < a.N) *(int *)(a.hq + p * a.ldh + n) = q;
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < TM; ++j) {
        int64_t p = p0 + (wm * TM + j) * 16 + c;
        if (p >= end) continue;
        float w = 1.0f;
        if (a.pair_w) {
            p = a.perm[p];
            w = a.pair_w[p];
        }
#pragma unroll
        for (int i = 0; i < TN; ++i) {
            const int n = n0 + (wn * TN + i) * 16 + 4 * g;
            store4(a.y, p * a.ldy + n, a.y_type, a.pair_w ? acc[i][j] * w : acc[i][j], a.N - n);
        }
    }
}

template <bool GATED, int NS, int KG, int WN, int WM, int TN, int TM>
static hipError_t launch_tile_n(const Fp8Args &a, hipStream_t st) {
    constexpr int ROWS = 16 * TN * WN / (GATED ? 2 : 1), BM = 16 * TM * WM;
    const int64_t n_tiles = (a.N + ROWS - 1) / ROWS;
    // (a dispatch: whole runs, and one for each used expert that is not whole)
    const int64_t runs = a.offsets ? a.M / BM + std::min(a.E, a.M) : (a.M + BM - 1) / BM;
    hipLaunchKernelGGL((fp8_tile_kernel<GATED, NS, KG, WN, WM, TN, TM>), dim3((unsigned)(n_tiles * runs)), dim3(64 * WN * WM * KG), 0,
                       st, a, (int)n_tiles, (int)runs);
    return hipGetLastError();
}
template <bool GATED, int NS, int KG, int WN, int WM, int TN, int TM>
static hipError_t launch_tile_d(const Fp8Args &a, hipStream_t st) {
    // rows on 16 bytes, and a workgroup's within 4 GiB (those of x from a dispatch: all)
    auto near = [](const Fp8Mat &m) { return ((uintptr_t)m.w | m.ld | m.ex) % 16 == 0 && 256 * m.ld < 1ll << 32; };
    const int64_t rows = a.top ? (a.M + a.top - 1) / a.top : 256;
    if (!near(a.m[0]) || (GATED && !near(a.m[1])) || ((uintptr_t)a.x | a.ldx) % 16 || a.ldx * rows >= 1ll << 32)
        return launch_tile_n<GATED, 1, 1, WN, WM, TN, TM>(a, st);
    return launch_tile_n<GATED, NS, KG, WN, WM, TN, TM>(a, st);
}
template <bool GATED>
static hipError_t launch_tile(const Fp8Args &a, hipStream_t st) {
    if constexpr (GATED) {
        // 64 rows of x a tile up to 128 of an expert, then 128 (experts of 768 of 2,048, the layer: 12 rows 165 us and 183, 64 239 and 253,
        // 128 341 and 343, 256 573 and 556; of down 128 rows always: 12 rows 160 us with 64, 165; 64 238 and 239; 128 358 and 341)
        if (a.M <= 128ll * a.E) return launch_tile_d<true, 3, 1, 4, 2, 4, 2>(a, st);
        return launch_tile_d<true, 3, 1, 4, 2, 4, 4>(a, st);
    } else {
        return launch_tile_d<false, 3, 1, 4, 2, 4, 4>(a, st);
    }
}

hipError_t launch_fp8_product(const Fp8Args &a, hipStream_t st) {
    if (!a.offsets) {
        if (a.M <= 16) return launch_stream<OF_ALL, false, 4>(a, st);
        // 256 x 128 tiles where they are many enough for every compute unit (1,800 rows through 3,600 x 2,048: 42.4 us, 64 x 64 51; 1,024 through
        // 4,096 x 2,048 40.3 and 35); else 64 x 64 (128 through 8,192 x 2,048: 15.0, 32 x 64 18.8); else 32 x 64 with K shared, by two groups of
        // waves or from 32 blocks on by four, which are held to 128 registers and spill 24 bytes a lane (64 rows through 2,048 x 2,048: two
        // groups 10.9 us, four 11.8; 2,048 x 3,328 14.2 and 14.4; 2,048 x 4,096 16.1 and 15.6; 24 through 2,048 x 7,168 21.2 and 18.9)
        auto tiles = [&](int n, int m) { return (int64_t)((a.N + n - 1) / n) * ((a.M + m - 1) / m); };
        if (tiles(256, 128) >= 200) return launch_tile<false>(a, st);
        if (tiles(64, 64) >= 200) return launch_tile_d<false, 3, 1, 2, 2, 2, 2>(a, st);
        return a.K < 32 * FB ? launch_tile_d<false, 3, 2, 2, 2, 1, 2>(a, st) : launch_tile_d<false, 3, 4, 2, 2, 1, 2>(a, st);
    }
    if (a.tiles) return a.gated ? launch_tile<true>(a, st) : launch_tile<false>(a, st);
    return a.gated ? launch_stream<OF_DISPATCH, true, 1>(a, st) : launch_stream<OF_DISPATCH, false, 1>(a, st);
}

// out[t] = the sum over k, in order, of the rows of t's pairs; a pair whose id is no expert's has none.  Four columns a thread, four rows on
// their way at once: 22 us for 2,048 tokens of eight rows of 2,048 (6.5 TB/s).
__global__ __launch_bounds__(256) void fp8_combine_kernel(Fp8CombineArgs a) {
    const int h = 4 * (blockIdx.x * 256 + threadIdx.x), n = a.H - h;
    const int64_t t = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
    if (n <= 0 || t >= a.n_tok) return;
    const int32_t *ids = a.ids + t * a.K;
    const float *rows = a.rows + t * a.K * a.H + h;
    float4_v s = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < a.K; k0 += 4) {
        float4_v v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[k] = float4_v{0.0f, 0.0f, 0.0f, 0.0f};
            if (k0 + k >= a.K || (uint32_t)ids[k0 + k] >= (uint32_t)a.E) continue;
            const float *p = rows + (int64_t)(k0 + k) * a.H;
            if (n >= 4) __builtin_memcpy(&v[k], p, 16);
            else
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (i < n) v[k][i] = p[i];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) s += v[k];
    }
    store4(a.out, t * a.ldo + h, a.out_type, s, n);
}
hipError_t launch_fp8_combine(const Fp8CombineArgs &a, hipStream_t st) {
    const unsigned y = (unsigned)(a.n_tok < 32768 ? a.n_tok : 32768);
    hipLaunchKernelGGL(fp8_combine_kernel, dim3((unsigned)((a.H + 1023) / 1024), y, (unsigned)((a.n_tok + y - 1) / y)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace mp
