// mp_fp8.hip -- e4m3 weights with a scale for each block of 128 x 128: the
// quantizer (moe_fp8_quantize), products (moe_fp8_product) and a layer of experts
// (moe_fp8_layer).
//
// y[m][n] = sum over the blocks b of K of  sx[m][b] sw[n/128][b] (xq[m] . wq[n])_b:  a block's
// dot runs on the matrix cores, and one fma adds it, scaled, to the f32 sum of the row.  The weight's 16 rows are the A
// operand, so that a lane holds four of them for one row of x: one scale a lane and block.
//
// The codes become fp16 for the matrix cores (exactly), whose fp16 products are exact and their sums f32.  The cores' own e4m3
// instructions add eight neighbouring products at 13 bits below the largest of them, what is below cut off (found by
// products of powers of two: 2^-13 of the largest stays, 2^-14 does not): 1.4e-5 of the result for normal numbers, where f32 sums
// have 1e-8.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

typedef int int8_v __attribute__((ext_vector_type(8)));
typedef float float4_v __attribute__((ext_vector_type(4)));
typedef _Float16 half2_v __attribute__((ext_vector_type(2)));
typedef _Float16 half8_v __attribute__((ext_vector_type(8)));

constexpr int FB = FP8_BLOCK;

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

// n of eight elements of a row
template <int T>
__device__ inline void load8(const typename Elem<T>::raw *p, int n, float *v) {
    typename Elem<T>::raw q[8] = {};
    if (n >= 8) __builtin_memcpy(q, p, sizeof q);
    else
        for (int i = 0; i < n; ++i) q[i] = p[i];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = finite_or_nan(Elem<T>::load(q[i]));
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

// sixteen lanes a block of one row, eight neighbouring elements each
template <int T>
__global__ __launch_bounds__(256) void fp8_quant_rows_kernel(Fp8QuantArgs a) {
    const uint32_t nb = (uint32_t)((a.K + FB - 1) / FB);
    const uint64_t g = (uint64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (g >= (uint64_t)a.n_tok * nb) return;
    const int64_t row = (int64_t)(g / nb);
    const int b = (int)(g % nb), l = threadIdx.x % 16;
    const int k = b * FB + 8 * l, n = a.K - k;
    float v[8] = {};
    if (n > 0) load8<T>((const typename Elem<T>::raw *)a.x + row * a.ldx + k, n, v);
    const int e = scale_exp(max16(amax8(v, 0.0f)));
    if (n > 0) store8(a.q + row * a.ldq + k, n, codes8(v, pow2(-e)));
    if (l == 0) a.s[row * a.lds + b] = pow2(e);
}

// a workgroup a block of 128 rows
template <int T>
__global__ __launch_bounds__(256) void fp8_quant_block_kernel(Fp8QuantArgs a) {
    __shared__ float s_max[4];
    const int64_t r0 = (int64_t)blockIdx.y * FB;
    const int b = blockIdx.x, l = threadIdx.x % 16, k = b * FB + 8 * l, n = a.K - k;
    float v[8][8] = {};
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = r0 + threadIdx.x / 16 + 16 * i;
        if (n > 0 && row < a.n_tok) load8<T>((const typename Elem<T>::raw *)a.x + row * a.ldx + k, n, v[i]);
        m = amax8(v[i], m);
    }
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
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
    const int64_t nb = (a.K + FB - 1) / FB;
    if (a.rows == 1)
        hipLaunchKernelGGL((fp8_quant_rows_kernel<T>), dim3((unsigned)((a.n_tok * nb + 15) / 16)), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((fp8_quant_block_kernel<T>), dim3((unsigned)nb, (unsigned)((a.n_tok + FB - 1) / FB)), dim3(256), 0, st, a);
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
__device__ inline float4_v mfma_block(int8_v w, int8_v x) {
    float4_v d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(w[i], w[i + 1]), halves(x[i], x[i + 1]), d, 0, 0, 0);
    return d;
}

// A lane's 32 of the 128 codes of a row's block: bytes 16 g .. and 64 + 16 g .., g = lane / 16 (which codes meet which is the same
// for both operands).  n: bytes of the row from here on; codes past it are zeros.
__device__ inline uint4 load16(const uint8_t *p, int n) {
    uint64_t v[2] = {0, 0};
    if (n >= 16) __builtin_memcpy(v, p, 16);
    else {
        for (int i = min(n, 8) - 1; i >= 0; --i) v[0] = v[0] << 8 | p[i];
        for (int i = n - 1; i >= 8; --i) v[1] = v[1] << 8 | p[i];
    }
    return make_uint4((uint32_t)v[0], (uint32_t)(v[0] >> 32), (uint32_t)v[1], (uint32_t)(v[1] >> 32));
}
__device__ inline int8_v load_frag(const uint8_t *row, int k, int K, int g) {
    const uint4 a = load16(row + k + 16 * g, K - k - 16 * g), b = load16(row + k + 64 + 16 * g, K - k - 64 - 16 * g);
    return int8_v{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

__device__ inline void store_elem(void *p, int64_t i, int type, float v) {
    if (type == T_F32) ((float *)p)[i] = v;
    else if (type == T_BF16) ((uint16_t *)p)[i] = Elem<T_BF16>::store(v);
    else ((uint16_t *)p)[i] = Elem<T_F16>::store(v);
}

__device__ inline float silu_times(float g, float u) { return u * (g / (1.0f + expf(-g))); }

// Sixteen rows of a weight (of gate and up: GATED), sixteen rows of x at a time; four waves, every fourth block of K each, whose sums
// are added in their order.
template <bool GATED>
__global__ __launch_bounds__(256) void fp8_stream_kernel(Fp8Args a) {
    __shared__ float s_acc[2][4][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, c = lane & 15;
    const int e = blockIdx.y, n0 = blockIdx.x * 16;
    const int begin = a.offsets ? a.offsets[e] : 0, end = a.offsets ? a.offsets[e + 1] : a.M;
    const int nb = (a.K + FB - 1) / FB;
    const int64_t wrow = min(n0 + c, a.N - 1);
    const uint8_t *w0 = a.m[0].w + e * a.m[0].ex + wrow * a.m[0].ld;
    const float *s0 = a.m[0].s + e * a.m[0].sex + (int64_t)(n0 / FB) * a.m[0].sld;
    const uint8_t *w1 = nullptr;
    const float *s1 = nullptr;
    if (GATED) {
        w1 = a.m[1].w + e * a.m[1].ex + wrow * a.m[1].ld;
        s1 = a.m[1].s + e * a.m[1].sex + (int64_t)(n0 / FB) * a.m[1].sld;
    }
    for (int64_t p0 = begin + 16ll * blockIdx.z; p0 < end; p0 += 16ll * gridDim.z) {
        const int64_t p = p0 + c < end ? p0 + c : end - 1;
        const int64_t xrow = a.top ? a.perm[p] / a.top : p;
        const uint8_t *x = a.x + xrow * a.ldx;
        const float *xs = a.xs + xrow * a.ldxs;
        float4_v t0 = {}, t1 = {};
        for (int b = wave; b < nb; b += 4) {
            const int8_v xf = load_frag(x, b * FB, a.K, g);
            const float s = xs[b];
            const float4_v d0 = mfma_block(load_frag(w0, b * FB, a.K, g), xf);
            for (int i = 0; i < 4; ++i) t0[i] = fmaf(d0[i], s * s0[b], t0[i]);
            if (GATED) {
                const float4_v d1 = mfma_block(load_frag(w1, b * FB, a.K, g), xf);
                for (int i = 0; i < 4; ++i) t1[i] = fmaf(d1[i], s * s1[b], t1[i]);
            }
        }
        __syncthreads();
        for (int i = 0; i < 4; ++i) {
            s_acc[0][wave][c][4 * g + i] = t0[i];
            if (GATED) s_acc[1][wave][c][4 * g + i] = t1[i];
        }
        __syncthreads();
        const int r = threadIdx.x & 15, col = threadIdx.x >> 4;
        if (n0 + r >= a.N || p0 + col >= end) continue;
        float y = s_acc[0][0][col][r];
        for (int i = 1; i < 4; ++i) y += s_acc[0][i][col][r];
        if (GATED) {
            float u = s_acc[1][0][col][r];
            for (int i = 1; i < 4; ++i) u += s_acc[1][i][col][r];
            y = silu_times(y, u);
        }
        int64_t out = p0 + col;
        if (a.pair_w) {
            out = a.perm[out];
            y *= a.pair_w[out];
        }
        store_elem(a.y, out * a.ldy + n0 + r, a.y_type, y);
    }
}

hipError_t launch_fp8_product(const Fp8Args &a, hipStream_t st) {
    const int64_t chunks = a.offsets ? 4 : (a.M + 15) / 16;
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)a.E, (unsigned)(chunks < 1024 ? chunks : 1024));
    if (a.gated) hipLaunchKernelGGL((fp8_stream_kernel<true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((fp8_stream_kernel<false>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// out[t] = the sum over k, in order, of the rows of t's pairs; a pair whose id is no expert's has none
__global__ __launch_bounds__(256) void fp8_combine_kernel(Fp8CombineArgs a) {
    const int h = blockIdx.x * 256 + threadIdx.x;
    const int64_t t = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
    if (h >= a.H || t >= a.n_tok) return;
    float s = 0.0f;
    for (int k = 0; k < a.K; ++k) {
        const int64_t i = t * a.K + k;
        if ((uint32_t)a.ids[i] < (uint32_t)a.E) s += a.rows[i * a.H + h];
    }
    store_elem(a.out, t * a.ldo + h, a.out_type, s);
}
hipError_t launch_fp8_combine(const Fp8CombineArgs &a, hipStream_t st) {
    const unsigned y = (unsigned)(a.n_tok < 32768 ? a.n_tok : 32768);
    hipLaunchKernelGGL(fp8_combine_kernel, dim3((unsigned)((a.H + 255) / 256), y, (unsigned)((a.n_tok + y - 1) / y)), dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace mp
