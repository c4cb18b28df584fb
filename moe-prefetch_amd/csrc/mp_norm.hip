// mp_norm.hip -- the residual stream between two blocks (moe_block_norm): the
// sum of a token's branch rows, the norm after the block, its gate, the
// residual scale and add, and the norm before the next block, in one launch.
//
// Every element is read once and stays in registers between the sums over its
// row: a workgroup has a row, a thread four neighbouring elements of it (up to
// four times), so that all of a row's loads are on their way at once, those of
// the weights and the gate too.  Sums are f32: four to sixteen terms a thread, a
// wave's by DPP, the waves' through LDS, one barrier each.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

constexpr int NORM_MAX_WAVES = 16, NORM_ROWS = 8;     // branch rows on their way at once

struct alignas(8) Half4 { uint16_t v[4]; };

// elements i .. i + 3 of a row (those below H; zero from there on); vec: the row may be read in whole vectors
template <int T>
__device__ inline float4 load4(const void *row, int64_t o, int i, int H, bool vec) {
    typedef typename Elem<T>::raw raw;
    const raw *p = (const raw *)row + o + i;
    if (vec && i + 4 <= H) {
        if constexpr (T == T_F32) {
            return *(const float4 *)p;
        } else {
            const Half4 q = *(const Half4 *)p;
            return make_float4(Elem<T>::load(q.v[0]), Elem<T>::load(q.v[1]), Elem<T>::load(q.v[2]), Elem<T>::load(q.v[3]));
        }
    }
    float f[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = i + e < H ? Elem<T>::load(p[e]) : 0.0f;
    return make_float4(f[0], f[1], f[2], f[3]);
}
template <int T>
__device__ inline void store4(void *row, int64_t o, int i, int H, bool vec, float4 v) {
    typedef typename Elem<T>::raw raw;
    raw *p = (raw *)row + o + i;
    if (vec && i + 4 <= H) {
        if constexpr (T == T_F32) *(float4 *)p = v;
        else *(Half4 *)p = Half4{{Elem<T>::store(v.x), Elem<T>::store(v.y), Elem<T>::store(v.z), Elem<T>::store(v.w)}};
        return;
    }
    const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < H) p[e] = Elem<T>::store(f[e]);
}
// f32 or T
template <int T>
__device__ inline float4 load4_or(int type, const void *row, int64_t o, int i, int H, bool vec) {
    return type == T_F32 ? load4<T_F32>(row, o, i, H, vec) : load4<T>(row, o, i, H, vec);
}

template <class F>
__device__ inline float4 each4(float4 a, F f) { return make_float4(f(a.x), f(a.y), f(a.z), f(a.w)); }
template <class F>
__device__ inline float4 each4(float4 a, float4 b, F f) {
    return make_float4(f(a.x, b.x), f(a.y, b.y), f(a.z, b.z), f(a.w, b.w));
}

// the sum of v over the workgroup, the same bits on every thread; s: LDS words of this sum alone
__device__ inline float row_sum(float v, float *s) {
    v = wave_sum_canon(v);
    const int waves = (int)blockDim.x >> 6;
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = s[0];
    for (int i = 1; i < waves; ++i) t += s[i];
    return t;
}

// the mean (layer norms) and 1 / sqrt(mean square about it + eps) of a row held in z, two passes over registers
template <int NV>
__device__ inline void moments(const float4 (&z)[NV], int H, int kind, float eps, float (*s)[NORM_MAX_WAVES], float &mu,
                               float &inv) {
    mu = 0.0f;
    if (kind == 1) {
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = 4 * ((int)threadIdx.x + (int)blockDim.x * j);
            const float d[4] = {z[j].x, z[j].y, z[j].z, z[j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (i + e < H) t += d[e];
        }
        mu = row_sum(t, s[0]) / (float)H;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = 4 * ((int)threadIdx.x + (int)blockDim.x * j);
        const float d[4] = {z[j].x - mu, z[j].y - mu, z[j].z - mu, z[j].w - mu};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (i + e < H) q = fmaf(d[e], d[e], q);
    }
    inv = 1.0f / sqrtf(row_sum(q, s[1]) / (float)H + eps);
}

// B: the branch's type, or -1 without one
template <int T, int B, int NV>
__global__ __launch_bounds__(64 * NORM_MAX_WAVES) void block_norm_kernel(NormArgs a) {
    // weights and gate are read with the row where registers hold them, else where they are used
    constexpr bool EARLY = NV <= 2;
    __shared__ float s_sum[4][NORM_MAX_WAVES];
    const int64_t tok = blockIdx.x;
    int at[NV];
    float4 z[NV], x[NV], w[NV], c[NV], p[NV], pc[NV], g[NV];
    auto vec_of = [&](const void *q, int j) { return load4_or<T>(a.w_type, q, 0, at[j], a.H, a.vec & NORM_VEC_W); };
    auto gate_of = [&](int j) {
        if (a.gate_col) return load4_or<T>(a.gate_type, a.gate, tok * a.gate_row, at[j], a.H, a.vec & NORM_VEC_G);
        const float u = a.gate_type == T_F32 ? ((const float *)a.gate)[tok * a.gate_row]
                                             : Elem<T>::load(((const typename Elem<T>::raw *)a.gate)[tok * a.gate_row]);
        return make_float4(u, u, u, u);
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = at[j] = 4 * ((int)threadIdx.x + (int)blockDim.x * j);
        if (i >= a.H) {
            x[j] = z[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            continue;
        }
        x[j] = load4<T>(a.x, tok * a.ldx, i, a.H, a.vec & NORM_VEC_X);
        if (EARLY && a.w) w[j] = vec_of(a.w, j);
        if (EARLY && a.c) c[j] = vec_of(a.c, j);
        if (B < 0) continue;
        if (EARLY && a.pw) p[j] = vec_of(a.pw, j);
        if (EARLY && a.pc) pc[j] = vec_of(a.pc, j);
        if (EARLY && a.gate) g[j] = gate_of(j);
        int64_t o = tok * a.n_sum * a.ldb;
        for (int k0 = 0; k0 < a.n_sum; k0 += NORM_ROWS) {
            float4 b[NORM_ROWS];
#pragma unroll
            for (int k = 0; k < NORM_ROWS; ++k)
                if (k0 + k < a.n_sum) b[k] = load4<B < 0 ? T : B>(a.branch, o + (k0 + k) * a.ldb, i, a.H, a.vec & NORM_VEC_B);
#pragma unroll
            for (int k = 0; k < NORM_ROWS; ++k)
                if (k0 + k < a.n_sum) z[j] = k0 + k == 0 ? b[0] : each4(z[j], b[k], [](float s, float v) { return s + v; });
        }
    }
    float mu, inv;
    if (B >= 0) {
        if (a.post) moments(z, a.H, a.kind, a.post_eps, s_sum, mu, inv);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (at[j] >= a.H) continue;
            if (a.post) {
                z[j] = each4(z[j], [&](float v) { return (v - mu) * inv; });
                if (a.pw) z[j] = each4(z[j], EARLY ? p[j] : vec_of(a.pw, j), [&](float v, float u) { return v * (u + a.offset); });
                if (a.pc) z[j] = each4(z[j], EARLY ? pc[j] : vec_of(a.pc, j), [](float v, float u) { return v + u; });
            }
            if (a.gate) {
                if (!EARLY) g[j] = gate_of(j);
                if (a.gate_act == 1) g[j] = each4(g[j], [](float u) { return 1.0f / (1.0f + expf(-u)); });
                z[j] = each4(z[j], g[j], [](float v, float u) { return v * u; });
            }
            z[j] = each4(z[j], x[j], [&](float v, float u) { return fmaf(a.scale, v, u); });
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) z[j] = x[j];
    }
    if (a.r)
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (at[j] < a.H) store4<T>(a.r, tok * a.ldr, at[j], a.H, a.vec & NORM_VEC_R, z[j]);
    if (!a.y) return;
    moments(z, a.H, a.kind, a.eps, s_sum + 2, mu, inv);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (at[j] >= a.H) continue;
        float4 y = each4(z[j], [&](float v) { return (v - mu) * inv; });
        if (a.w) y = each4(y, EARLY ? w[j] : vec_of(a.w, j), [&](float v, float u) { return v * (u + a.offset); });
        if (a.c) y = each4(y, EARLY ? c[j] : vec_of(a.c, j), [](float v, float u) { return v + u; });
        if (a.y_type == T_F32) store4<T_F32>(a.y, tok * a.ldy, at[j], a.H, a.vec & NORM_VEC_Y, y);
        else store4<T>(a.y, tok * a.ldy, at[j], a.H, a.vec & NORM_VEC_Y, y);
    }
}

template <int T, int B>
static hipError_t launch_norm_b(const NormArgs &a, hipStream_t st) {
    // a thread four elements, up to 1,024 threads; more elements a thread beyond that
    const int groups = (a.H + 3) / 4, nv = groups <= 1024 ? 1 : groups <= 2048 ? 2 : 4;
    const dim3 grid((unsigned)a.n_tok), block((unsigned)(((groups + nv - 1) / nv + 63) / 64 * 64));
    if (nv == 1) hipLaunchKernelGGL((block_norm_kernel<T, B, 1>), grid, block, 0, st, a);
    else if (nv == 2) hipLaunchKernelGGL((block_norm_kernel<T, B, 2>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((block_norm_kernel<T, B, 4>), grid, block, 0, st, a);
    return hipGetLastError();
}
template <int T>
static hipError_t launch_norm_t(const NormArgs &a, hipStream_t st) {
    if (!a.branch) return launch_norm_b<T, -1>(a, st);
    return a.b_type == T_F32 ? launch_norm_b<T, T_F32>(a, st) : launch_norm_b<T, T>(a, st);
}

hipError_t launch_block_norm(NormArgs a, hipStream_t st) {
    // which tensors' rows all begin at whole vectors of four elements
    auto whole = [](const void *p, int type, int64_t ld) { return (uintptr_t)p % (type == T_F32 ? 16 : 8) == 0 && ld % 4 == 0; };
    a.vec = 0;
    if (whole(a.x, a.x_type, a.ldx)) a.vec |= NORM_VEC_X;
    if (whole(a.branch, a.b_type, a.ldb)) a.vec |= NORM_VEC_B;
    if (whole(a.gate, a.gate_type, a.gate_row)) a.vec |= NORM_VEC_G;
    if (whole(a.w, a.w_type, 0) && whole(a.c, a.w_type, 0) && whole(a.pw, a.w_type, 0) && whole(a.pc, a.w_type, 0))
        a.vec |= NORM_VEC_W;
    if (whole(a.r, a.x_type, a.ldr)) a.vec |= NORM_VEC_R;
    if (whole(a.y, a.y_type, a.ldy)) a.vec |= NORM_VEC_Y;
    return a.x_type == T_F32 ? launch_norm_t<T_F32>(a, st)
         : a.x_type == T_BF16 ? launch_norm_t<T_BF16>(a, st) : launch_norm_t<T_F16>(a, st);
}

}  // namespace mp
