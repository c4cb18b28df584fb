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

constexpr int NORM_MAX_WAVES = 16;

template <int N> struct Vals { float v[N]; };         // N elements of a row

// Where a thread's elements lie: with WHOLE, N neighbouring ones at a time, in one vector (every row at whole
// vectors, H a multiple of N); without, a workgroup's width apart, which keeps the single loads of a wave together.
template <bool WHOLE, int N>
__device__ inline int place(int j, int e) {
    const int tid = (int)threadIdx.x, width = (int)blockDim.x;
    return WHOLE ? N * (tid + width * j) + e : tid + width * (N * j + e);
}
// the thread's j-th elements of the row at o (0 beyond H)
template <int T, bool WHOLE, int N>
__device__ inline Vals<N> load_n(const void *row, int64_t o, int j, int H) {
    typedef typename Elem<T>::raw raw;
    const raw *p = (const raw *)row + o;
    struct alignas(N * sizeof(raw) < 16 ? N * sizeof(raw) : 16) Vec { raw v[N]; } q;
    Vals<N> f;
    if constexpr (WHOLE) {
        q = *(const Vec *)(p + place<WHOLE, N>(j, 0));
#pragma unroll
        for (int e = 0; e < N; ++e) f.v[e] = Elem<T>::load(q.v[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) q.v[e] = p[min(place<WHOLE, N>(j, e), H - 1)];      // (no branch: the loads go out together)
#pragma unroll
        for (int e = 0; e < N; ++e) f.v[e] = place<WHOLE, N>(j, e) < H ? Elem<T>::load(q.v[e]) : 0.0f;
    }
    return f;
}
template <int T, bool WHOLE, int N>
__device__ inline void store_n(void *row, int64_t o, int j, int H, const Vals<N> &f) {
    typedef typename Elem<T>::raw raw;
    raw *p = (raw *)row + o;
    struct alignas(N * sizeof(raw) < 16 ? N * sizeof(raw) : 16) Vec { raw v[N]; } q;
    if constexpr (WHOLE) {
#pragma unroll
        for (int e = 0; e < N; ++e) q.v[e] = Elem<T>::store(f.v[e]);
        *(Vec *)(p + place<WHOLE, N>(j, 0)) = q;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (place<WHOLE, N>(j, e) < H) p[place<WHOLE, N>(j, e)] = Elem<T>::store(f.v[e]);
    }
}
// f32 or T
template <int T, bool WHOLE, int N>
__device__ inline Vals<N> load_or(int type, const void *row, int64_t o, int j, int H) {
    return type == T_F32 ? load_n<T_F32, WHOLE, N>(row, o, j, H) : load_n<T, WHOLE, N>(row, o, j, H);
}

template <int N, class F>
__device__ inline Vals<N> each(Vals<N> a, F f) {
#pragma unroll
    for (int e = 0; e < N; ++e) a.v[e] = f(a.v[e]);
    return a;
}
template <int N, class F>
__device__ inline Vals<N> each(Vals<N> a, const Vals<N> &b, F f) {
#pragma unroll
    for (int e = 0; e < N; ++e) a.v[e] = f(a.v[e], b.v[e]);
    return a;
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
template <bool WHOLE, int N, int NV>
__device__ inline void moments(const Vals<N> (&z)[NV], int H, int kind, float eps, float (*s)[NORM_MAX_WAVES], float &mu,
                               float &inv) {
    mu = 0.0f;
    if (kind == 1) {
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (place<WHOLE, N>(j, e) < H) t += z[j].v[e];
        mu = row_sum(t, s[0]) / (float)H;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = z[j].v[e] - mu;
            if (place<WHOLE, N>(j, e) < H) q = fmaf(d, d, q);
        }
    inv = 1.0f / sqrtf(row_sum(q, s[1]) / (float)H + eps);
}

// B: the branch's type, or -1 without one
template <int T, int B, bool WHOLE, int N, int NV>
__global__ __launch_bounds__(64 * NORM_MAX_WAVES) void block_norm_kernel(NormArgs a) {
    // weights and gate are read with the row where registers hold them, else where they are used
    constexpr bool EARLY = NV * N <= (WHOLE ? 8 : 4);
    constexpr int ROWS = WHOLE && N == 4 ? 8 : 4;     // branch rows on their way at once
    __shared__ float s_sum[4][NORM_MAX_WAVES];
    const int64_t tok = blockIdx.x;
    Vals<N> z[NV], x[NV], w[NV], c[NV], p[NV], pc[NV], g[NV];
    auto in = [&](int j) { return place<WHOLE, N>(j, 0) < a.H; };
    auto vec_of = [&](const void *q, int j) { return load_or<T, WHOLE, N>(a.w_type, q, 0, j, a.H); };
    auto gate_of = [&](int j) {
        if (a.gate_col) return load_or<T, WHOLE, N>(a.gate_type, a.gate, tok * a.gate_row, j, a.H);
        const float u = a.gate_type == T_F32 ? ((const float *)a.gate)[tok * a.gate_row]
                                             : Elem<T>::load(((const typename Elem<T>::raw *)a.gate)[tok * a.gate_row]);
        Vals<N> v;
        for (int e = 0; e < N; ++e) v.v[e] = u;
        return v;
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        x[j] = z[j] = Vals<N>{};
        if (!in(j)) continue;
        x[j] = load_n<T, WHOLE, N>(a.x, tok * a.ldx, j, a.H);
        if (EARLY && a.w) w[j] = vec_of(a.w, j);
        if (EARLY && a.c) c[j] = vec_of(a.c, j);
        if (B < 0) continue;
        if (EARLY && a.pw) p[j] = vec_of(a.pw, j);
        if (EARLY && a.pc) pc[j] = vec_of(a.pc, j);
        if (EARLY && a.gate) g[j] = gate_of(j);
        const int64_t o = tok * a.n_sum * a.ldb;
        for (int k0 = 0; k0 < a.n_sum; k0 += ROWS) {
            Vals<N> b[ROWS];
#pragma unroll
            for (int k = 0; k < ROWS; ++k)
                if (k0 + k < a.n_sum) b[k] = load_n<B < 0 ? T : B, WHOLE, N>(a.branch, o + (k0 + k) * a.ldb, j, a.H);
#pragma unroll
            for (int k = 0; k < ROWS; ++k)
                if (k0 + k < a.n_sum) z[j] = k0 + k == 0 ? b[0] : each(z[j], b[k], [](float s, float v) { return s + v; });
        }
    }
    float mu, inv;
    if (B >= 0) {
        if (a.post) moments<WHOLE>(z, a.H, a.kind, a.post_eps, s_sum, mu, inv);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (!in(j)) continue;
            if (a.post) {
                z[j] = each(z[j], [&](float v) { return (v - mu) * inv; });
                if (a.pw) z[j] = each(z[j], EARLY ? p[j] : vec_of(a.pw, j), [&](float v, float u) { return v * (u + a.offset); });
                if (a.pc) z[j] = each(z[j], EARLY ? pc[j] : vec_of(a.pc, j), [](float v, float u) { return v + u; });
            }
            if (a.gate) {
                if (!EARLY) g[j] = gate_of(j);
                if (a.gate_act == 1) g[j] = each(g[j], [](float u) { return 1.0f / (1.0f + expf(-u)); });
                z[j] = each(z[j], g[j], [](float v, float u) { return v * u; });
            }
            z[j] = each(z[j], x[j], [&](float v, float u) { return fmaf(a.scale, v, u); });
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) z[j] = x[j];
    }
    if (a.r)
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in(j)) store_n<T, WHOLE, N>(a.r, tok * a.ldr, j, a.H, z[j]);
    if (!a.y) return;
    moments<WHOLE>(z, a.H, a.kind, a.eps, s_sum + 2, mu, inv);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (!in(j)) continue;
        Vals<N> y = each(z[j], [&](float v) { return (v - mu) * inv; });
        if (a.w) y = each(y, EARLY ? w[j] : vec_of(a.w, j), [&](float v, float u) { return v * (u + a.offset); });
        if (a.c) y = each(y, EARLY ? c[j] : vec_of(a.c, j), [](float v, float u) { return v + u; });
        if (a.y_type == T_F32) store_n<T_F32, WHOLE, N>(a.y, tok * a.ldy, j, a.H, y);
        else store_n<T, WHOLE, N>(a.y, tok * a.ldy, j, a.H, y);
    }
}

template <int T, int B, bool WHOLE, int N>
static hipError_t launch_norm_n(const NormArgs &a, hipStream_t st) {
    // N elements a thread, up to 1,024 threads; more elements a thread beyond that
    const int groups = (a.H + N - 1) / N, nv = groups <= 1024 ? 1 : groups <= 2048 ? 2 : 4;
    const dim3 grid((unsigned)a.n_tok), block((unsigned)(((groups + nv - 1) / nv + 63) / 64 * 64));
    if (nv == 1) hipLaunchKernelGGL((block_norm_kernel<T, B, WHOLE, N, 1>), grid, block, 0, st, a);
    else if (nv == 2) hipLaunchKernelGGL((block_norm_kernel<T, B, WHOLE, N, 2>), grid, block, 0, st, a);
    else if constexpr (N == 4) hipLaunchKernelGGL((block_norm_kernel<T, B, WHOLE, N, 4>), grid, block, 0, st, a);
    return hipGetLastError();
}

// whether every row of every tensor begins at whole vectors of n elements (at 16 bytes if those are longer)
static bool whole_vectors(const NormArgs &a, int n) {
    auto whole = [n](const void *p, int type, int64_t ld) {
        const int size = type == T_F32 ? 4 : 2, bytes = size * n < 16 ? size * n : 16;
        return (uintptr_t)p % bytes == 0 && ld * size % bytes == 0;
    };
    return a.H % n == 0 && whole(a.x, a.x_type, a.ldx) && whole(a.branch, a.b_type, a.ldb) &&
           (!a.gate_col || whole(a.gate, a.gate_type, a.gate_row)) && whole(a.w, a.w_type, 0) && whole(a.c, a.w_type, 0) &&
           whole(a.pw, a.w_type, 0) && whole(a.pc, a.w_type, 0) && whole(a.r, a.x_type, a.ldr) && whole(a.y, a.y_type, a.ldy);
}

template <int T, int B>
static hipError_t launch_norm_b(const NormArgs &a, hipStream_t st) {
    // eight elements a thread where x and the branch are of 16 bits: half the waves, whole 16-byte loads
    if constexpr (T != T_F32 && B != T_F32)
        if (whole_vectors(a, 8)) return launch_norm_n<T, B, true, 8>(a, st);
    return whole_vectors(a, 4) ? launch_norm_n<T, B, true, 4>(a, st) : launch_norm_n<T, B, false, 4>(a, st);
}
template <int T>
static hipError_t launch_norm_t(const NormArgs &a, hipStream_t st) {
    if (!a.branch) return launch_norm_b<T, -1>(a, st);
    return a.b_type == T_F32 ? launch_norm_b<T, T_F32>(a, st) : launch_norm_b<T, T>(a, st);
}

hipError_t launch_block_norm(const NormArgs &a, hipStream_t st) {
    return a.x_type == T_F32 ? launch_norm_t<T_F32>(a, st)
         : a.x_type == T_BF16 ? launch_norm_t<T_BF16>(a, st) : launch_norm_t<T_F16>(a, st);
}

}  // namespace mp
