// mp_norm.hip -- the residual stream between two blocks (moe_block_norm): the
// sum of a token's branch rows, the norm after the block, its gate, the
// residual scale and add, and the norm before the next block, in one launch.
//
// Every element is read once and stays in registers between the sums over its
// row: a workgroup has a row, a thread eight neighbouring elements of it (or twice
// that), so that all of a row's loads are on their way at once, those of the
// weights and the gate too.  Sums are f32: up to sixteen terms a thread, a wave's
// by DPP, the waves' through LDS, one barrier each.  A layer norm's squares are
// taken about the mean, in a second pass over the registers: sums of squares lose
// the small variance of a row far from 0.
// Large calls are bound by memory: 4,096 tokens of eight f32 rows, hidden 2048,
// bf16, 319 MB in 60 to 62 us (5.2 TB/s; a copy of 2 GiB reaches 4.9, a read 6.3), 8,191 bf16 rows alone 67 MB in
// 15.7 (4.3; 13.6 where the same rows are read each time).  Wide rows with both norms and a full gate stay further
// from it: 4,096 of 4,096, fp16 layer norms, 168 MB in 59 (2.8), of 4,095 in 69 (2.4).  Small ones are bound by the
// launch and two trips to memory: one token 3.5 us.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

constexpr int NORM_MAX_WAVES = 16;

template <int N> struct Vals { float v[N]; };         // N elements of a row

// A thread's j-th N elements are the row's from N (tid + width j) on.  Where H is no multiple of N (not WHOLE) the last thread's
// are the row's last N: the ones before its own are another thread's, too, and do not count in its sums.
template <int N>
__device__ inline int own(int j) { return N * ((int)threadIdx.x + (int)blockDim.x * j); }
template <bool WHOLE, int N>
__device__ inline int place(int j, int H) { return WHOLE ? own<N>(j) : min(own<N>(j), H - N); }
// One load or store at the element's own alignment: what a vector off its boundary costs is the line that it spreads into
// (8,191 rows of 2048 bf16 and a branch, x's rows an odd number of elements apart: 31 us, 29 of whole vectors, 55 of single elements).
template <int T, int N>
__device__ inline Vals<N> load_n(const void *row, int64_t o) {
    typename Elem<T>::raw q[N];
    __builtin_memcpy(q, (const typename Elem<T>::raw *)row + o, sizeof q);
    Vals<N> f;
#pragma unroll
    for (int e = 0; e < N; ++e) f.v[e] = Elem<T>::load(q[e]);
    return f;
}
template <int T, int N>
__device__ inline void store_n(void *row, int64_t o, const Vals<N> &f) {
    typename Elem<T>::raw q[N];
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = Elem<T>::store(f.v[e]);
    __builtin_memcpy((typename Elem<T>::raw *)row + o, q, sizeof q);
}
// f32 or T
template <int T, int N>
__device__ inline Vals<N> load_or(int type, const void *row, int64_t o) {
    return type == T_F32 ? load_n<T_F32, N>(row, o) : load_n<T, N>(row, o);
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
    auto counts = [H](int j, int e) { return own<N>(j) < H && (WHOLE || place<WHOLE, N>(j, H) + e >= own<N>(j)); };
    mu = 0.0f;
    if (kind == 1) {
        float t = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (counts(j, e)) t += z[j].v[e];
        mu = row_sum(t, s[0]) / (float)H;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float d = z[j].v[e] - mu;
            if (counts(j, e)) q = fmaf(d, d, q);
        }
    inv = 1.0f / sqrtf(row_sum(q, s[1]) / (float)H + eps);
}

// B: the branch's type, or -1 without one
template <int T, int B, bool WHOLE, int N, int NV>
__global__ __launch_bounds__(64 * NORM_MAX_WAVES) void block_norm_kernel(NormArgs a) {
    // weights and gate are read with the row where registers hold them, else where they are used
    constexpr bool EARLY = NV == 1;
    constexpr int ROWS = 4;                               // branch rows on their way at once
    __shared__ float s_sum[4][NORM_MAX_WAVES];
    const int64_t tok = blockIdx.x;
    Vals<N> z[NV], x[NV], w[NV], c[NV], p[NV], pc[NV], g[NV];
    auto in = [&](int j) { return own<N>(j) < a.H; };
    auto at = [&](int j) { return place<WHOLE, N>(j, a.H); };
    auto vec_of = [&](const void *q, int j) { return load_or<T, N>(a.w_type, q, at(j)); };
    auto gate_of = [&](int j) {
        if (a.gate_col) return load_or<T, N>(a.gate_type, a.gate, tok * a.gate_row + at(j));
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
        x[j] = load_n<T, N>(a.x, tok * a.ldx + at(j));
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
                if (k0 + k < a.n_sum) b[k] = load_n<B < 0 ? T : B, N>(a.branch, o + (k0 + k) * a.ldb + at(j));
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
    if (a.r) {
        if (!WHOLE) __syncthreads();                  // r may be x, whose last elements two threads read
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (in(j)) store_n<T, N>(a.r, tok * a.ldr + at(j), z[j]);
    }
    if (!a.y) return;
    moments<WHOLE>(z, a.H, a.kind, a.eps, s_sum + 2, mu, inv);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (!in(j)) continue;
        Vals<N> y = each(z[j], [&](float v) { return (v - mu) * inv; });
        if (a.w) y = each(y, EARLY ? w[j] : vec_of(a.w, j), [&](float v, float u) { return v * (u + a.offset); });
        if (a.c) y = each(y, EARLY ? c[j] : vec_of(a.c, j), [](float v, float u) { return v + u; });
        if (a.y_type == T_F32) store_n<T_F32, N>(a.y, tok * a.ldy + at(j), y);
        else store_n<T, N>(a.y, tok * a.ldy + at(j), y);
    }
}

template <int T, int B, bool WHOLE, int N, int NV>
static hipError_t launch_norm_n(const NormArgs &a, hipStream_t st) {
    const int threads = ((a.H + N - 1) / N + NV - 1) / NV;
    hipLaunchKernelGGL((block_norm_kernel<T, B, WHOLE, N, NV>), dim3((unsigned)a.n_tok), dim3((unsigned)((threads + 63) / 64 * 64)),
                       0, st, a);
    return hipGetLastError();
}
template <int T, int B>
static hipError_t launch_norm_b(const NormArgs &a, hipStream_t st) {
    // Eight elements a thread, up to 1,024 threads, then sixteen.  8,191 rows of 2048 bf16, the same each time: 13.6 us alone, 29 with a bf16
    // branch and 33 with an f32 one; of four elements, twice the waves with half the bytes on their way, 20.7, 38 and 37.
    // A row shorter than eight is read by elements.
    static_assert(MAX_NORM_H <= 2 * 8 * 64 * NORM_MAX_WAVES, "two vectors a thread");
    if (a.H < 8) return launch_norm_n<T, B, true, 1, 1>(a, st);
    const bool whole = a.H % 8 == 0;
    if (a.H <= 8 * 64 * NORM_MAX_WAVES)
        return whole ? launch_norm_n<T, B, true, 8, 1>(a, st) : launch_norm_n<T, B, false, 8, 1>(a, st);
    return whole ? launch_norm_n<T, B, true, 8, 2>(a, st) : launch_norm_n<T, B, false, 8, 2>(a, st);
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
