// mp_norm.hip -- the residual stream between two blocks (moe_block_norm): the
// sum of a token's branch rows, the norm after the block, its gate, the
// residual scale and add, and the norm before the next block, in one launch.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

constexpr int NORM_THREADS = 256;

__device__ inline float load_as(const void *p, int type, int64_t i) {
    return type == T_F32 ? ((const float *)p)[i]
         : type == T_BF16 ? Elem<T_BF16>::load(((const uint16_t *)p)[i]) : Elem<T_F16>::load(((const uint16_t *)p)[i]);
}
__device__ inline void store_as(void *p, int type, int64_t i, float v) {
    if (type == T_F32) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = type == T_BF16 ? Elem<T_BF16>::store(v) : Elem<T_F16>::store(v);
}

// the sum of v over the workgroup, the same bits on every thread
__device__ inline float block_sum(float v, float *s_red) {
    v = wave_sum_canon(v);
    __syncthreads();                                  // earlier readers of s_red are done
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = s_red[0];
    for (int i = 1; i < NORM_THREADS / 64; ++i) t += s_red[i];
    return t;
}

// z - mean (layer norms) and 1 / sqrt(mean square + eps), two passes over registers
template <int N>
__device__ inline void moments(const float (&z)[N], int H, int kind, float eps, float *s_red, float &mu, float &inv) {
    mu = 0.0f;
    if (kind == 1) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < N; ++j) s += z[j];
        mu = block_sum(s, s_red) / (float)H;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float d = (int)threadIdx.x + NORM_THREADS * j < H ? z[j] - mu : 0.0f;
        q = fmaf(d, d, q);
    }
    inv = 1.0f / sqrtf(block_sum(q, s_red) / (float)H + eps);
}

// One workgroup per token, thread t holding elements t, t + 256, ... in registers.
template <int N>
__global__ __launch_bounds__(NORM_THREADS) void block_norm_kernel(NormArgs a) {
    __shared__ float s_red[NORM_THREADS / 64];
    const int64_t tok = blockIdx.x;
    float z[N];
    float mu, inv;
    if (a.branch) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int h = (int)threadIdx.x + NORM_THREADS * j;
            z[j] = 0.0f;
            if (h < a.H) {
                int64_t o = tok * a.n_sum * a.ldb + h;
                z[j] = load_as(a.branch, a.b_type, o);
                for (int k = 1; k < a.n_sum; ++k) z[j] += load_as(a.branch, a.b_type, o += a.ldb);
            }
        }
        if (a.post) moments(z, a.H, a.kind, a.post_eps, s_red, mu, inv);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int h = (int)threadIdx.x + NORM_THREADS * j;
        if (h >= a.H) { z[j] = 0.0f; continue; }
        const float x = load_as(a.x, a.x_type, tok * a.ldx + h);
        if (!a.branch) { z[j] = x; continue; }
        float p = z[j];
        if (a.post) {
            p = (p - mu) * inv * (a.pw ? load_as(a.pw, a.w_type, h) + a.offset : 1.0f);
            if (a.pc) p += load_as(a.pc, a.w_type, h);
        }
        float g = a.scale;
        if (a.gate) {
            const float u = load_as(a.gate, a.gate_type, tok * a.gate_row + (int64_t)h * a.gate_col);
            g *= a.gate_act == 1 ? 1.0f / (1.0f + expf(-u)) : u;
        }
        z[j] = fmaf(g, p, x);
    }
    if (a.r)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int h = (int)threadIdx.x + NORM_THREADS * j;
            if (h < a.H) store_as(a.r, a.x_type, tok * a.ldr + h, z[j]);
        }
    if (!a.y) return;
    moments(z, a.H, a.kind, a.eps, s_red, mu, inv);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int h = (int)threadIdx.x + NORM_THREADS * j;
        if (h >= a.H) continue;
        float y = (z[j] - mu) * inv * (a.w ? load_as(a.w, a.w_type, h) + a.offset : 1.0f);
        if (a.c) y += load_as(a.c, a.w_type, h);
        store_as(a.y, a.y_type, tok * a.ldy + h, y);
    }
}

hipError_t launch_block_norm(const NormArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)a.n_tok), block(NORM_THREADS);
    if (a.H <= 8 * NORM_THREADS) hipLaunchKernelGGL(block_norm_kernel<8>, grid, block, 0, st, a);
    else if (a.H <= 32 * NORM_THREADS) hipLaunchKernelGGL(block_norm_kernel<32>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(block_norm_kernel<64>, grid, block, 0, st, a);
    return hipGetLastError();
}

}  // namespace mp
