// mp_scored.hip -- routing by scores (moe_route_scored): softmax or sigmoid, a
// selection bias, expert groups, top-k, renormalised and scaled weights.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

constexpr int SCORED_WAVES = 4;

template <int CTRL>
__device__ inline double dpp_d(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)dpp_i<CTRL>((int)(uint32_t)b), hi = (uint32_t)dpp_i<CTRL>((int)(uint32_t)(b >> 32));
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ inline double lane_d(double v, int l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
// maximum and sum over the wave, the same bits on every lane
__device__ inline double wave_max_d(double v) {
    v = fmax(v, dpp_d<DPP_XOR1>(v));
    v = fmax(v, dpp_d<DPP_XOR2>(v));
    v = fmax(v, dpp_d<DPP_HALF_MIRROR>(v));
    v = fmax(v, dpp_d<DPP_MIRROR>(v));
    return fmax(fmax(lane_d(v, 0), lane_d(v, 16)), fmax(lane_d(v, 32), lane_d(v, 48)));
}
__device__ inline double wave_sum_d(double v) {
    v = v + dpp_d<DPP_XOR1>(v);
    v = v + dpp_d<DPP_XOR2>(v);
    v = v + dpp_d<DPP_HALF_MIRROR>(v);
    v = v + dpp_d<DPP_MIRROR>(v);
    return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}

// One wave per token; lane j holds experts NV j .. NV j + NV - 1, so that of two
// equal values the one on the lower lane, or lower on the same lane, has the
// lower id.  K rounds take the largest value left.
template <int T, int NV>
__global__ __launch_bounds__(64 * SCORED_WAVES) void route_scored_kernel(ScoredArgs a) {
    __shared__ double s_s[SCORED_WAVES][64 * NV];     // scores (0: switched off)
    __shared__ double s_v[SCORED_WAVES][64 * NV];     // selection values
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * SCORED_WAVES + wave;
    const bool live = row < a.n_tok;
    const int64_t tok = live ? row : a.n_tok - 1;
    const typename Elem<T>::raw *l = (const typename Elem<T>::raw *)a.logits + tok * a.ld;
    double s[NV], v[NV];
    bool on[NV];
    double m = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int e = NV * lane + j;
        const float x = e < a.E ? Elem<T>::load(l[e]) : -INFINITY;
        on[j] = x > -INFINITY;                        // false for a NaN
        s[j] = on[j] ? (double)x : -INFINITY;
        m = fmax(m, s[j]);
    }
    if (a.score == 0) {
        m = wave_max_d(m);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            s[j] = !on[j] ? 0.0 : m == INFINITY ? (s[j] == INFINITY ? 1.0 : 0.0) : exp(s[j] - m);
            sum += s[j];
        }
        sum = wave_sum_d(sum);
#pragma unroll
        for (int j = 0; j < NV; ++j) s[j] = on[j] ? s[j] / sum : 0.0;
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) s[j] = on[j] ? 1.0 / (1.0 + exp(-s[j])) : 0.0;
    }
    if (a.scores && live)
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (NV * lane + j < a.E) a.scores[tok * a.E + NV * lane + j] = (float)s[j];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int e = NV * lane + j;
        v[j] = on[j] && a.bias ? s[j] + (double)a.bias[e] : s[j];
        if (!on[j] || !(v[j] > -INFINITY)) v[j] = -INFINITY;
        s_s[wave][e] = v[j] > -INFINITY ? s[j] : 0.0;
        s_v[wave][e] = v[j];
    }
    __syncthreads();
    if (a.groups > 1) {
        const int n = a.E / a.groups;
        double gs = -INFINITY;                        // lane g: group g's score
        if (lane < a.groups) {
            double b0 = -INFINITY, b1 = -INFINITY;
            for (int i = 0; i < n; ++i) {
                const double u = s_v[wave][lane * n + i];
                b1 = u > b0 ? b0 : fmax(b1, u);
                b0 = fmax(b0, u);
            }
            gs = a.group_best == 2 && b1 > -INFINITY ? b0 + b1 : b0;
        }
        int rank = 0;
        for (int g = 0; g < a.groups; ++g) {
            const double o = lane_d(gs, g);
            rank += o > gs || (o == gs && g < lane);
        }
        const uint64_t keep = __ballot(lane < a.groups && rank < a.top_groups);
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (!(keep >> (min(NV * lane + j, a.E - 1) / n) & 1)) {
                v[j] = -INFINITY;
                s_s[wave][NV * lane + j] = 0.0;
            }
    }
    uint32_t taken = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
        if (NV * lane + j >= a.E) taken |= 1u << j;
    int id = 0;
    for (int k = 0; k < a.K; ++k) {
        double b = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (!(taken >> j & 1)) b = fmax(b, v[j]);
        const double M = wave_max_d(b);
        // M = -inf: only experts switched off are left, every lane that has one holds it
        const bool mine = taken != (1u << NV) - 1u && b == M;
        const int win = __ffsll((unsigned long long)__ballot(mine)) - 1;
        int j0 = 0;
#pragma unroll
        for (int j = NV - 1; j >= 0; --j)
            if (!(taken >> j & 1) && v[j] == M) j0 = j;
        const int e = NV * win + __builtin_amdgcn_readlane(j0, win);
        if (lane == win) taken |= 1u << j0;
        if (lane == k) id = e;
    }
    __syncthreads();
    double w = lane < a.K ? s_s[wave][id] : 0.0;
    if (a.renorm) {
        const double sum = wave_sum_d(w);
        w = sum > 0.0 ? w / sum : 0.0;
    }
    if (live && lane < a.K) {
        const int64_t o = tok * a.K + lane;
        a.ids[o] = id;
        a.w[o] = (float)((double)a.scale * w);
        if (a.slots) a.slots[o] = a.table ? a.table[id] : a.dummy;
    }
}

template <int T>
static hipError_t launch_scored_t(const ScoredArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.n_tok + (int64_t)SCORED_WAVES - 1) / SCORED_WAVES)), block(64 * SCORED_WAVES);
    if (a.E <= 64) hipLaunchKernelGGL((route_scored_kernel<T, 1>), grid, block, 0, st, a);
    else if (a.E <= 128) hipLaunchKernelGGL((route_scored_kernel<T, 2>), grid, block, 0, st, a);
    else if (a.E <= 256) hipLaunchKernelGGL((route_scored_kernel<T, 4>), grid, block, 0, st, a);
    else if (a.E <= 512) hipLaunchKernelGGL((route_scored_kernel<T, 8>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((route_scored_kernel<T, 16>), grid, block, 0, st, a);
    return hipGetLastError();
}

hipError_t launch_route_scored(const ScoredArgs &a, hipStream_t st) {
    return a.type == T_F32 ? launch_scored_t<T_F32>(a, st)
         : a.type == T_BF16 ? launch_scored_t<T_BF16>(a, st) : launch_scored_t<T_F16>(a, st);
}

}  // namespace mp
