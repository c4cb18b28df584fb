// mp_scored.hip -- routing by scores (moe_route_scored): softmax or sigmoid, a
// selection bias, expert groups, top-k, renormalised and scaled weights.
//
// One wave per token; lane j holds experts NV j .. NV j + NV - 1, so that of two
// equal values the one on the lower lane, or earlier on the same lane, has the
// lower id.  Scores and selection values are f64: two experts' order, and a
// group's, has to be that of the definition however near they are.  The K best
// come out in K rounds of a wave maximum over the lanes' best; a round compares the
// upper words and looks at the lower ones only where two lanes agree in them.
// One token of 256 experts in 8 groups, 8 chosen: 4.7 us, launch and latency.  8,191
// of them: 15 us a call among others for 8.9 MB (1.4 at the rate of a large read), of which the instructions of
// eight waves a SIMD are 13.3: about 5 for the scores in f64, 3 for the groups and 4.5
// for the rounds (K = 1: 8.2 us a call).  512 experts: 7.9 us one token, 33 for 8,191; 1,024, whose lanes order sixteen
// values each, 28 and 137.
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
// sum over the wave, the same bits on every lane
__device__ inline double wave_sum_d(double v) {
    v = v + dpp_d<DPP_XOR1>(v);
    v = v + dpp_d<DPP_XOR2>(v);
    v = v + dpp_d<DPP_HALF_MIRROR>(v);
    v = v + dpp_d<DPP_MIRROR>(v);
    return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}
// e^x for x <= 0 in 64 bits, within 2^-52: e^r to r^13 on |r| <= ln 2 / 2 (the next term is
// below 5e-18) times a power of two, down to 0
__device__ inline double exp_d(double x) {
    constexpr double MAGIC = 6755399441055744.0;      // 1.5 * 2^52: adding it rounds to a whole number
    x = fmax(x, -800.0);
    const double m = fma(x, 1.4426950408889634074, MAGIC);
    const int n = (int)(uint32_t)__builtin_bit_cast(uint64_t, m);
    const double f = m - MAGIC;
    // ln 2 in two parts, the first so short that its product with f is exact (Cody and Waite, Software Manual for the
    // Elementary Functions, 1980)
    const double r = fma(f, -1.9082149292705877e-10, fma(f, -0.693147180369123816490, x));
    double p = 1.0 / 6227020800.0;
    p = fma(p, r, 1.0 / 479001600.0);
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, n);
}

// The order of selection values as that of unsigned 64-bit numbers: above 1 for every number but NaN, 1 for an
// expert switched off, 0 for none.
constexpr uint64_t KEY_OFF = 1;
__device__ inline uint64_t value_key(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);     // -0 as +0
    return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}

// the best two of a group that spans `lanes` (a power of two) neighbouring lanes, on each of them
__device__ inline void best_two(double &b0, double &b1, double c0, double c1) {
    b1 = fmax(fmin(b0, c0), fmax(b1, c1));
    b0 = fmax(b0, c0);
}
__device__ inline void group_best_two(double &b0, double &b1, int lanes) {
    // quads hold one pair after two steps, eights after three: the mirrors reach another's
    if (lanes > 1) best_two(b0, b1, dpp_d<DPP_XOR1>(b0), dpp_d<DPP_XOR1>(b1));
    if (lanes > 2) best_two(b0, b1, dpp_d<DPP_XOR2>(b0), dpp_d<DPP_XOR2>(b1));
    if (lanes > 4) best_two(b0, b1, dpp_d<DPP_HALF_MIRROR>(b0), dpp_d<DPP_HALF_MIRROR>(b1));
    if (lanes > 8) best_two(b0, b1, dpp_d<DPP_MIRROR>(b0), dpp_d<DPP_MIRROR>(b1));
    if (lanes > 16) best_two(b0, b1, __shfl_xor(b0, 16, 64), __shfl_xor(b1, 16, 64));
}

template <int T, int NV>
__global__ __launch_bounds__(64 * SCORED_WAVES) void route_scored_kernel(ScoredArgs a) {
    __shared__ double s_s[SCORED_WAVES][64 * NV];     // scores
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * SCORED_WAVES + wave;
    if (row >= a.n_tok) return;                       // (a wave's LDS is its own: no barrier)
    const int64_t tok = row;
    typedef typename Elem<T>::raw raw;
    const raw *l = (const raw *)a.logits + tok * a.ld;
    double s[NV], v[NV];
    bool on[NV];
    float x[NV], bias[NV];
    if (a.vec) {
        const bool in = NV * lane < a.E;
        raw q[NV] = {};
        float b[NV] = {};
        if (in) __builtin_memcpy(q, l + NV * lane, sizeof q);     // (vectors at the element's own alignment)
        if (in && a.bias) __builtin_memcpy(b, a.bias + NV * lane, sizeof b);
#pragma unroll
        for (int j = 0; j < NV; ++j) { x[j] = in ? Elem<T>::load(q[j]) : -INFINITY; bias[j] = b[j]; }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = NV * lane + j;
            x[j] = e < a.E ? Elem<T>::load(l[e]) : -INFINITY;
            bias[j] = e < a.E && a.bias ? a.bias[e] : 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) on[j] = x[j] > -INFINITY;        // false for a NaN
    if (a.score == 0) {
        float mf = -INFINITY;
#pragma unroll
        for (int j = 0; j < NV; ++j) mf = fmaxf(mf, x[j]);        // passes over a NaN
        mf = wave_max(mf);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            s[j] = !on[j] ? 0.0 : mf == INFINITY ? (x[j] == INFINITY ? 1.0 : 0.0) : exp_d((double)x[j] - (double)mf);
            sum += s[j];
        }
        sum = wave_sum_d(sum);
#pragma unroll
        for (int j = 0; j < NV; ++j) s[j] = on[j] ? s[j] / sum : 0.0;
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const double e = exp_d(-fabs((double)x[j]));
            s[j] = on[j] ? (x[j] < 0.0f ? e : 1.0) / (1.0 + e) : 0.0;
        }
    }
    if (a.scores)
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (NV * lane + j < a.E) a.scores[tok * a.E + NV * lane + j] = (float)s[j];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        v[j] = on[j] ? s[j] + (double)bias[j] : -INFINITY;
        if (!(v[j] > -INFINITY)) v[j] = -INFINITY;
        s_s[wave][NV * lane + j] = s[j];
    }
    if (a.groups > 1) {
        const int n = a.E / a.groups;
        if (a.group_lanes) {                          // a group is group_lanes whole lanes
            double b0 = -INFINITY, b1 = -INFINITY;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                b1 = fmax(fmin(b0, v[j]), b1);
                b0 = fmax(b0, v[j]);
            }
            group_best_two(b0, b1, a.group_lanes);
            const double gs = a.group_best == 2 && b1 > -INFINITY ? b0 + b1 : b0;
            const int mine = lane / a.group_lanes;
            int rank = 0;
            for (int g = 0; g < a.groups; ++g) {
                const double o = lane_d(gs, g * a.group_lanes);
                rank += o > gs || (o == gs && g < mine);
            }
            const bool stay = rank < a.top_groups;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (!stay) v[j] = -INFINITY;
        } else {                                      // lane g looks through group g's values
            double *sv = s_s[wave];                   // (the scores are put back below)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int j = 0; j < NV; ++j) sv[NV * lane + j] = v[j];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            double b0 = -INFINITY, b1 = -INFINITY;
            if (lane < a.groups)
                for (int i = 0; i < n; ++i) {
                    const double u = sv[lane * n + i];
                    b1 = fmax(fmin(b0, u), b1);
                    b0 = fmax(b0, u);
                }
            const double gs = a.group_best == 2 && b1 > -INFINITY ? b0 + b1 : b0;
            int rank = 0;
            for (int g = 0; g < a.groups; ++g) {
                const double o = lane_d(gs, g);
                rank += o > gs || (o == gs && g < lane);
            }
            const uint64_t keep = __ballot(lane < a.groups && rank < a.top_groups);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int e = NV * lane + j;
                if (!(keep >> (min(e, a.E - 1) / n) & 1)) v[j] = -INFINITY;
                sv[e] = s[j];
            }
        }
    }
    // each lane's values in order, equal ones in that of their ids
    uint64_t k[NV];
    int id[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        id[j] = NV * lane + j;
        k[j] = id[j] >= a.E ? 0 : v[j] > -INFINITY ? value_key(v[j]) : KEY_OFF;
    }
#pragma unroll
    for (int i = 1; i < NV; ++i)
#pragma unroll
        for (int j = i; j > 0; --j)
            if (k[j] > k[j - 1]) {
                const uint64_t t = k[j];
                k[j] = k[j - 1];
                k[j - 1] = t;
                const int u = id[j];
                id[j] = id[j - 1];
                id[j - 1] = u;
            }
    int my_id = 0;
    bool my_on = false;
    for (int r = 0; r < a.K; ++r) {
        const uint32_t hi = (uint32_t)(k[0] >> 32);
        const uint32_t M = wave_max_u32_bcast(hi);
        uint64_t who = __ballot(hi == M);
        if (who & (who - 1)) {                        // (uniform) two lanes or more agree in the upper word
            const uint32_t lo = hi == M ? (uint32_t)k[0] : 0;
            const uint32_t L = wave_max_u32_bcast(lo);
            who = __ballot(hi == M && lo == L);
        }
        const int win = __ffsll((unsigned long long)who) - 1;
        const int e = __builtin_amdgcn_readlane(id[0], win);
        if (lane == r) {
            my_id = e;
            my_on = M != 0;                           // a key above KEY_OFF has an upper word
        }
        const bool pop = lane == win;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            k[j] = pop ? (j + 1 < NV ? k[j + 1] : 0) : k[j];
            id[j] = pop && j + 1 < NV ? id[j + 1] : id[j];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    double w = lane < a.K && my_on ? s_s[wave][my_id] : 0.0;
    if (a.renorm) {
        const double sum = wave_sum_d(w);
        w = sum > 0.0 ? w / sum : 0.0;
    }
    if (lane < a.K) {
        const int64_t o = tok * a.K + lane;
        a.ids[o] = my_id;
        a.w[o] = (float)((double)a.scale * w);
        if (a.slots) a.slots[o] = a.table ? a.table[my_id] : a.dummy;
    }
}

template <int T, int NV>
static hipError_t launch_scored_n(ScoredArgs a, hipStream_t st) {
    a.vec = a.E % NV == 0;
    // a group of whole lanes is reduced by DPP, others one to a lane out of LDS (8 groups of 32: 15 us a call for 8,191 tokens; of 25: 17)
    const int n = a.E / a.groups, lanes = n / NV;
    a.group_lanes = n % NV == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    hipLaunchKernelGGL((route_scored_kernel<T, NV>), dim3((unsigned)((a.n_tok + SCORED_WAVES - 1) / SCORED_WAVES)),
                       dim3(64 * SCORED_WAVES), 0, st, a);
    return hipGetLastError();
}
template <int T>
static hipError_t launch_scored_t(const ScoredArgs &a, hipStream_t st) {
    return a.E <= 64 ? launch_scored_n<T, 1>(a, st) : a.E <= 128 ? launch_scored_n<T, 2>(a, st)
         : a.E <= 256 ? launch_scored_n<T, 4>(a, st) : a.E <= 512 ? launch_scored_n<T, 8>(a, st)
                      : launch_scored_n<T, 16>(a, st);
}

hipError_t launch_route_scored(const ScoredArgs &a, hipStream_t st) {
    return a.type == T_F32 ? launch_scored_t<T_F32>(a, st)
         : a.type == T_BF16 ? launch_scored_t<T_BF16>(a, st) : launch_scored_t<T_F16>(a, st);
}

}  // namespace mp
