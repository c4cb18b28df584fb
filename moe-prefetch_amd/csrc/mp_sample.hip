// mp_sample.hip -- the next token of a row of logits (moe_sample): temperature,
// top-k, top-p, min-p and the draw from a given uniform number.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

constexpr int SMP_THREADS = 1024, SMP_WAVES = SMP_THREADS / 64;
constexpr int SMP_BINS = 2048;

// f32 in the order of unsigned integers (-0 as +0)
__device__ inline uint32_t sort_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t KEY_NONE = 0x007fffffu;            // of -inf; NaN is read as -inf

struct SampleShared {
    uint32_t cnt[SMP_BINS];
    uint64_t mass[SMP_BINS];
    uint64_t wm[SMP_WAVES];
    uint32_t wc[SMP_WAVES];
    uint64_t found_m;
    uint32_t found_c, found_bin;
};

// A row's masses: e = exp((value - max) / temperature) as an integer of `shift` fractional bits
struct Mass {
    double vmax, inv_t;
    int shift;
    __device__ double e(uint32_t key) const {
        const double v = (double)key_value(key);
        if (vmax == INFINITY) return v == INFINITY ? 1.0 : 0.0;
        return exp((v - vmax) * inv_t);
    }
    __device__ uint64_t fixed(uint32_t key) const { return (uint64_t)(ldexp(e(key), shift) + 0.5); }
};

template <int T>
struct Row {
    const typename Elem<T>::raw *l;
    int V;
    template <class F>
    __device__ void each(F f) const {                 // f(key) of every token that is on
        for (int i = threadIdx.x; i < V; i += SMP_THREADS) {
            const uint32_t k = key(i);
            if (k > KEY_NONE) f(k);
        }
    }
    __device__ uint32_t key(int i) const {
        const float v = Elem<T>::load(l[i]);
        return v != v ? KEY_NONE : sort_key(v);
    }
};

__device__ inline uint64_t shfl_up_u64(uint64_t v, int o) {
    const uint32_t lo = __shfl_up((uint32_t)v, o, 64), hi = __shfl_up((uint32_t)(v >> 32), o, 64);
    return ((uint64_t)hi << 32) | lo;
}

__device__ inline uint64_t block_sum_u64(uint64_t v, SampleShared &s) {
    const int lane = threadIdx.x & 63;
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t lo = __shfl_xor((uint32_t)v, o, 64), hi = __shfl_xor((uint32_t)(v >> 32), o, 64);
        v += ((uint64_t)hi << 32) | lo;
    }
    __syncthreads();
    if (lane == 0) s.wm[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t t = 0;
    for (int w = 0; w < SMP_WAVES; ++w) t += s.wm[w];
    return t;
}

// The key at which the running count (by_mass 0) or mass (1) of the tokens in
// descending order first reaches target >= 1, and the count and mass before it:
// three levels of 11, 11 and 10 key bits.
struct Cut {
    uint32_t key, n_before;
    uint64_t m_before;
};
template <int T>
__device__ Cut locate(const Row<T> &row, const Mass &ms, bool by_mass, uint64_t target, SampleShared &s) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Cut c{0, 0, 0};
    for (int level = 0; level < 3; ++level) {
        const int sh = level == 0 ? 21 : level == 1 ? 10 : 0;
        const uint32_t mask = level == 2 ? 1023u : 2047u;
        const int up = level == 0 ? 31 : level == 1 ? 21 : 10;     // bits above: fixed by the levels before
        const uint32_t fixed_bits = c.key;
        __syncthreads();
        for (int i = tid; i < SMP_BINS; i += SMP_THREADS) { s.cnt[i] = 0; s.mass[i] = 0; }
        __syncthreads();
        row.each([&](uint32_t k) {
            if (level && (k >> up) != (fixed_bits >> up)) return;
            const uint32_t b = (k >> sh) & mask;
            atomicAdd(&s.cnt[b], 1u);
            atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)ms.fixed(k));
        });
        __syncthreads();
        // thread t: bins 2047 - 2t and the next lower; inclusive scan from the highest bin down
        const int b0 = SMP_BINS - 1 - 2 * tid;
        const uint32_t c0 = s.cnt[b0], c1 = s.cnt[b0 - 1];
        const uint64_t m0 = s.mass[b0], m1 = s.mass[b0 - 1];
        uint32_t cs = c0 + c1;
        uint64_t msum = m0 + m1;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t uc = __shfl_up(cs, o, 64);
            const uint64_t um = shfl_up_u64(msum, o);
            if (lane >= o) { cs += uc; msum += um; }
        }
        if (lane == 63) { s.wc[wave] = cs; s.wm[wave] = msum; }
        __syncthreads();
        uint32_t cb = c.n_before + cs - (c0 + c1);
        uint64_t mb = c.m_before + msum - (m0 + m1);
        for (int w = 0; w < wave; ++w) { cb += s.wc[w]; mb += s.wm[w]; }
        const uint64_t before = by_mass ? mb : cb, mid = before + (by_mass ? m0 : c0), end = mid + (by_mass ? m1 : c1);
        if (before < target && target <= end) {
            const bool first = target <= mid;
            s.found_bin = (uint32_t)(first ? b0 : b0 - 1);
            s.found_c = first ? cb : cb + c0;
            s.found_m = first ? mb : mb + m0;
        }
        __syncthreads();
        c.key = fixed_bits | (s.found_bin << sh);
        c.n_before = s.found_c;
        c.m_before = s.found_m;
    }
    return c;
}

// One workgroup per row.
template <int T>
__global__ __launch_bounds__(SMP_THREADS) void sample_kernel(SampleArgs a) {
    __shared__ SampleShared s;
    const int64_t tok = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Row<T> row{(const typename Elem<T>::raw *)a.logits + tok * a.ld, a.V};
    const float temp = a.temp ? a.temp[tok] : a.temp_all, u = a.u[tok];
    const float top_p = a.top_p ? a.top_p[tok] : a.top_p_all, min_p = a.min_p ? a.min_p[tok] : a.min_p_all;
    const int top_k = a.top_k ? a.top_k[tok] : a.top_k_all;
    uint32_t kmax = KEY_NONE;
    row.each([&](uint32_t k) { kmax = max(kmax, k); });
    for (int o = 32; o > 0; o >>= 1) kmax = max(kmax, (uint32_t)__shfl_xor(kmax, o, 64));
    if (lane == 0) s.wc[wave] = kmax;
    __syncthreads();
    for (int w = 0; w < SMP_WAVES; ++w) kmax = max(kmax, s.wc[w]);
    if (kmax == KEY_NONE) {                           // nothing is on
        if (tid == 0) {
            a.tokens[tok] = -1;
            if (a.probs) a.probs[tok] = 0.0f;
        }
        return;
    }
    uint32_t key = kmax;                              // of the token, and its place among the equal ones
    uint32_t place = 1;
    double prob = 1.0;
    if (temp > 0.0f) {
        const Mass ms{(double)key_value(kmax), 1.0 / (double)temp, 62 - (a.V > 1 ? 32 - __clz(a.V - 1) : 0)};
        uint64_t total;
        uint32_t cut_key = 0;
        bool all = true;                              // nothing was cut by count yet
        if (top_k > 0 && top_k < a.V) {
            uint64_t on = 0;
            row.each([&](uint32_t) { ++on; });
            on = block_sum_u64(on, s);
            if ((uint64_t)top_k < on) {
                const Cut c = locate(row, ms, false, (uint64_t)top_k, s);
                cut_key = c.key;
                total = c.m_before + ((uint32_t)top_k - c.n_before) * ms.fixed(c.key);
                all = false;
            }
        }
        if (all) {
            uint64_t sum = 0;
            row.each([&](uint32_t k) { sum += ms.fixed(k); });
            total = block_sum_u64(sum, s);
        }
        if (top_p < 1.0f) {
            const double want = ceil((double)fmaxf(top_p, 0.0f) * (double)total);
            const uint64_t m = want >= (double)total ? total : max((uint64_t)want, (uint64_t)1);
            const Cut c = locate(row, ms, true, m, s);
            const uint64_t f = ms.fixed(c.key);
            cut_key = c.key;
            total = c.m_before + (m - c.m_before + f - 1) / f * f;
        }
        if (min_p > 0.0f) {
            // the lowest key with e >= min_p, 64 ways a step
            uint32_t lo = KEY_NONE, hi = kmax;
            if ((double)min_p > 1.0) {
                total = ms.fixed(kmax);
            } else {
                while (hi - lo > 1) {
                    const uint32_t mid = lo + (uint32_t)(((uint64_t)(hi - lo) * (uint32_t)(lane + 1)) >> 6);
                    const uint64_t ge = __ballot(mid >= hi || (mid > lo && ms.e(mid) >= (double)min_p));
                    const int f = __ffsll((unsigned long long)ge) - 1;      // lane 63's mid is hi
                    const uint32_t nhi = __shfl(mid, f, 64);
                    const uint32_t nlo = f ? __shfl(mid, f - 1, 64) : lo;
                    lo = nlo;
                    hi = nhi;
                }
                if (hi > cut_key) {
                    uint64_t sum = 0;
                    row.each([&](uint32_t k) { if (k >= hi) sum += ms.fixed(k); });
                    total = block_sum_u64(sum, s);
                }
            }
        }
        const double at = u > 0.0f ? (double)u * (double)total : 0.0;
        const uint64_t t = at >= (double)total ? total - 1 : min((uint64_t)at, total - 1);
        const Cut c = locate(row, ms, true, t + 1, s);
        key = c.key;
        place = (uint32_t)((t - c.m_before) / ms.fixed(key)) + 1;
        prob = ldexp(ms.e(key), ms.shift) / (double)total;
    }
    // the place-th token of that key, by index: wave w holds a run of the row
    const int seg = (a.V + SMP_WAVES - 1) / SMP_WAVES;
    const int i0 = wave * seg, i1 = min(i0 + seg, a.V);
    uint32_t n = 0;
    for (int i = i0; i < i1; i += 64) n += (uint32_t)__popcll(__ballot(i + lane < i1 && row.key(min(i + lane, a.V - 1)) == key));
    __syncthreads();
    if (lane == 0) s.wc[wave] = n;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += s.wc[w];
    if (before >= place || before + n < place) return;
    for (int i = i0; i < i1; i += 64) {
        uint64_t m = __ballot(i + lane < i1 && row.key(min(i + lane, a.V - 1)) == key);
        const uint32_t c = (uint32_t)__popcll(m);
        if (before + c >= place) {
            for (uint32_t r = before + 1; r < place; ++r) m &= m - 1;
            if (lane == 0) {
                a.tokens[tok] = i + __ffsll((unsigned long long)m) - 1;
                if (a.probs) a.probs[tok] = (float)prob;
            }
            return;
        }
        before += c;
    }
}

hipError_t launch_sample(const SampleArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)a.n_tok), block(SMP_THREADS);
    if (a.type == T_F32) hipLaunchKernelGGL(sample_kernel<T_F32>, grid, block, 0, st, a);
    else if (a.type == T_BF16) hipLaunchKernelGGL(sample_kernel<T_BF16>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(sample_kernel<T_F16>, grid, block, 0, st, a);
    return hipGetLastError();
}

}  // namespace mp
