// mp_sample.hip -- the next token of a row of logits (moe_sample): temperature,
// top-k, top-p, min-p and the draw from a given uniform number.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

constexpr int SMP_THREADS = 1024, SMP_WAVES = SMP_THREADS / 64;
constexpr int SMP_BINS = 2048;
constexpr int SMP_LIST = 2048;                        // candidates that one row's workgroup sorts

// 2^(y / 64) for y <= 0 in 64 bits, within 2^-50: 64 powers from a table, e^x to x^5
// on |x| <= ln 2 / 128 (the next term is below 4e-17).  y below -64000 counts as that, and so does a NaN.
constexpr double EXP_MAGIC = 6755399441055744.0;      // 1.5 * 2^52: adding it rounds to a whole number
__device__ inline double exp64(double y, const double *tab) {
    constexpr double L = 0.6931471805599453094 / 64.0;
    y = fmax(y, -64000.0);
    const double n = y + EXP_MAGIC;
    const int i = (int)(uint32_t)__builtin_bit_cast(uint64_t, n);
    const double r = y - (n - EXP_MAGIC);
    double p = fma(r, L * L * L * L * L / 120.0, L * L * L * L / 24.0);
    p = fma(p, r, L * L * L / 6.0);
    p = fma(p, r, L * L / 2.0);
    p = fma(p, r, L);
    p = fma(p, r, 1.0);
    const uint64_t b = __builtin_bit_cast(uint64_t, tab[i & 63] * p);
    return __builtin_bit_cast(double, b + ((uint64_t)(int64_t)(i >> 6) << 52));
}
__device__ inline void exp64_table(double *tab) {     // by the first 64 threads
    if (threadIdx.x < 64) tab[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
}

// f32 in the order of unsigned integers (-0 as +0)
__device__ inline uint32_t sort_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t KEY_NONE = 0x007fffffu;            // of -inf; NaN is read as -inf

struct SampleCuts {
    float temp, top_p, min_p;
    int top_k;
    double u;                                         // in [0, 1)
};

struct SampleShared {
    uint32_t cnt[SMP_BINS];
    uint64_t mass[SMP_BINS];
    uint64_t wm[SMP_WAVES];
    uint32_t wc[SMP_WAVES];
    uint64_t found_m;
    uint32_t found_c, found_bin;
};

// A row's masses: e = exp((value - max) / temperature), as integers of `shift` fractional bits where
// sums of any order have to agree
struct Mass {
    double vmax, c;                                   // c = 64 / (temperature ln 2)
    const double *tab;
    int shift;
    __device__ double e(uint32_t key) const {
        const double v = (double)key_value(key);
        if (vmax == INFINITY) return v == INFINITY ? 1.0 : 0.0;
        return v == vmax ? 1.0 : exp64((v - vmax) * c, tab);
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

// The row's token from the whole row, in any case: what the candidates cannot decide.
template <int T>
__device__ void sample_row(const SampleArgs &a, int64_t tok, uint32_t kmax, const SampleCuts &cut, const Mass &ms,
                           SampleShared &s) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Row<T> row{(const typename Elem<T>::raw *)a.logits + tok * a.ld, a.V};
    uint64_t total;
    uint32_t cut_key = 0;
    bool all = true;                                  // nothing was cut by count yet
    if (cut.top_k > 0 && cut.top_k < a.V) {
        uint64_t on = 0;
        row.each([&](uint32_t) { ++on; });
        on = block_sum_u64(on, s);
        if ((uint64_t)cut.top_k < on) {
            const Cut c = locate(row, ms, false, (uint64_t)cut.top_k, s);
            cut_key = c.key;
            total = c.m_before + ((uint32_t)cut.top_k - c.n_before) * ms.fixed(c.key);
            all = false;
        }
    }
    if (all) {
        uint64_t sum = 0;
        row.each([&](uint32_t k) { sum += ms.fixed(k); });
        total = block_sum_u64(sum, s);
    }
    if (cut.top_p < 1.0f) {
        const double want = ceil((double)fmaxf(cut.top_p, 0.0f) * (double)total);
        const uint64_t m = want >= (double)total ? total : max((uint64_t)want, (uint64_t)1);
        const Cut c = locate(row, ms, true, m, s);
        const uint64_t f = ms.fixed(c.key);
        cut_key = c.key;
        total = c.m_before + (m - c.m_before + f - 1) / f * f;
    }
    if (cut.min_p > 0.0f) {
        // the lowest key with e >= min_p, 64 ways a step
        uint32_t lo = KEY_NONE, hi = kmax;
        if (cut.min_p > 1.0f) {
            total = ms.fixed(kmax);
        } else {
            while (hi - lo > 1) {
                const uint32_t mid = lo + (uint32_t)(((uint64_t)(hi - lo) * (uint32_t)(lane + 1)) >> 6);
                const uint64_t ge = __ballot(mid >= hi || (mid > lo && ms.e(mid) >= (double)cut.min_p));
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
    const uint64_t t = min((uint64_t)(cut.u * (double)total), total - 1);
    const Cut c = locate(row, ms, true, t + 1, s);
    const uint32_t key = c.key, place = (uint32_t)((t - c.m_before) / ms.fixed(key)) + 1;
    const double prob = ldexp(ms.e(key), ms.shift) / (double)total;
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

// ---------------------------------------------------------------------------
// Two launches.  The first reads the logits once, a workgroup per run of
// SLICE of a row: its maximum, its mass where the row's whole mass counts, and its
// candidates -- every logit from a bound on, which is the R-th largest of the
// threads' maxima, so that about SLICE_KEEP / S of them are kept whatever the
// values are.  The second, a workgroup per row, has the row's order complete down to
// the highest of the bounds, sorts that and cuts and draws; what needs more than
// these candidates is worked out from the whole row (sample_row).
constexpr int SLICE_THREADS = 256, SLICE_EPT = 64, SLICE = SLICE_THREADS * SLICE_EPT;
constexpr int SLICE_KEEP = 320;
static_assert(SMP_LIST >= 2 * SLICE_KEEP, "a row's candidates");

struct SliceHead {
    double mass;                                      // sum of exp((l - vmax) / temperature), 0 if not needed
    float vmax;                                       // of the logits that are on, -inf if none is
    uint32_t bound;                                   // every key of the slice from here on is in its list
    uint32_t n;                                       // candidates
    uint32_t at;                                      // greedy rows: the lowest index of vmax
};

__device__ inline SampleCuts load_cuts(const SampleArgs &a, int64_t tok) {
    SampleCuts c;
    c.temp = a.temp ? a.temp[tok] : a.temp_all;
    c.top_k = a.top_k ? a.top_k[tok] : a.top_k_all;
    c.top_p = a.top_p ? a.top_p[tok] : a.top_p_all;
    c.min_p = a.min_p ? a.min_p[tok] : a.min_p_all;
    const float u = a.u[tok];
    c.u = u > 0.0f ? (double)fminf(u, 0x1.fffffep-1f) : 0.0;
    return c;
}

template <int T>
__global__ __launch_bounds__(SLICE_THREADS) void sample_slice_kernel(SampleArgs a) {
    typedef typename Elem<T>::raw raw;
    constexpr int VEC = 16 / sizeof(raw), NV = SLICE_EPT / VEC;
    __shared__ __attribute__((aligned(16))) float s_max[SLICE_THREADS];
    __shared__ double s_sum[SLICE_THREADS / 64];
    __shared__ double s_tab[64];
    __shared__ uint32_t s_at[SLICE_THREADS / 64];
    __shared__ uint32_t s_n;
    __shared__ float s_bound;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t tok = blockIdx.x / a.slices;
    const int slice = blockIdx.x % a.slices, base = slice * SLICE;
    const SampleCuts cut = load_cuts(a, tok);
    const raw *l = (const raw *)a.logits + tok * a.ld + base;
    const int n_el = min(SLICE, a.V - base);
    exp64_table(s_tab);
    if (tid == 0) s_n = 0;
    float v[SLICE_EPT];
    if ((uintptr_t)l % 16 == 0) {
        uint4 q[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = (SLICE_THREADS * j + tid) * VEC;
            if (i + VEC <= n_el) {
                q[j] = *(const uint4 *)(l + i);
            } else {
                raw t[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) t[e] = i + e < n_el ? l[i + e] : Elem<T>::store(-INFINITY);
                __builtin_memcpy(&q[j], t, 16);
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            raw t[VEC];
            __builtin_memcpy(t, &q[j], 16);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[VEC * j + e] = Elem<T>::load(t[e]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < SLICE_EPT; ++j) {
            const int i = (SLICE_THREADS * (j / VEC) + tid) * VEC + j % VEC;
            v[j] = i < n_el ? Elem<T>::load(l[i]) : -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < SLICE_EPT; ++j) m = fmaxf(m, v[j]);       // passes over a NaN
    s_max[tid] = m;
    __syncthreads();
    float vmax = -INFINITY;
    {
        const float4 q = ((const float4 *)s_max)[lane];
        vmax = wave_max(fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)));
    }
    SliceHead h{};
    h.vmax = vmax;
    SliceHead *head = (SliceHead *)a.heads + blockIdx.x;
    if (!(cut.temp > 0.0f)) {
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int j = SLICE_EPT - 1; j >= 0; --j)
            if (v[j] == vmax) at = (uint32_t)((SLICE_THREADS * (j / VEC) + tid) * VEC + j % VEC);
        for (int o = 32; o > 0; o >>= 1) at = min(at, (uint32_t)__shfl_xor(at, o, 64));
        if (lane == 0) s_at[wave] = at;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < SLICE_THREADS / 64; ++w) h.at = w ? min(h.at, s_at[w]) : s_at[0];
            h.at += (uint32_t)base;
            *head = h;
        }
        return;
    }
    const bool by_k = cut.top_k > 0 && cut.top_k < a.V;
    if (!by_k) {                                      // the row's whole mass counts
        const double c = 64.0 / (0.6931471805599453094 * (double)cut.temp), vm = (double)vmax;
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < SLICE_EPT; ++j) sum += exp64(((double)v[j] - vm) * c, s_tab);
        for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);
        if (lane == 0) s_sum[wave] = sum;
    }
    // the R-th largest of the threads' maxima
    int rank = 0;
    for (int i = 0; i < SLICE_THREADS; i += 4) {
        const float4 q = *(const float4 *)&s_max[i];
        rank += (q.x > m) || (q.x == m && i < tid);
        rank += (q.y > m) || (q.y == m && i + 1 < tid);
        rank += (q.z > m) || (q.z == m && i + 2 < tid);
        rank += (q.w > m) || (q.w == m && i + 3 < tid);
    }
    if (rank == a.keep - 1) s_bound = m;
    __syncthreads();
    const float bound = s_bound;
    uint64_t *list = (uint64_t *)a.lists + (size_t)blockIdx.x * a.cap;
    if (m >= bound)
#pragma unroll
        for (int j = 0; j < SLICE_EPT; ++j)
            if (v[j] >= bound && v[j] > -INFINITY) {
                const uint32_t at = atomicAdd(&s_n, 1u);
                const uint32_t i = (uint32_t)(base + (SLICE_THREADS * (j / VEC) + tid) * VEC + j % VEC);
                if (at < (uint32_t)a.cap) list[at] = ((uint64_t)sort_key(v[j]) << 32) | (uint32_t)~i;
            }
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; !by_k && w < SLICE_THREADS / 64; ++w) h.mass += s_sum[w];
        h.n = min(s_n, (uint32_t)a.cap);
        h.bound = s_n > (uint32_t)a.cap ? 0xffffffffu : bound == -INFINITY ? 0u : sort_key(bound);
        *head = h;
    }
}

struct SampleList {
    uint64_t raw[SMP_LIST], sorted[SMP_LIST];         // key << 32 | ~index: descending order, the lower index first
    double wsum[SMP_WAVES];
    uint32_t n, cut, by_p, by_min, at;
    double total;
};
union SampleLds {
    SampleShared row;
    SampleList list;
};

template <int T>
__global__ __launch_bounds__(SMP_THREADS) void sample_pick_kernel(SampleArgs a) {
    __shared__ SampleLds s;
    __shared__ double s_tab[64];
    __shared__ SliceHead s_head[64];
    const int64_t tok = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const SampleCuts cut = load_cuts(a, tok);
    const SliceHead *heads = (const SliceHead *)a.heads + tok * a.slices;
    exp64_table(s_tab);
    if (tid < a.slices) s_head[tid] = heads[tid];
    if (tid == 0) s.list.n = 0;
    __syncthreads();
    float vmax = -INFINITY;
    uint32_t bound = 0;
    for (int i = 0; i < a.slices; ++i) {
        vmax = fmaxf(vmax, s_head[i].vmax);
        bound = max(bound, s_head[i].bound);
    }
    if (vmax == -INFINITY) {                          // nothing is on
        if (tid == 0) {
            a.tokens[tok] = -1;
            if (a.probs) a.probs[tok] = 0.0f;
        }
        return;
    }
    if (!(cut.temp > 0.0f)) {
        if (tid == 0) {
            int i = 0;
            while (s_head[i].vmax != vmax) ++i;
            a.tokens[tok] = (int32_t)s_head[i].at;
            if (a.probs) a.probs[tok] = 1.0f;
        }
        return;
    }
    const Mass ms{(double)vmax, 64.0 / (0.6931471805599453094 * (double)cut.temp), s_tab,
                  62 - (a.V > 1 ? 32 - __clz(a.V - 1) : 0)};
    const uint32_t kmax = sort_key(vmax);
    const bool by_k = cut.top_k > 0 && cut.top_k < a.V;
    for (int i = tid; i < a.slices * a.cap; i += SMP_THREADS) {
        const int sl = i / a.cap, j = i % a.cap;
        if (j >= (int)s_head[sl].n) continue;
        const uint64_t e = ((const uint64_t *)a.lists)[(size_t)(tok * a.slices) * a.cap + i];
        if ((uint32_t)(e >> 32) < bound) continue;
        const uint32_t at = atomicAdd(&s.list.n, 1u);
        if (at < SMP_LIST) s.list.raw[at] = e;
    }
    __syncthreads();
    const int n = (int)s.list.n;
    bool done = vmax < INFINITY && n > 0 && n <= SMP_LIST;
    __syncthreads();
    if (done) {
        // sorted by rank: the entries differ
        for (int i = tid; i < n; i += SMP_THREADS) {
            const uint64_t mine = s.list.raw[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += s.list.raw[j] > mine;
            s.list.sorted[rank] = mine;
        }
        if (tid == 0) {
            s.list.cut = s.list.by_p = s.list.by_min = s.list.at = 0xffffffffu;
            double total = 0.0;
            if (!by_k)
                for (int i = 0; i < a.slices; ++i)
                    if (s_head[i].vmax > -INFINITY)
                        total += s_head[i].mass * exp64(((double)s_head[i].vmax - ms.vmax) * ms.c, s_tab);
            s.list.total = total;
        }
        __syncthreads();
        // running masses: thread t has entries 2t and 2t + 1
        const int j0 = 2 * tid, j1 = j0 + 1;
        const double e0 = j0 < n ? ms.e((uint32_t)(s.list.sorted[j0] >> 32)) : 0.0;
        const double e1 = j1 < n ? ms.e((uint32_t)(s.list.sorted[j1] >> 32)) : 0.0;
        double run = e0 + e1;
        for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(run, o, 64);
            if (lane >= o) run += up;
        }
        if (lane == 63) s.list.wsum[wave] = run;
        __syncthreads();
        double before = 0.0;
        for (int w = 0; w < wave; ++w) before += s.list.wsum[w];
        const double c1 = before + run, c0 = c1 - e1;
        const bool whole = bound == 0;                // the candidates are all the row has
        uint32_t kept = (uint32_t)n;                  // how many of the sorted stay, if that is known
        bool open = !whole;                           // tokens behind the candidates may stay, too
        double total = s.list.total;
        if (by_k) {
            if (cut.top_k <= n) {
                kept = (uint32_t)cut.top_k;
                open = false;
            }
            done = !open;
            if (j0 == (int)kept - 1) s.list.total = c0;
            if (j1 == (int)kept - 1) s.list.total = c1;
            __syncthreads();
            total = s.list.total;
        } else if (whole) {
            if (j0 == n - 1) s.list.total = c0;
            if (j1 == n - 1) s.list.total = c1;
            __syncthreads();
            total = s.list.total;
        }
        if (cut.top_p < 1.0f) {
            const double want = (double)fmaxf(cut.top_p, 0.0f) * total;
            if (j0 < (int)kept && c0 >= want) atomicMin(&s.list.by_p, (uint32_t)j0);
            if (j1 < (int)kept && c1 >= want) atomicMin(&s.list.by_p, (uint32_t)j1);
            __syncthreads();
            const uint32_t f = s.list.by_p;
            if (f < kept) { kept = f + 1; open = false; }
        }
        if (cut.min_p > 0.0f) {
            if (j0 < (int)kept && !(e0 >= (double)cut.min_p)) atomicMin(&s.list.by_min, (uint32_t)j0);
            if (j1 < (int)kept && !(e1 >= (double)cut.min_p)) atomicMin(&s.list.by_min, (uint32_t)j1);
            __syncthreads();
            const uint32_t f = s.list.by_min;
            if (f < kept) { kept = max(f, 1u); open = false; }
        }
        if (done && !(open && (cut.top_p < 1.0f || cut.min_p > 0.0f))) {
            __syncthreads();
            if (!open) {
                if (j0 == (int)kept - 1) s.list.total = c0;
                if (j1 == (int)kept - 1) s.list.total = c1;
            }
            __syncthreads();
            total = s.list.total;
            const double t = cut.u * total;
            if (j0 < (int)kept && c0 > t) atomicMin(&s.list.at, (uint32_t)j0);
            if (j1 < (int)kept && c1 > t) atomicMin(&s.list.at, (uint32_t)j1);
            __syncthreads();
            const uint32_t at = s.list.at;
            done = at != 0xffffffffu;
            if (done && (j0 == (int)at || j1 == (int)at)) {
                a.tokens[tok] = (int32_t)~(uint32_t)s.list.sorted[at];
                if (a.probs) a.probs[tok] = (float)((j0 == (int)at ? e0 : e1) / total);
            }
        } else {
            done = false;
        }
    }
    if (done) return;
    __syncthreads();
    sample_row<T>(a, tok, kmax, cut, ms, s.row);
}

// slices of a row, candidates a slice keeps room for, and the rank of its bound
struct SamplePlan {
    int slices, cap, keep;
};
static SamplePlan sample_plan(int V) {
    SamplePlan p;
    p.slices = (V + SLICE - 1) / SLICE;
    // of SLICE_THREADS maxima over runs of random values, those above the value that x of them exceed on
    // average: 1 - exp(-x / threads)
    const double want = (double)SLICE_KEEP / p.slices;
    p.keep = (int)ceil(SLICE_THREADS * (1.0 - exp(-want / SLICE_THREADS)));
    p.keep = p.keep < 8 ? 8 : p.keep;
    p.cap = (2 * (int)want + 64 + 15) / 16 * 16;
    return p;
}

size_t sample_ws_bytes(int n_tok, int V) {
    const SamplePlan p = sample_plan(V);
    return (size_t)n_tok * p.slices * (sizeof(SliceHead) + 8 * (size_t)p.cap);
}

template <int T>
static hipError_t launch_sample_t(const SampleArgs &a, hipStream_t st) {
    hipLaunchKernelGGL(sample_slice_kernel<T>, dim3((unsigned)a.n_tok * (unsigned)a.slices), dim3(SLICE_THREADS), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(sample_pick_kernel<T>, dim3((unsigned)a.n_tok), dim3(SMP_THREADS), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_sample(SampleArgs a, void *ws, hipStream_t st) {
    const SamplePlan p = sample_plan(a.V);
    a.slices = p.slices;
    a.cap = p.cap;
    a.keep = p.keep;
    a.lists = ws;
    a.heads = (uint8_t *)ws + (size_t)a.n_tok * p.slices * 8 * p.cap;
    return a.type == T_F32 ? launch_sample_t<T_F32>(a, st)
         : a.type == T_BF16 ? launch_sample_t<T_BF16>(a, st) : launch_sample_t<T_F16>(a, st);
}

}  // namespace mp
