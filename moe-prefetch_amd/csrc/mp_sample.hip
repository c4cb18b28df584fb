// mp_sample.hip -- the next token of a row of logits (moe_sample): temperature,
// top-k, top-p, min-p and the draw from a given uniform number.
//
// With e_i = exp((l_i - max) / temperature) and the tokens in descending order (the
// lower index first), every cut keeps a front part of that order, and the draw takes
// the first token whose running mass exceeds u times the mass kept.  So what is
// needed is a front part of the order long enough to decide, and the whole row's
// mass where top-k does not bound it; the row itself is read once:
//   1 slice   one wave per 4,096 logits of a row, in registers: the maximum, the
//             candidates (every logit from a bound on) and, if the mass counts, its sum
//   2 pick    one workgroup per row: the order is complete down to the highest of
//             the slices' bounds; sorts that, cuts, draws
//   3 rest    rows that step 2 could not decide (a flat distribution: the cut or the
//             draw lies behind the candidates): a histogram of counts and masses by
//             several workgroups, the last of which reads the one bin that matters.
//             A bin of more than 2,048 tokens (many equal 16-bit logits, or a row nearly flat) ends in a radix search.
// 256 rows of 151,936 bf16 logits (78 MB, 12 us at the rate of a large read), each with cuts of its own: 36 us + 14 us,
// and about 30 more if a row or a few need step 3; under top-k alone 33 in all; one row 15.
// Step 3 is slow where many rows need it, one workgroup ending each: rows under a top-k of 1,000 take 44 us (one row), 79
// (16), 271 (64) and 1,100 (256) in all, under top-p of 0.9 over normal logits of deviation 1 68, 115, 400 and 1,570.  The
// radix search more so: under top-p of 0.9 over bf16 logits of mean 20 and deviation 1.5 0.82 ms (one row) and 12.3 (256),
// of one value only 0.94 and 15, and those under top-k and top-p both 2.5 and 39.
#include <hip/hip_runtime.h>

#include "mp_device.h"
#include "mp_elem.h"
#include "mp_internal.h"

namespace mp {

constexpr int SMP_THREADS = 512, SMP_WAVES = SMP_THREADS / 64;
constexpr int SMP_BINS = 2048;
constexpr int SMP_LIST = 2048;                        // tokens that a workgroup sorts
constexpr int SMP_PER = SMP_LIST / SMP_THREADS;       // of them, or of the bins, to a thread
static_assert(SMP_BINS == SMP_LIST, "bins and tokens to a thread");
constexpr int SLICE_WAVES = 4, SLICE_EPT = 64, SLICE = 64 * SLICE_EPT, SLICES_MAX = 256;
constexpr int REST_GRID = 256;

// 2^(j / 64), rounded to the nearest
__constant__ double EXP_TAB[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};

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

// f32 in the order of unsigned integers (-0 as +0)
__device__ inline uint32_t sort_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
constexpr uint32_t KEY_NONE = 0x007fffffu;            // of -inf
// An entry of the order: key and index as the mantissa of a number in [1, 2), so that the larger comes first (the
// lower index of equal keys) and a comparison is one of f64: four clocks where one of 64-bit integers takes
// sixteen.  0 is none.
static_assert(SLICES_MAX * SLICE == 1 << 20 && MAX_SAMPLE_V + 7 <= 1 << 20, "20 bits of index");
__device__ inline uint64_t entry_from(uint32_t key) { return (0x3ffull << 52) | ((uint64_t)key << 20); }    // the key's last
__device__ inline uint64_t entry(float v, uint32_t i) { return entry_from(sort_key(v)) | (i ^ 0xfffffu); }
__device__ inline uint32_t entry_key(uint64_t e) { return (uint32_t)(e >> 20); }
__device__ inline int32_t entry_token(uint64_t e) { return (int32_t)(~(uint32_t)e & 0xfffffu); }
__device__ inline bool gt(uint64_t a, uint64_t b) { return __builtin_bit_cast(double, a) > __builtin_bit_cast(double, b); }
__device__ inline bool ge(uint64_t a, uint64_t b) { return __builtin_bit_cast(double, a) >= __builtin_bit_cast(double, b); }

struct SampleCuts {
    float temp, top_p, min_p;
    int top_k;
    double u;                                         // in [0, 1)
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
__device__ inline double exp64_scale(float temp) { return 64.0 / (0.6931471805599453094 * (double)temp); }

// A row's masses, and as integers of `shift` fractional bits where sums of any order have to agree
struct Mass {
    double vmax, c;                                   // e = 2^((value - vmax) c / 64)
    const double *tab;
    int shift;
    __device__ double e(uint32_t key) const {
        const double v = (double)key_value(key);
        if (vmax == INFINITY) return v == INFINITY ? 1.0 : 0.0;
        return exp64((v - vmax) * c, tab);
    }
    __device__ uint64_t fixed(uint32_t key) const { return (uint64_t)(ldexp(e(key), shift) + 0.5); }
};
__device__ inline Mass row_mass(float vmax, float temp, const double *tab, int shift) {
    return {(double)vmax, exp64_scale(temp), tab, shift};
}

template <int CTRL, int ROWS, int BANKS, class N>
__device__ inline N scan_step(N v) {                  // v plus the lane's that CTRL names, where it is one
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, BANKS, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, BANKS, false);
    return v + __builtin_bit_cast(N, ((uint64_t)hi << 32) | lo);
}
// the sums of a wave's 64-bit values up to each lane, in a fixed order
template <class N>
__device__ inline N wave_scan(N v) {
    v = scan_step<0x111, 0xf, 0xf>(v);                // row_shr 1, 2, 4, 8, then the rows' last lanes
    v = scan_step<0x112, 0xf, 0xf>(v);
    v = scan_step<0x114, 0xf, 0xe>(v);
    v = scan_step<0x118, 0xf, 0xc>(v);
    v = scan_step<0x142, 0xa, 0xf>(v);
    return scan_step<0x143, 0xc, 0xf>(v);
}
// ---------------------------------------------------------------------------
// 1: slices

struct SliceHead {
    double mass;                                      // sum of exp((l - vmax) / temperature), 0 if not needed
    float vmax;                                       // of the logits that are on, -inf if none is
    uint32_t bound;                                   // every key of the slice from here on is in its list
    uint32_t n;                                       // candidates
    uint32_t at;                                      // greedy rows: the lowest index of vmax
};

// Chunks of 64 lanes x 16 bytes go to a row's slices in turn, so that neighbouring
// likely tokens spread over them.  The bound is the value that about `keep` lanes' maxima
// reach (a bisection; any value would do); should more than `cap` logits lie above it, a higher one.
// One slice to a wave, 64 logits in its lane's registers: 112 of them, four waves a SIMD, and no barrier behind the first.
// 256 rows of 151,936 bf16 logits: 27 us where every row is under top-k (2.9 TB/s), 48 where none is: the 39 million
// exponentials in f64 are some 19 vector operations each, 20 us of every SIMD's time, and a wave's loads come before
// its own.  (A second slice on its way, or 16-bit logits kept packed, spilled or cost a wave a SIMD, and were slower.)
template <int T>
__global__ __launch_bounds__(64 * SLICE_WAVES, 4) void sample_slice_kernel(SampleArgs a) {
    typedef typename Elem<T>::raw raw;
    constexpr int VEC = 16 / sizeof(raw), NV = SLICE_EPT / VEC;
    __shared__ double s_tab[64];
    const int lane = threadIdx.x & 63;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.n_rest = 0;
    const int64_t id = (int64_t)blockIdx.x * SLICE_WAVES + (threadIdx.x >> 6);
    const bool live = id < (int64_t)a.n_tok * a.slices;
    const int64_t tok = live ? id / a.slices : 0;
    const int slice = (int)(id - tok * a.slices);
    // counted from the 16 bytes that the row begins in: element i is token i - m
    const raw *l = (const raw *)a.logits + tok * a.ld;
    const int m0 = (int)((uintptr_t)l % 16 / sizeof(raw)), end = a.V + m0;
    l -= m0;
    float v[SLICE_EPT];
    const int i0 = (slice * 64 + lane) * VEC, step = a.slices * 64 * VEC;      // vector j at i0 + j step
    uint4 q[NV];
    const bool whole = live && (m0 == 0 || slice > 0) && (NV - 1) * step + (slice + 1) * 64 * VEC <= end;
    if (whole) {                                      // every vector of the slice lies in the row
#pragma unroll
        for (int j = 0; j < NV; ++j) q[j] = *(const uint4 *)(l + i0 + j * step);
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = i0 + j * step;
            if (live && i >= m0 && i + VEC <= end) {
                q[j] = *(const uint4 *)(l + i);
            } else {
                raw t[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    t[e] = live && i + e >= m0 && i + e < end ? l[i + e] : Elem<T>::store(-INFINITY);
                __builtin_memcpy(&q[j], t, 16);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        raw t[VEC];
        __builtin_memcpy(t, &q[j], 16);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[VEC * j + e] = Elem<T>::load(t[e]);
    }
    const SampleCuts cut = load_cuts(a, tok);
    if (threadIdx.x < 64) s_tab[threadIdx.x] = EXP_TAB[threadIdx.x];
    __syncthreads();
    if (!live) return;
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < SLICE_EPT; ++j) m = fmaxf(m, v[j]);       // passes over a NaN
    const float vmax = wave_max(m);
    SliceHead h{};
    h.vmax = vmax;
    const bool greedy = !(cut.temp > 0.0f);
    if (!greedy && !(cut.top_k > 0 && cut.top_k < a.V)) {         // the row's whole mass counts
        const double c = exp64_scale(cut.temp), vm = (double)vmax;
        double sum[2] = {};
#pragma unroll
        for (int j = 0; j < SLICE_EPT; ++j) sum[j & 1] += exp64(((double)v[j] - vm) * c, s_tab);
        double t = sum[0] + sum[1];
        for (int o = 1; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
        h.mass = t;
    }
    uint64_t *list = (uint64_t *)a.lists + (size_t)id * a.cap;
    const uint32_t mk = sort_key(m), top = (uint32_t)__builtin_amdgcn_readfirstlane((int)sort_key(vmax));
    const uint32_t low = ~wave_max_u32_bcast(~mk);    // the least of the lanes' maxima
    int keep = greedy ? 1 : a.keep;
    for (;;) {
        uint32_t lo = low, hi = top;                  // at least keep lanes reach lo
        if (keep > 64) {
            lo = KEY_NONE;                            // a row short enough to keep whole
        } else if (keep > 1) {
            for (int it = 0; it < 20 && hi > lo; ++it) {
                const uint32_t mid = hi - (hi - lo) / 2;
                const int c = __popcll(__ballot(mk >= mid));
                if (c >= keep) lo = mid;
                else hi = mid - 1;
                if (c == keep) break;
            }
        } else {
            lo = top;
        }
        // the lane's logits from the bound on, the last in bit 0 (all that are on above a bound of -inf)
        const float bound = lo > KEY_NONE ? key_value(lo) : -__FLT_MAX__;
        uint64_t in = 0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 32; ++j) w = 2 * w + (v[32 * half + j] >= bound);
            in = (in << 32) | w;
        }
        int n = __popcll(in);
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
        if (greedy) {
            const int j = __clzll((long long)in);
            uint32_t at = in ? (uint32_t)(i0 + (j / VEC) * step + j % VEC - m0) : 0xffffffffu;
            for (int o = 32; o > 0; o >>= 1) at = min(at, (uint32_t)__shfl_xor(at, o, 64));
            h.at = at;
            break;
        }
        h.n = (uint32_t)n;
        h.bound = lo > KEY_NONE ? lo : 0;
        if (n <= a.cap) {
            // few lanes have any: their values are read again, four at a time, rather than picked from 64
            // registers (an unrolled pick spills)
            uint32_t p = (uint32_t)(wave_scan((uint64_t)__popcll(in)) - __popcll(in));
            while (__ballot(in != 0)) {
                raw t[4];
                uint32_t at[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int j = in ? __clzll((long long)in) : 0;
                    at[u] = in ? (uint32_t)(i0 + (j / VEC) * step + j % VEC) : 0xffffffffu;
                    if (in) t[u] = l[at[u]];
                    in &= ~(0x8000000000000000ull >> j);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (at[u] != 0xffffffffu) list[p++] = entry(Elem<T>::load(t[u]), at[u] - (uint32_t)m0);
            }
            break;
        }
        if (keep <= 1) {                              // more equal maxima than cap
            h.n = 0;
            h.bound = 0xffffffffu;
            break;
        }
        keep = keep / 2;
    }
    if (lane == 0) ((SliceHead *)a.heads)[id] = h;
}

// ---------------------------------------------------------------------------
// the order of up to SMP_LIST entries, and running sums over it

struct SampleList {
    __attribute__((aligned(16))) uint64_t raw[SMP_LIST], sorted[SMP_LIST];
    uint32_t n, hits;
};
// sorted[0 .. n) = raw[0 .. n) in descending order (the entries differ).  Up to 1,024 entries by each one's rank, four
// lanes counting for four entries (348 of them: 2 us against 9 of the network, whose every step waits for LDS); more by a
// bitonic network, whose strides of 64 and below stay within a wave's 128 entries and need no barrier.
__device__ inline void sort_list(SampleList &s, int n) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (n <= 1024) {
        for (int i = n + tid; i < (n + 31) / 32 * 32; i += SMP_THREADS) s.raw[i] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < n; i0 += SMP_THREADS) {
            uint64_t mine[4];
            int rank[4] = {};
#pragma unroll
            for (int e = 0; e < 4; ++e) mine[e] = s.raw[min(i0 + (tid >> 2) + e * (SMP_THREADS / 4), n - 1)];
            for (int j = 2 * (tid & 3); j < n; j += 32) {
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    const ulonglong2 q = *(const ulonglong2 *)&s.raw[j + k];
#pragma unroll
                    for (int e = 0; e < 4; ++e) rank[e] += gt(q.x, mine[e]) + gt(q.y, mine[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                rank[e] += dpp_i<DPP_XOR1>(rank[e]);
                rank[e] += dpp_i<DPP_XOR2>(rank[e]);
                if ((tid & 3) == e && i0 + (tid >> 2) + e * (SMP_THREADS / 4) < n) s.sorted[rank[e]] = mine[e];
            }
        }
        __syncthreads();
        return;
    }
    constexpr int m = SMP_LIST;
    for (int i = tid; i < m; i += SMP_THREADS) s.sorted[i] = i < n ? s.raw[i] : 0;
    __syncthreads();
    for (int k = 2; k <= m; k <<= 1)
        for (int d = k / 2; d > 0; d >>= 1) {
            for (int p = tid; p < m / 2; p += SMP_THREADS) {
                const int i = 2 * p - (p & (d - 1));  // pairs (i, i + d)
                const uint64_t x = s.sorted[i], y = s.sorted[i + d];
                if (gt(y, x) == ((i & k) == 0)) {
                    s.sorted[i] = y;
                    s.sorted[i + d] = x;
                }
            }
            if (d >= 128 || (d == 1 && k >= 128)) __syncthreads();
            else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    __syncthreads();
}

// the sum of v over the threads before this one
__device__ inline uint64_t block_before(uint64_t v, uint64_t *s_w) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t run = wave_scan(v);
    __syncthreads();
    if (lane == 63) s_w[wave] = run;
    __syncthreads();
    uint64_t before = run - v;
    for (int w = 0; w < wave; ++w) before += s_w[w];
    return before;
}

// ---------------------------------------------------------------------------
// 3: whole rows

struct SampleShared {
    uint32_t cnt[SMP_BINS];
    uint64_t mass[SMP_BINS];
    uint64_t wm[SMP_WAVES];
    uint64_t wc[SMP_WAVES];
    uint64_t found_m, found_e;
    uint32_t found_c, found_bin, last, key[2];
    SampleList list;
};

template <int T>
struct Row {
    typedef typename Elem<T>::raw raw;
    const raw *l;
    int V;
    __device__ float at(int i) const { return Elem<T>::load(l[i]); }
    // (What follows runs once per row on one CU: its time is that of fetching its instructions as much as of running
    // them, so the ends of a row go through a short loop of their own instead of tests beside every vector.)
    // f(value, index) of every token that is on, of [i0, i1); f a vector's elements times in the code, or once
    template <bool UNROLL, class F>
    __device__ inline void each(int i0, int i1, F f) const {
        constexpr int VEC = 16 / sizeof(raw);
        int head, tail;
        vectors(i0, i1, head, tail);
        int i = head + (int)threadIdx.x * VEC;
        uint4 next = {};
        if (i < tail) next = *(const uint4 *)(l + i);
#pragma unroll 1
        for (; i < tail; i += SMP_THREADS * VEC) {
            uint4 q = next;                           // the next vector is on its way meanwhile
            if (i + SMP_THREADS * VEC < tail) next = *(const uint4 *)(l + i + SMP_THREADS * VEC);
            if constexpr (UNROLL) {
                raw t[VEC];
                __builtin_memcpy(t, &q, 16);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float v = Elem<T>::load(t[e]);
                    if (v > -INFINITY) f(v, i + e);
                }
            } else {
#pragma unroll 1
                for (int e = 0; e < VEC; ++e) {
                    const float v = T == T_F32 ? __uint_as_float(q.x) : Elem<T>::load((raw)q.x);
                    constexpr int B = 8 * sizeof(raw) % 32;       // the vector moves down by one element
                    q.x = B ? __builtin_amdgcn_alignbit(q.y, q.x, B) : q.y;
                    q.y = B ? __builtin_amdgcn_alignbit(q.z, q.y, B) : q.z;
                    q.z = B ? __builtin_amdgcn_alignbit(q.w, q.z, B) : q.w;
                    q.w = q.w >> B;
                    if (v > -INFINITY) f(v, i + e);
                }
            }
        }
#pragma unroll 1
        for (int k = threadIdx.x; k < head - i0 + i1 - tail; k += SMP_THREADS) {
            const int j = k < head - i0 ? i0 + k : tail + k - (head - i0);
            const float v = at(j);
            if (v > -INFINITY) f(v, j);
        }
    }
    // [head, tail): the part of [i0, i1) in whole vectors on 16 bytes
    __device__ inline void vectors(int i0, int i1, int &head, int &tail) const {
        constexpr int VEC = 16 / sizeof(raw);
        const int m = (int)((uintptr_t)(l + i0) % 16 / sizeof(raw));
        head = min(i1, i0 + (m ? VEC - m : 0));
        tail = head + (i1 - head) / VEC * VEC;
    }
    template <class F>
    __device__ inline void each(F f) const { each<false>(0, V, f); }
    // The tokens of [from, to], at most SMP_LIST of them, into list.raw.  Values of one sign lie between two bit patterns, so
    // a token takes a subtraction and a minimum, two 16-bit ones at once; the vectors that hold one are listed first
    // and read again all at the same time.
    __device__ inline void among(float from, float to, SampleList &list) const {
        constexpr int VEC = 16 / sizeof(raw), NV = 16, STEP = SMP_THREADS * VEC;
        auto take = [&](float v, int i) {
            if (v >= from && v <= to) list.raw[atomicAdd(&list.n, 1u)] = entry(v, (uint32_t)i);
        };
        uint32_t *hit = (uint32_t *)list.sorted;
        if (threadIdx.x == 0) list.n = list.hits = 0;
        __syncthreads();
        const bool same = (__float_as_uint(from) ^ __float_as_uint(to)) >> 31 == 0;
        if (!same) {
            each(take);
            return;
        }
        // the type's own values next to the ends, inside: a vector listed holds a token of the bin, so that the list,
        // the bin's 2,048 at most, has room for the vectors
        const bool neg = __float_as_uint(from) >> 31;
        auto a = bits_of(from), b = bits_of(to);
        if (Elem<T>::load(raw_of(a)) < from) a += neg ? -1 : 1;
        if (Elem<T>::load(raw_of(b)) > to) b += neg ? 1 : -1;
        const uint32_t x = neg ? b : a, y = neg ? a : b;              // x <= y as unsigned
        int head, tail;
        vectors(0, V, head, tail);
        for (int base = head; base < tail; base += NV * STEP) {
            const int i0 = base + (int)threadIdx.x * VEC;
            uint4 q[NV];
#pragma unroll
            for (int k = 0; k < NV; ++k) q[k] = *(const uint4 *)(l + min(i0 + k * STEP, tail - VEC));
            uint32_t in = 0;
#pragma unroll
            for (int k = 0; k < NV; ++k) in = 2 * in + (near(q[k], x, y - x) && i0 + k * STEP < tail);
            for (; in; in &= in - 1) hit[atomicAdd(&list.hits, 1u)] = (uint32_t)(i0 + (NV - __ffs(in)) * STEP);
        }
        __syncthreads();
        for (int j = threadIdx.x; j < (int)list.hits; j += SMP_THREADS) {
            const int i = (int)hit[j];
            const uint4 q = *(const uint4 *)(l + i);
            raw t[VEC];
            __builtin_memcpy(t, &q, 16);
#pragma unroll
            for (int e = 0; e < VEC; ++e) take(Elem<T>::load(t[e]), i + e);
        }
        for (int k = threadIdx.x; k < head + V - tail; k += SMP_THREADS) {
            const int j = k < head ? k : tail + k - head;
            take(at(j), j);
        }
    }

private:
    static __device__ inline auto bits_of(float v) {
        if constexpr (T == T_F32) return __float_as_uint(v);
        else return (uint32_t)Elem<T>::store(v);
    }
    static __device__ inline raw raw_of(uint32_t b) {
        if constexpr (T == T_F32) return __uint_as_float(b);
        else return (raw)b;
    }
    // whether one of the vector's elements e has e - x <= d as unsigned
    static __device__ inline bool near(uint4 q, uint32_t x, uint32_t d) {
        if constexpr (T == T_F32) {
            return min(min(q.x - x, q.y - x), min(q.z - x, q.w - x)) <= d;
        } else {
            typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
            const u16x2 xx = {(uint16_t)x, (uint16_t)x};
            auto sub = [&](uint32_t v) { return __builtin_bit_cast(u16x2, v) - xx; };
            const u16x2 m = __builtin_elementwise_min(__builtin_elementwise_min(sub(q.x), sub(q.y)),
                                                      __builtin_elementwise_min(sub(q.z), sub(q.w)));
            return min((uint32_t)m.x, (uint32_t)m.y) <= d;
        }
    }
};

__device__ inline uint64_t block_sum(uint64_t v, SampleShared &s) {
    const uint64_t run = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) s.wm[threadIdx.x >> 6] = run;
    __syncthreads();
    uint64_t t = 0;
    for (int w = 0; w < SMP_WAVES; ++w) t += s.wm[w];
    return t;
}

// Where the running count or mass of the order first reaches a target >= 1: the
// key there, the count and mass before it (before its first equal), and the token, or -1 if it is
// yet to be looked up among the equal ones.
constexpr int32_t CUT_FULL = -2;                      // as token: more entries in the bin than can be sorted
struct Cut {
    uint32_t key;
    int32_t token;
    uint64_t n_before, m_before;
};

// by a radix search: three levels of 11, 11 and 10 key bits, whatever the values are
template <int T>
struct RadixSearch {
    Row<T> row;
    Mass ms;
    SampleShared &s;
    __device__ void totals(uint64_t &n, uint64_t &m) const {
        uint64_t c = 0, sum = 0;
        row.each([&](float v, int) { ++c; sum += ms.fixed(sort_key(v)); });
        n = block_sum(c, s);
        m = block_sum(sum, s);
    }
    __device__ uint64_t mass_from(uint32_t key) const {
        uint64_t sum = 0;
        row.each([&](float v, int) { const uint32_t k = sort_key(v); if (k >= key) sum += ms.fixed(k); });
        return block_sum(sum, s);
    }
    __device__ Cut find(bool by_mass, uint64_t target) const {
        const int tid = threadIdx.x;
        Cut c{0, -1, 0, 0};
        for (int level = 0; level < 3; ++level) {
            const int sh = level == 0 ? 21 : level == 1 ? 10 : 0;
            const uint32_t mask = level == 2 ? 1023u : 2047u;
            const int up = level == 1 ? 21 : 10;      // bits above: fixed by the levels before
            const uint32_t fixed_bits = c.key;
            __syncthreads();
            for (int i = tid; i < SMP_BINS; i += SMP_THREADS) { s.cnt[i] = 0; s.mass[i] = 0; }
            __syncthreads();
            row.each([&](float v, int) {
                const uint32_t k = sort_key(v);
                if (level && (k >> up) != (fixed_bits >> up)) return;
                const uint32_t b = mask - ((k >> sh) & mask);      // bin 0: the largest
                atomicAdd(&s.cnt[b], 1u);
                atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)ms.fixed(k));
            });
            __syncthreads();
            find_bin(s, by_mass, target, c.n_before, c.m_before);
            c.key = fixed_bits | ((mask - s.found_bin) << sh);
            c.n_before = s.found_c;
            c.m_before = s.found_m;
        }
        return c;
    }
    // the bin that holds the target, and the count and mass before it
    static __device__ void find_bin(SampleShared &s, bool by_mass, uint64_t target, uint64_t n0, uint64_t m0) {
        const int b = SMP_PER * (int)threadIdx.x;
        uint64_t c = 0, m = 0;
        for (int j = 0; j < SMP_PER; ++j) { c += s.cnt[b + j]; m += s.mass[b + j]; }
        c = n0 + block_before(c, s.wc);
        m = m0 + block_before(m, s.wm);
        for (int j = 0; j < SMP_PER; ++j) {
            const uint64_t before = by_mass ? m : c, end = before + (by_mass ? s.mass[b + j] : s.cnt[b + j]);
            if (before < target && target <= end) {
                s.found_bin = (uint32_t)(b + j);
                s.found_c = (uint32_t)c;
                s.found_m = m;
            }
            c += s.cnt[b + j];
            m += s.mass[b + j];
        }
        __syncthreads();
    }
};

// by a histogram of the row over bins of equal width below the maximum (s.cnt, s.mass), and the sorted
// entries of the one bin that holds the target
__device__ inline int bin_of(float v, float vmax, float per) { return (int)fminf((vmax - v) * per, (float)(SMP_BINS - 1)); }
// bins of 1/64 of a factor of two: 2,048 span 32 of them, and of 152k logits spread like a normal
// distribution's with a deviation of 1 the fullest holds about 660
__device__ inline float bins_per(float temp) { return (float)fmin(64.0 / (0.6931471805599453094 * (double)temp), 1e30); }

// The lowest key above lo with pred, which holds from some key up to hi on: 64 ways a step.
template <class F>
__device__ inline uint32_t lowest_key(uint32_t lo, uint32_t hi, F pred) {
    const int lane = threadIdx.x & 63;
    while (hi - lo > 1) {
        const uint32_t mid = lo + (uint32_t)(((uint64_t)(hi - lo) * (uint32_t)(lane + 1)) >> 6);
        const uint64_t b = __ballot(mid >= hi || (mid > lo && pred(mid)));
        const int f = __ffsll((unsigned long long)b) - 1;         // lane 63's mid is hi
        const uint32_t nhi = (uint32_t)__builtin_amdgcn_readlane((int)mid, f);
        if (f) lo = (uint32_t)__builtin_amdgcn_readlane((int)mid, f - 1);
        hi = nhi;
    }
    return hi;
}

// What the slices of a row left: every token of a key from `bound` on
struct Candidates {
    const SliceHead *heads;
    const uint64_t *lists;
    int slices, cap_log;
    uint32_t bound;
    template <class F>
    __device__ void among(float from, float to, F f) const {
        for (int p = threadIdx.x; p < slices << cap_log; p += SMP_THREADS) {
            const uint64_t e = lists[p];              // (what lies behind a list's end is read and left out)
            const float v = key_value(entry_key(e));
            if (((uint32_t)p & ((1u << cap_log) - 1)) < heads[p >> cap_log].n && v >= from && v <= to) f(e);
        }
    }
};

template <int T>
struct BinSearch {
    Row<T> row;
    Mass ms;
    SampleShared &s;
    float vmax, per;
    Candidates cand;
    uint64_t n_all, m_all;
    // the histogram's counts and masses of all parts to s.cnt and s.mass, as those of the bins before each
    __device__ void prepare(const uint32_t *cnt, const uint64_t *mass) {
        const int b = SMP_PER * (int)threadIdx.x;
        uint64_t q[SMP_PER], m = 0;
        uint32_t k[SMP_PER], c = 0;
#pragma unroll
        for (int j = 0; j < SMP_PER; ++j) {
            k[j] = __hip_atomic_load(&cnt[b + j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            q[j] = __hip_atomic_load(&mass[b + j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (int j = 0; j < SMP_PER; ++j) {
            c += k[j];
            m += q[j];
        }
        uint64_t cb = block_before(c, s.wc), mb = block_before(m, s.wm);
        n_all = m_all = 0;
        for (int w = 0; w < SMP_WAVES; ++w) {
            n_all += s.wc[w];
            m_all += s.wm[w];
        }
#pragma unroll
        for (int j = 0; j < SMP_PER; ++j) {
            s.cnt[b + j] = (uint32_t)cb;
            s.mass[b + j] = mb;
            cb += k[j];
            mb += q[j];
        }
        __syncthreads();
    }
    __device__ uint64_t cnt_to(int b) const { return b < SMP_BINS ? s.cnt[b] : n_all; }
    __device__ uint64_t mass_to(int b) const { return b < SMP_BINS ? s.mass[b] : m_all; }
    __device__ void totals(uint64_t &n, uint64_t &m) const { n = n_all; m = m_all; }
    __device__ uint64_t mass_from(uint32_t key) const {
        const int b = bin_of(key_value(key), vmax, per);
        uint64_t sum = 0;
        const float from = key_value(key), to = b == 0 ? vmax + 0.0f : key_value(lowest_in(b - 1) - 1);
        if (key >= cand.bound) cand.among(from, to, [&](uint64_t e) { sum += ms.fixed(entry_key(e)); });
        else row.each([&](float v, int) { if (v >= from && v <= to) sum += ms.fixed(sort_key(v)); });
        return mass_to(b) + block_sum(sum, s);
    }
    // the lowest key of bins 0 to b
    __device__ uint32_t lowest_in(int b) const {
        return lowest_key(KEY_NONE, sort_key(vmax), [&](uint32_t k) { return bin_of(key_value(k), vmax, per) <= b; });
    }
    __device__ Cut find(bool by_mass, uint64_t target) const {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SMP_PER; ++j) {
            const int b = SMP_PER * (int)threadIdx.x + j;
            const uint64_t before = by_mass ? mass_to(b) : cnt_to(b), end = by_mass ? mass_to(b + 1) : cnt_to(b + 1);
            if (before < target && target <= end) s.found_bin = (uint32_t)b;
        }
        __syncthreads();
        const int b = (int)s.found_bin, n = (int)(cnt_to(b + 1) - cnt_to(b));
        uint64_t nb = cnt_to(b), mb = mass_to(b);
        if (n > SMP_LIST) return Cut{0, CUT_FULL, 0, 0};
        // the bin's values, so that the pass over the row only compares; a wave to each end
        const int wave = (int)threadIdx.x >> 6;
        if (wave < 2 && wave <= b) {
            const uint32_t k = lowest_in(b - wave);
            if ((threadIdx.x & 63) == 0) s.key[wave] = k;
        }
        __syncthreads();
        const float from = key_value(s.key[0]), to = b == 0 ? vmax + 0.0f : key_value(s.key[1] - 1);
        if (s.key[0] >= cand.bound) {                 // every token of the bin is among the candidates
            if (threadIdx.x == 0) s.list.n = 0;
            __syncthreads();
            cand.among(from, to, [&](uint64_t e) { s.list.raw[atomicAdd(&s.list.n, 1u)] = e; });
        } else {
            row.among(from, to, s.list);
        }
        sort_list(s.list, n);
        const int j0 = SMP_PER * (int)threadIdx.x;
        uint64_t q[SMP_PER], m = 0;
        for (int j = 0; j < SMP_PER; ++j) m += q[j] = j0 + j < n ? ms.fixed(entry_key(s.list.sorted[j0 + j])) : 0;
        mb += block_before(m, s.wm);
        nb += (uint64_t)j0;
        for (int j = 0; j < SMP_PER && j0 + j < n; ++j) {
            const uint64_t before = by_mass ? mb : nb;
            if (before < target && target <= before + (by_mass ? q[j] : 1)) {
                s.found_e = s.list.sorted[j0 + j];
                s.found_c = (uint32_t)nb;
                s.found_m = mb;
            }
            mb += q[j];
            ++nb;
        }
        __syncthreads();
        return Cut{entry_key(s.found_e), entry_token(s.found_e), s.found_c, s.found_m};
    }
};

// The row's token by a search over the whole row.  A cut's n_before and m_before may stand before the first of the
// equal keys (a radix search) or right before the token itself: (target - before) counts on from there either way.
template <int T, class Search>
__device__ inline bool sample_row(const SampleArgs &a, int64_t tok, uint32_t kmax, const SampleCuts &cut, const Search search,
                                  SampleShared &s) {
    const Row<T> row = search.row;
    const Mass ms = search.ms;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t on, total, t = 0;
    search.totals(on, total);
    uint32_t cut_key = 0;
    Cut c{};
    for (int step = 0; step < 3; ++step) {            // top-k, top-p, the draw
        uint64_t target;
        if (step == 0) {
            if (!(cut.top_k > 0 && cut.top_k < a.V && (uint64_t)cut.top_k < on)) continue;
            target = (uint64_t)cut.top_k;
        } else if (step == 1) {
            if (!(cut.top_p < 1.0f)) continue;
            const double want = ceil((double)fmaxf(cut.top_p, 0.0f) * (double)total);
            target = want >= (double)total ? total : max((uint64_t)want, (uint64_t)1);
        } else {
            if (cut.min_p > 1.0f) {
                total = ms.fixed(kmax);
            } else if (cut.min_p > 0.0f) {
                const uint32_t hi = lowest_key(KEY_NONE, kmax, [&](uint32_t k) { return ms.e(k) >= (double)cut.min_p; });
                if (hi > cut_key) total = search.mass_from(hi);
            }
            t = min((uint64_t)(cut.u * (double)total), total - 1);
            target = t + 1;
        }
        c = search.find(step > 0, target);
        if (c.token == CUT_FULL) return false;
        const uint64_t f = ms.fixed(c.key);
        if (step < 2) {
            cut_key = c.key;
            total = c.m_before + (step == 0 ? (target - c.n_before) * f : (target - c.m_before + f - 1) / f * f);
        }
    }
    const float prob = (float)(ldexp(ms.e(c.key), ms.shift) / (double)total);
    if (c.token >= 0) {
        if (threadIdx.x == 0) {
            a.tokens[tok] = c.token;
            if (a.probs) a.probs[tok] = prob;
        }
        return true;
    }
    // the place-th token of that key, by index: wave w holds a run of the row
    const uint32_t place = (uint32_t)((t - c.m_before) / ms.fixed(c.key)) + 1;
    const float value = key_value(c.key);
    const int seg = (a.V + SMP_WAVES - 1) / SMP_WAVES;
    const int i0 = wave * seg, i1 = min(i0 + seg, a.V);
    uint32_t n = 0;
    for (int i = i0; i < i1; i += 64) n += (uint32_t)__popcll(__ballot(i + lane < i1 && row.at(min(i + lane, a.V - 1)) == value));
    __syncthreads();
    if (lane == 0) s.wc[wave] = n;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += (uint32_t)s.wc[w];
    if (before >= place || before + n < place) return true;
    for (int i = i0; i < i1; i += 64) {
        uint64_t m = __ballot(i + lane < i1 && row.at(min(i + lane, a.V - 1)) == value);
        const uint32_t k = (uint32_t)__popcll(m);
        if (before + k >= place) {
            for (uint32_t r = before + 1; r < place; ++r) m &= m - 1;
            if (lane == 0) {
                a.tokens[tok] = i + __ffsll((unsigned long long)m) - 1;
                if (a.probs) a.probs[tok] = prob;
            }
            return true;
        }
        before += k;
    }
    return true;
}

// what step 2 hands to step 3
struct RestRow {
    uint64_t mass[SMP_BINS];
    uint32_t cnt[SMP_BINS];
    int64_t tok;
    float vmax;
    int shift;                                        // Mass::shift
    uint32_t bound;                                   // Candidates::bound
    uint32_t parts;                                   // finished
};

// A fixed number of workgroups take the parts of the undecided rows in turn; the one
// that finishes a row's last part decides the row.  No workgroup waits for another.
// One row of 151,936 takes 30 us where its bins are small (top-k 1,000 over a peaked row) to 52 (top-p over a broad one), all
// latency: the histogram 4.5 (16 parts), its sums to memory 3 and back 3, and a bin's tokens found, gathered and
// sorted in 11 and more, for the cut and for the draw; 6 less where the candidates hold all of the bin, as they do for
// most draws.  16 rows take twice that, 64 rows 256 us.  (Reading the bins of both in one
// pass over the row gained 1 us of 54 and was not kept.)
template <int T>
__global__ __launch_bounds__(SMP_THREADS) void sample_rest_kernel(SampleArgs a) {
    __shared__ SampleShared s;
    __shared__ double s_tab[64];
    const int tid = threadIdx.x;
    const uint32_t n = *a.n_rest, parts = (uint32_t)a.parts;
    if (blockIdx.x >= n * parts) return;
    if (tid < 64) s_tab[tid] = EXP_TAB[tid];
    for (uint32_t task = blockIdx.x; task < n * parts; task += gridDim.x) {
        RestRow &r = ((RestRow *)a.rest)[task / parts];
        const int part = (int)(task % parts);
        const int64_t tok = r.tok;
        const float vmax = r.vmax;
        const SampleCuts cut = load_cuts(a, tok);
        const Row<T> row{(const typename Elem<T>::raw *)a.logits + tok * a.ld, a.V};
        const Mass ms = row_mass(vmax, cut.temp, s_tab, r.shift);
        const float per = bins_per(cut.temp);
        const int run = ((a.V + a.parts - 1) / a.parts + 7) / 8 * 8;
        __syncthreads();
        for (int i = tid; i < SMP_BINS; i += SMP_THREADS) { s.cnt[i] = 0; s.mass[i] = 0; }
        __syncthreads();
        if (vmax < INFINITY)
            row.template each<true>(min(part * run, a.V), min((part + 1) * run, a.V), [&](float v, int) {
                const int b = bin_of(v, vmax, per);
                atomicAdd(&s.cnt[b], 1u);
                atomicAdd((unsigned long long *)&s.mass[b], (unsigned long long)ms.fixed(sort_key(v)));
            });
        __syncthreads();
        for (int i = tid; i < SMP_BINS; i += SMP_THREADS)
            if (s.cnt[i]) {
                __hip_atomic_fetch_add(&r.cnt[i], s.cnt[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_fetch_add(&r.mass[i], s.mass[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        __threadfence();
        __syncthreads();
        if (tid == 0)
            s.last = __hip_atomic_fetch_add(&r.parts, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
        __syncthreads();
        if (!s.last) continue;
        __threadfence();
        const uint32_t kmax = sort_key(vmax);
        const Candidates cand = {(const SliceHead *)a.heads + tok * a.slices, (const uint64_t *)a.lists + (size_t)(tok * a.slices) * a.cap,
                                 a.slices, a.cap_log, r.bound};
        BinSearch<T> bins{row, ms, s, vmax, per, cand, 0, 0};
        bins.prepare(r.cnt, r.mass);
        if (vmax == INFINITY || !sample_row<T>(a, tok, kmax, cut, bins, s))
            sample_row<T>(a, tok, kmax, cut, RadixSearch<T>{row, ms, s}, s);
    }
}

// ---------------------------------------------------------------------------
// 2: one workgroup per row

constexpr int PICK_WAVES = 4, PICK_THREADS = 64 * PICK_WAVES;
// PER: candidates a lane holds
template <int PER>
struct PickLds {
    static constexpr int MAX = 64 * PER;
    uint64_t list[SMP_LIST];                          // candidates, in no order
    uint64_t order[MAX];                              // the front of the order
    double cum[MAX];                                  // and its running masses
    double tab[64];
    double mass, part[PICK_WAVES];
    uint32_t n, rest;
};

__device__ inline uint64_t lane_u64(uint64_t v, int l) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
__device__ inline void wave_lds() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }    // a wave's LDS accesses stay in order

// All four waves read the candidates; the first one decides, without a barrier (6 to 7 us for one row, 8 to 14 for 256: a
// chain of LDS and DPP steps, each waiting for the last): up to 512 (or 1,024) candidates in
// its registers, of which it sorts the next up to 64 at a time (bounded by a bisection) until
// the cuts and the draw fall within what is sorted.  Returns whether they did.
template <int PICK_PER>
__device__ inline bool pick_row(const SampleArgs &a, int64_t tok, const SampleCuts &cut, const Mass &ms, uint32_t bound,
                                double mass, PickLds<PICK_PER> &s) {
    constexpr int PICK_MAX = PickLds<PICK_PER>::MAX;
    const int lane = threadIdx.x & 63;
    const bool by_k = cut.top_k > 0 && cut.top_k < a.V;
    int n = (int)s.n;
    if (n == 0 || n > SMP_LIST || ms.vmax == INFINITY) return false;
    bool open = bound != 0;                           // tokens behind the candidates may stay, too
    uint64_t x[PICK_PER];
    if (n <= PICK_MAX) {
#pragma unroll
        for (int j = 0; j < PICK_PER; ++j) x[j] = 64 * j + lane < n ? s.list[64 * j + lane] : 0;
    } else {                                          // the largest of them that fit
        uint64_t lo = entry_from(0), hi = entry_from(sort_key((float)ms.vmax) + 1);    // more than fit reach lo, at most hi
        while (hi - lo > 1) {
            const uint64_t mid = lo + (hi - lo) / 2;
            int c = 0;
            for (int j = lane; j < n; j += 64) c += ge(s.list[j], mid);
            for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o, 64);
            if (c > PICK_MAX) lo = mid;
            else hi = mid;
            if (c == PICK_MAX) break;
        }
        int c = 0;
        for (int j0 = 0; j0 < n; j0 += 64) {          // moved to the front: never past where they are read
            const uint64_t e = j0 + lane < n ? s.list[j0 + lane] : 0;
            const uint64_t b = __ballot(ge(e, hi));
            wave_lds();
            if (ge(e, hi)) s.list[c + __popcll(b & ((1ull << lane) - 1))] = e;
            wave_lds();
            c += __popcll(b);
        }
        n = c;
        open = true;
#pragma unroll
        for (int j = 0; j < PICK_PER; ++j) x[j] = 64 * j + lane < n ? s.list[64 * j + lane] : 0;
    }
    int have = 0;                                     // sorted so far
    double sum = 0.0;                                 // their mass
    uint64_t below = ~0ull;                           // those left are below
    auto extend = [&]() {                             // sorts the next
        int c = n - have;
        uint64_t from = 1;
        if (c > 64) {
            // more than 64 of those left reach lo, at most 64 reach hi
            uint64_t lo = entry_from(bound), hi = min(below, entry_from(sort_key((float)ms.vmax) + 1));
            for (;;) {
                const uint64_t mid = lo + (hi - lo) / 2;
                c = 0;
#pragma unroll
                for (int j = 0; j < PICK_PER; ++j) c += __popcll(__ballot(ge(x[j], mid)));
                if (c > 64) lo = mid;
                else hi = mid;
                if (hi - lo == 1 || (c <= 64 && c >= 40)) break;
            }
            from = hi;
        }
        c = 0;
#pragma unroll
        for (int j = 0; j < PICK_PER; ++j) {
            const bool in = ge(x[j], from);
            const uint64_t b = __ballot(in);
            if (in) s.order[have + c + __popcll(b & ((1ull << lane) - 1))] = x[j];
            if (in) x[j] = 0;                         // taken
            c += __popcll(b);
        }
        wave_lds();
        const uint64_t mine = lane < c ? s.order[have + lane] : 0;
        int rank = 0;
#pragma unroll 16
        for (int l = 0; l < 64; ++l) rank += gt(lane_u64(mine, l), mine);
        wave_lds();
        if (lane < c) s.order[have + rank] = mine;
        wave_lds();
        const uint64_t sorted = lane < c ? s.order[have + lane] : 0;
        const double run = sum + wave_scan(lane < c ? ms.e(entry_key(sorted)) : 0.0);
        if (lane < c) s.cum[have + lane] = run;
        wave_lds();
        sum = s.cum[have + c - 1];
        below = from;
        have += c;
    };
    // the first of [0, to) with pred, or to
    auto first_of = [&](int to, auto pred) {
        for (int j0 = 0; j0 < to; j0 += 64) {
            const uint64_t b = __ballot(j0 + lane < to && pred(min(j0 + lane, to - 1)));
            if (b) return j0 + __ffsll((unsigned long long)b) - 1;
        }
        return to;
    };
    auto low = [&](int j) { return !(ms.e(entry_key(s.order[j])) >= (double)cut.min_p); };
    const double top_p = (double)fmaxf(cut.top_p, 0.0f);
    const bool with_p = cut.top_p < 1.0f, with_min = cut.min_p > 0.0f;
    if (by_k && cut.top_k <= n && cut.top_k <= 64) {  // (about what one round sorts)
        while (have < cut.top_k) extend();
        n = have = cut.top_k;
        sum = s.cum[n - 1];
        open = false;
    } else if (by_k && cut.top_k <= n) {              // the top_k candidates alone
        // at least top_k reach lo, fewer reach hi
        uint64_t lo = entry_from(bound), hi = entry_from(sort_key((float)ms.vmax) + 1);
        while (cut.top_k < n && hi - lo > 1) {
            const uint64_t mid = lo + (hi - lo) / 2;
            int c = 0;
#pragma unroll
            for (int j = 0; j < PICK_PER; ++j) c += __popcll(__ballot(ge(x[j], mid)));
            if (c >= cut.top_k) lo = mid;
            else hi = mid;
            if (c == cut.top_k) break;
        }
#pragma unroll
        for (int j = 0; j < PICK_PER; ++j)
            if (!ge(x[j], lo)) x[j] = 0;
        n = cut.top_k;
        open = false;
    }
    const bool sure = !by_k || !open;                 // the mass that top-p takes its share of is known
    double total = mass;
    if (have < n) {
        // the mass of the candidates, which lie in no certain order: a sum of integers, the 53 bits of e below 1 and the
        // 53 after them (1,024 of at most 2^53)
        uint64_t hi = 0, lo = 0;
        bool low_one = false;
#pragma unroll
        for (int j = 0; j < PICK_PER; ++j) {
            const double e = x[j] ? ms.e(entry_key(x[j])) : 0.0, h = e * 0x1p53, f = floor(h);
            hi += (uint64_t)f;
            lo += (uint64_t)((h - f) * 0x1p53);
            low_one |= x[j] && !(e >= (double)cut.min_p);
        }
        hi = lane_u64(wave_scan(hi), 63);
        lo = lane_u64(wave_scan(lo), 63);
        const double all = (double)hi * 0x1p-53 + (double)lo * 0x1p-106;
        const bool any_low = with_min && __ballot(low_one);
        if (!open) total = all;
        if (open) {                                   // all candidates together may not reach far enough
            if (!sure && (with_p || !any_low)) return false;
            const double reach = with_p || with_min ? top_p * total : cut.u * total;
            if (all * (1.0 + 1e-12) < reach && !any_low) return false;
        }
        do extend();
        while (have < n && !(with_p && sure && sum >= top_p * total) && !(with_min && low(have - 1)) &&
               !(!with_p && !with_min && sum > cut.u * total));
    }
    int kept = have;                                  // how many of the order stay
    if (!open && have == n) total = sum;
    if (with_p && sure) {
        const double want = top_p * total;
        const int f = first_of(kept, [&](int j) { return s.cum[j] >= want; });
        if (f < kept) { kept = f + 1; open = false; total = s.cum[f]; }
    }
    if (with_min) {
        const int f = first_of(kept, low);
        if (f < kept) { kept = max(f, 1); open = false; total = s.cum[kept - 1]; }
    }
    if (open && (with_p || with_min || by_k)) return false;
    const double t = cut.u * total;
    const int at = first_of(kept, [&](int j) { return s.cum[j] > t; });
    if (at == kept) return false;                     // behind the candidates
    if (lane == 0) {
        const uint64_t e = s.order[at];
        a.tokens[tok] = entry_token(e);
        if (a.probs) a.probs[tok] = (float)(ms.e(entry_key(e)) / total);
    }
    return true;
}

template <int PER>
__global__ __launch_bounds__(PICK_THREADS) void sample_pick_kernel(SampleArgs a) {
    __shared__ PickLds<PER> s;
    const int64_t tok = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const SliceHead *heads = (const SliceHead *)a.heads + tok * a.slices;
    const uint64_t *lists = (const uint64_t *)a.lists + (size_t)(tok * a.slices) * a.cap;
    // every load first: each wave the heads of all slices, each thread its places in the slices' lists (what lies
    // behind a list's end is read and left out)
    constexpr int HEADS = SLICES_MAX / 64, FIRST = 8;
    SliceHead hd[HEADS];
    uint64_t en[FIRST];
    uint32_t en_n[FIRST];
    const int places = a.slices << a.cap_log;
#pragma unroll
    for (int i = 0; i < HEADS; ++i)
        if (lane + 64 * i < a.slices) hd[i] = heads[lane + 64 * i];
        else hd[i] = SliceHead{0.0, -INFINITY, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < FIRST; ++i) {
        const int p = tid + PICK_THREADS * i;
        en_n[i] = p < places ? heads[p >> a.cap_log].n : 0;
        en[i] = p < places ? lists[p] : 0;
    }
    const SampleCuts cut = load_cuts(a, tok);
    if (tid < 64) s.tab[tid] = EXP_TAB[tid];
    if (tid == 0) s.n = 0;
    float vmax = -INFINITY;
    uint32_t bound = 0;
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        vmax = fmaxf(vmax, hd[i].vmax);
        bound = max(bound, hd[i].bound);
    }
    vmax = wave_max(vmax);
    for (int o = 32; o > 0; o >>= 1) bound = max(bound, (uint32_t)__shfl_xor(bound, o, 64));
    if (vmax == -INFINITY) {                          // nothing is on
        if (tid == 0) {
            a.tokens[tok] = -1;
            if (a.probs) a.probs[tok] = 0.0f;
        }
        return;
    }
    if (!(cut.temp > 0.0f)) {
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < HEADS; ++i)
            if (hd[i].vmax == vmax) at = min(at, hd[i].at);
        for (int o = 32; o > 0; o >>= 1) at = min(at, (uint32_t)__shfl_xor(at, o, 64));
        if (tid == 0) {
            a.tokens[tok] = (int32_t)at;
            if (a.probs) a.probs[tok] = 1.0f;
        }
        return;
    }
    const Mass ms = row_mass(vmax, cut.temp, s.tab, 0);
    __syncthreads();
    auto take = [&](bool in, uint64_t e) {            // one place in the list for a wave's at a time
        const uint64_t b = __ballot(in);
        if (!b) return;
        uint32_t at = 0;
        if (lane == 0) at = atomicAdd(&s.n, (uint32_t)__popcll(b));
        at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + (uint32_t)__popcll(b & ((1ull << lane) - 1));
        if (in && at < SMP_LIST) s.list[at] = e;
    };
    const uint32_t in_list = (1u << a.cap_log) - 1;
#pragma unroll
    for (int i = 0; i < FIRST; ++i) {
        const int p = tid + PICK_THREADS * i;
        take(((uint32_t)p & in_list) < en_n[i] && entry_key(en[i]) >= bound, en[i]);
    }
    for (int p0 = PICK_THREADS * FIRST; p0 < places; p0 += PICK_THREADS) {
        const int p = min(p0 + tid, places - 1);
        const uint64_t e = lists[p];
        take(p0 + tid < places && ((uint32_t)p & in_list) < heads[p >> a.cap_log].n && entry_key(e) >= bound, e);
    }
    __syncthreads();
    if (tid < 64) {
        double mass = 0.0;                            // of the row, where it counts
        if (!(cut.top_k > 0 && cut.top_k < a.V)) {
#pragma unroll
            for (int i = 0; i < HEADS; ++i)
                if (hd[i].vmax > -INFINITY) mass += hd[i].mass * exp64(((double)hd[i].vmax - ms.vmax) * ms.c, s.tab);
            for (int o = 1; o < 64; o <<= 1) mass += __shfl_xor(mass, o, 64);
        }
        const bool done = pick_row(a, tok, cut, ms, bound, mass, s);
        if (lane == 0) {
            s.rest = done ? 0xffffffffu : atomicAdd(a.n_rest, 1u);
            s.mass = mass;
        }
    }
    __syncthreads();
    if (s.rest == 0xffffffffu) return;
    RestRow &r = ((RestRow *)a.rest)[s.rest];         // undecided: step 3
    for (int i = tid; i < SMP_BINS; i += PICK_THREADS) { r.cnt[i] = 0; r.mass[i] = 0; }
    // Its masses are integers with as many fractional bits as the row's whole mass leaves of 62: a token far below the
    // first has its share to 2^-62 of the whole.  Under a top-k that mass is not known, but the candidates' and as much as the
    // bound's for every token are no less.
    double whole = s.mass;
    if (cut.top_k > 0 && cut.top_k < a.V) {
        double t = 0.0;
        for (int p = tid; p < places; p += PICK_THREADS) {
            const uint64_t e = lists[p];
            if (((uint32_t)p & in_list) < heads[p >> a.cap_log].n && entry_key(e) >= bound) t += ms.e(entry_key(e));
        }
        for (int o = 1; o < 64; o <<= 1) t += __shfl_xor(t, o, 64);
        if (lane == 0) s.part[tid >> 6] = t;
        __syncthreads();
        whole = bound ? (double)a.V * ms.e(min(bound, sort_key(vmax))) : 0.0;
        for (int w = 0; w < PICK_WAVES; ++w) whole += s.part[w];
    }
    if (vmax == INFINITY) whole = a.V;                // every one of them counts 1
    if (tid == 0) {
        int ex;
        frexp(whole * (1.0 + 1e-9), &ex);
        r.shift = 62 - ex;
        r.bound = bound;
        r.tok = tok;
        r.vmax = vmax;
        r.parts = 0;
    }
}

// ---------------------------------------------------------------------------
// slices of a row, candidates that a slice has room for, and lanes above its bound
struct SamplePlan {
    int slices, cap_log, keep, parts;
};
// `want` candidates of a slice, 300 to 600 of a row: enough for a top-k of 200 and most cuts by mass, and few enough for one
// wave's registers.  Half as many: 693 us against 80 for 256 rows of 151,936 with cuts of their own (top-k up to 200), whose
// undecided ones fill step 3; twice as many: 51 against 15 for one row under top-k, whose candidates do not fit.
// A row of up to 1,000 is kept whole: it needs no step 3 but for a logit of +inf.
static SamplePlan sample_plan(int V) {
    SamplePlan p;
    p.slices = (V + 7 + SLICE - 1) / SLICE;           // (7: a row may begin inside 16 bytes)
    const int want = p.slices >= 64 ? 8 : p.slices >= 25 ? 16 : 400 / p.slices;
    // of 64 maxima over runs of random values, those above the value that `want` of all exceed
    p.keep = V <= 1000 ? 65 : (int)ceil(64.0 * (1.0 - exp(-want / 64.0)));
    p.parts = V < 16384 ? 1 : V >= 131072 ? 16 : V / 8192;       // workgroups to an undecided row, 8,192 logits to each
    p.cap_log = 4;
    while ((1 << p.cap_log) < want + want / 2 + 8) ++p.cap_log;
    return p;
}

struct SampleWs {
    size_t lists, heads, rest, n_rest, total;
};
constexpr int SMP_ROWS = 4096;                        // of a launch: bounds the workspace
static SampleWs sample_ws(int n_tok, int V) {
    const SamplePlan p = sample_plan(V);
    if (n_tok > SMP_ROWS) n_tok = SMP_ROWS;
    SampleWs w;
    size_t o = 0;
    w.lists = o; o += (size_t)n_tok * p.slices << (p.cap_log + 3);
    w.heads = o; o += (size_t)n_tok * p.slices * sizeof(SliceHead);
    w.rest = o; o += (size_t)n_tok * sizeof(RestRow);
    w.n_rest = o; o += 8;
    w.total = o;
    return w;
}
size_t sample_ws_bytes(int n_tok, int V) { return sample_ws(n_tok, V).total; }

template <int T>
static hipError_t launch_sample_t(const SampleArgs &a, hipStream_t st) {
    const int64_t waves = (int64_t)a.n_tok * a.slices;
    hipLaunchKernelGGL(sample_slice_kernel<T>, dim3((unsigned)((waves + SLICE_WAVES - 1) / SLICE_WAVES)),
                       dim3(64 * SLICE_WAVES), 0, st, a);
    // short rows have all or most of theirs in one or two lists
    if (a.slices <= 2) hipLaunchKernelGGL(sample_pick_kernel<16>, dim3((unsigned)a.n_tok), dim3(PICK_THREADS), 0, st, a);
    else hipLaunchKernelGGL(sample_pick_kernel<8>, dim3((unsigned)a.n_tok), dim3(PICK_THREADS), 0, st, a);
    hipLaunchKernelGGL(sample_rest_kernel<T>, dim3((unsigned)min((int64_t)REST_GRID, (int64_t)a.n_tok * a.parts)), dim3(SMP_THREADS), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_sample(SampleArgs a, void *ws, hipStream_t st) {
    const SamplePlan p = sample_plan(a.V);
    const SampleWs w = sample_ws(a.n_tok, a.V);
    a.slices = p.slices;
    a.cap_log = p.cap_log;
    a.cap = 1 << p.cap_log;
    a.keep = p.keep;
    a.parts = p.parts;
    a.lists = (uint8_t *)ws + w.lists;
    a.heads = (uint8_t *)ws + w.heads;
    a.rest = (uint8_t *)ws + w.rest;
    a.n_rest = (uint32_t *)((uint8_t *)ws + w.n_rest);
    const int all = a.n_tok;
    for (int t = 0; t < all; t += SMP_ROWS) {         // one after the other in the same workspace
        a.n_tok = all - t < SMP_ROWS ? all - t : SMP_ROWS;
        const hipError_t e = a.type == T_F32 ? launch_sample_t<T_F32>(a, st)
                           : a.type == T_BF16 ? launch_sample_t<T_BF16>(a, st) : launch_sample_t<T_F16>(a, st);
        if (e != hipSuccess) return e;
        a.logits = (const uint8_t *)a.logits + (int64_t)SMP_ROWS * a.ld * (a.type == T_F32 ? 4 : 2);
        a.u += SMP_ROWS;
        a.tokens += SMP_ROWS;
        if (a.probs) a.probs += SMP_ROWS;
        if (a.temp) a.temp += SMP_ROWS;
        if (a.top_k) a.top_k += SMP_ROWS;
        if (a.top_p) a.top_p += SMP_ROWS;
        if (a.min_p) a.min_p += SMP_ROWS;
    }
    return hipSuccess;
}

}  // namespace mp
