/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_sample.hip - a token of each row of logits by temperature, top-k, top-p
 * and min-p from a given random number, on gfx950.
 *
 * With z = x log2(e) / T a token weighs 2^z. All limits cut the order of
 * descending logits after some token, and the pick is where a running sum of that
 * order passes u times the sum of what is left; so the rows need no sort but the
 * place of a few sums. The order is cut into bins by floor(32 z): a token's weight
 * is known to 2^(1/32) by its bin, and the sums over bins say which bin a limit or
 * the pick falls into. Only that bin's tokens are put in order.
 *
 * Sums are of whole numbers, 2^(z - E) 2^sh with E an integer that no z of the
 * row passes, so that they do not depend on their order. A workgroup that has seen
 * a slice of a row takes its own E; the bins are at the same z for all, and
 * sums are shifted to the row's E when they are added. z and the weights are in
 * 64 bits: a pick that is wrong by a rounding is another token.
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

namespace {

#include "dsv4_rows_io.h"

typedef unsigned long long u64;

constexpr int SM_THREADS = 256;
constexpr int SM_EACH = 32;                       /* tokens of a thread      */
constexpr int SM_SLICE = SM_THREADS * SM_EACH;
constexpr int SM_BINS = 1024;                     /* 32 octaves, the rest in the last */
constexpr int SM_CHUNK = 64;                      /* tokens with one maximum */
constexpr int SP_THREADS = 1024;                  /* of a row's pick         */
constexpr int SP_WAVES = SP_THREADS / 64;
static_assert(SP_THREADS == SM_BINS, "a bin a thread");

struct SampleJob {
    const void *x;
    long long stride;
    int n, vocab, ns, nc, sh;                     /* slices, chunks of a row */
    dsv4_gpu_sampling r;
    u64 *mass;                                    /* [n][ns][bins]           */
    uint32_t *count;
    double *top;                                  /* [n][ns]: the first bin's 32 z */
    float *cmax;                                  /* [n][nc]                 */
    int *kept;
    float *prob;
};

/* 2^f, |f| <= 1/2: the exponential's series to f^11, 6e-15 off at the most. */
__device__ __forceinline__ double sm_exp2_part(double f)
{
    double p = 4.44553827187081e-10;
    p = fma(p, f, 7.054911620801121e-09);
    p = fma(p, f, 1.0178086009239696e-07);
    p = fma(p, f, 1.3215486790144305e-06);
    p = fma(p, f, 1.5252733804059838e-05);
    p = fma(p, f, 0.00015403530393381606);
    p = fma(p, f, 0.0013333558146428441);
    p = fma(p, f, 0.009618129107628477);
    p = fma(p, f, 0.055504108664821576);
    p = fma(p, f, 0.2402265069591007);
    p = fma(p, f, 0.6931471805599453);
    return fma(p, f, 1.0);
}

/* 2^t, t <= 0; 0 below 2^-64. */
__device__ __forceinline__ double sm_exp2(double t)
{
    if (!(t > -64.0)) return 0.0;
    const double n = __builtin_rint(t);
    return sm_exp2_part(t - n) * __hiloint2double((1023 + (int)n) << 20, 0);
}

/* 2^t 2^sh as a whole number, t <= 0, sh <= 50: added to 2^52 it is rounded to
 * one, in the low bits. */
__device__ __forceinline__ u64 sm_weight(double t, int sh)
{
    if (!(t > -64.0)) return 0;
    const double n = __builtin_rint(t);
    const double s = __hiloint2double((1023 + (int)n + sh) << 20, 0);
    return (u64)__double_as_longlong(fma(sm_exp2_part(t - n), s, 4503599627370496.0)) &
           ((1ull << 52) - 1);
}

/* z of a row's tokens. Where its largest logit is infinite, z is 0 for those that
 * are and -infinity for the others. */
struct SmScale {
    double c;
    bool inf;
    __device__ __forceinline__ double z(float x) const
    {
        return inf ? (x == INFINITY ? 0.0 : -INFINITY) : (double)x * c;
    }
};
__device__ __forceinline__ double sm_q(double z) { return floor(z * 32.0); }
/* E of a row or slice whose first bin is q: no z passes it */
__device__ __forceinline__ double sm_e(double q) { return floor(q * (1.0 / 32.0)) + 1.0; }
__device__ __forceinline__ int sm_bin(double top, double q)
{
    const double d = top - q;
    return d < SM_BINS - 1 ? (int)d : SM_BINS - 1;
}

__device__ __forceinline__ float sm_temperature(const SampleJob &a, int row)
{
    return a.r.temperature ? a.r.temperature[row] : 1.0f;
}

/* A slice of a row: the maxima of its chunks, and its bins' counts and sums. */
template <class T>
__global__ void __launch_bounds__(SM_THREADS) k_sample_slices(SampleJob a)
{
    __shared__ u64 mass[SM_BINS];
    __shared__ uint32_t count[SM_BINS];
    __shared__ float wtop[SM_THREADS / 64];
    const int tid = threadIdx.x;
    const int row = blockIdx.x / a.ns, slice = blockIdx.x - row * a.ns;
    const int v0 = slice * SM_SLICE;
    const T *x = (const T *)a.x + (size_t)row * a.stride + v0;
    const int lim = min(SM_SLICE, a.vocab - v0);
    float v[SM_EACH];
#pragma unroll
    for (int p = 0; p < SM_EACH / 4; p++) {
        const int c = (p * SM_THREADS + tid) * 4;
        if (lim == SM_SLICE) {
            io_load<T, 4>(x + c, v + 4 * p);
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                v[4 * p + k] = -INFINITY;
                if (c + k < lim) io_load<T, 1>(x + c + k, v + 4 * p + k);
            }
        }
    }
    const float temp = sm_temperature(a, row);
    float top = -INFINITY;
#pragma unroll
    for (int p = 0; p < SM_EACH / 4; p++) {
        /* (NaN: fmaxf takes the other) */
        float m = fmaxf(fmaxf(v[4 * p], v[4 * p + 1]), fmaxf(v[4 * p + 2], v[4 * p + 3]));
        m = fmaxf(m, -INFINITY);
        m = fmaxf(m, dpp_f<DPP_QUAD_XOR1, 0xF>(m));
        m = fmaxf(m, dpp_f<DPP_QUAD_XOR2, 0xF>(m));
        m = fmaxf(m, dpp_f<DPP_ROW_HMIRROR, 0xF>(m));
        m = fmaxf(m, dpp_f<DPP_ROW_MIRROR, 0xF>(m));
        const int chunk = (v0 + p * SM_THREADS * 4) / SM_CHUNK + tid / 16;
        if ((tid & 15) == 0 && chunk < a.nc) a.cmax[(size_t)row * a.nc + chunk] = m;
        top = fmaxf(top, m);
    }
    if (!(temp > 0.0f)) return;                   /* the first is picked     */

    for (int i = tid; i < SM_BINS; i += SM_THREADS) {
        mass[i] = 0;
        count[i] = 0;
    }
    top = wave_max(top);
    if ((tid & 63) == 0) wtop[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SM_THREADS / 64; k++) top = fmaxf(top, wtop[k]);
    const size_t at = (size_t)row * a.ns + slice;
    if (top == -INFINITY) {
        if (tid == 0) a.top[at] = -INFINITY;
        return;
    }
    const SmScale sc{1.4426950408889634 / (double)temp, top == INFINITY};
    const double first = sm_q(sc.z(top)), e = sm_e(first);
#pragma unroll
    for (int k = 0; k < SM_EACH; k++) {
        if (!(v[k] > -INFINITY)) continue;
        const double z = sc.z(v[k]);
        const int bin = sm_bin(first, sm_q(z));
        const u64 w = sm_weight(z - e, a.sh);
        atomicAdd(&count[bin], 1u);
        if (w) atomicAdd(&mass[bin], w);
    }
    __syncthreads();
    for (int i = tid; i < SM_BINS; i += SM_THREADS) {
        a.mass[at * SM_BINS + i] = mass[i];
        a.count[at * SM_BINS + i] = count[i];
    }
    if (tid == 0) a.top[at] = sc.inf ? INFINITY : first;
}

/* u s for 0 <= u < 1 and s < 2^63, exactly, rounded down or up. */
__device__ __forceinline__ u64 sm_part(float u, u64 s, bool up)
{
    const uint32_t b = __float_as_uint(u), ex = b >> 23;
    const u64 m = ex ? (b & 0x7FFFFFu) | 0x800000u : b & 0x7FFFFFu;
    const int sh = 150 - (int)(ex ? ex : 1u);     /* u = m 2^-sh, sh >= 24   */
    const u64 lo = s * m, hi = __umul64hi(s, m);
    u64 f;
    bool rest;
    if (sh < 64) {
        f = lo >> sh | hi << (64 - sh);
        rest = (lo & ((1ull << sh) - 1)) != 0;
    } else if (sh < 128) {
        f = hi >> (sh - 64);
        rest = lo != 0 || (hi & ((1ull << (sh - 64)) - 1)) != 0;
    } else {
        f = 0;
        rest = (lo | hi) != 0;
    }
    return f + (up && rest ? 1 : 0);
}

__device__ __forceinline__ float sm_value(u64 key)
{
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ int sm_token(u64 key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }

/* A place in a row's order: a token (its key, am_key), with the tokens and the sum
 * through it. */
struct SmPlace {
    u64 key, sum;
    int bin, n;
};

/* The workgroup of a row. */
template <class T>
struct SmRow {
    struct Lds {
        u64 sum[SM_BINS];                         /* through a bin           */
        uint32_t n[SM_BINS];
        u64 mass[SP_THREADS], best[SP_THREADS];   /* a split of a key range  */
        uint32_t cnt[SP_THREADS];
        u64 key[SP_THREADS], w[SP_THREADS];       /* a bin's tokens          */
        u64 part[SP_WAVES];
        uint32_t npart[SP_WAVES];
        SmPlace hit;
        u64 range[2];
        int len, held;                            /* tokens listed, their bin */
        double slices[2];
        float top;
    };
    const SampleJob &a;
    Lds &s;
    const T *x;
    const float *cmax;
    SmScale sc;
    double first, e;

    /* Inclusive sums over the threads. */
    __device__ void scan(u64 &m, uint32_t &n)
    {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const u64 u = __shfl_up(m, o, 64);
            const uint32_t v = __shfl_up(n, o, 64);
            if (lane >= o) {
                m += u;
                n += v;
            }
        }
        __syncthreads();
        if (lane == 63) {
            s.part[w] = m;
            s.npart[w] = n;
        }
        __syncthreads();
        for (int k = 0; k < w; k++) {
            m += s.part[k];
            n += s.npart[k];
        }
    }

    /* f(key, weight) for every token of a bin, from the row. A chunk whose largest
     * is in a later bin has none. */
    template <class F>
    __device__ void each_of_row(int bin, F f)
    {
        constexpr int G = 8;                      /* chunks in flight        */
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        for (int c0 = w * 64; c0 < a.nc; c0 += SP_THREADS) {
            const int c = c0 + lane;
            const float top = c < a.nc ? cmax[c] : -INFINITY;
            u64 want = __ballot(top > -INFINITY && sm_bin(first, sm_q(sc.z(top))) <= bin);
            while (want) {
                float v[G];
                int t[G];
#pragma unroll
                for (int u = 0; u < G; u++) {
                    t[u] = a.vocab;
                    if (want) {
                        t[u] = (c0 + __builtin_ctzll(want)) * SM_CHUNK + lane;
                        want &= want - 1;
                    }
                    v[u] = -INFINITY;
                    if (t[u] < a.vocab) io_load<T, 1>(x + t[u], v + u);
                }
#pragma unroll
                for (int u = 0; u < G; u++) {
                    if (!(v[u] > -INFINITY)) continue;
                    const double z = sc.z(v[u]);
                    if (sm_bin(first, sm_q(z)) == bin)
                        f(am_key(v[u], t[u]), sm_weight(z - e, a.sh));
                }
            }
        }
    }

    /* List a bin's tokens, if they fit. */
    __device__ void hold(int bin)
    {
        if (s.held == bin) return;                /* the same in every thread */
        __syncthreads();
        if (threadIdx.x == 0) s.len = 0;
        __syncthreads();
        const uint32_t n = s.n[bin] - (bin ? s.n[bin - 1] : 0);
        if (n <= SP_THREADS)
            each_of_row(bin, [&](u64 key, u64 w) {
                const int at = atomicAdd(&s.len, 1);
                if (at < SP_THREADS) {
                    s.key[at] = key;
                    s.w[at] = w;
                }
            });
        __syncthreads();
        if (threadIdx.x == 0) s.held = n <= SP_THREADS ? bin : -1;
        __syncthreads();
    }

    template <class F>
    __device__ void each(int bin, F f)
    {
        if (s.held != bin) each_of_row(bin, f);
        else if ((int)threadIdx.x < s.len) f(s.key[threadIdx.x], s.w[threadIdx.x]);
    }

    /* Where the order passes `need` tokens (tokens true) or the sum `need`, in a bin
     * which that is known to be: the first token through which there are as many,
     * or, where roundings of the bins' sums leave them short, the bin's last. The
     * bin's range of keys is split by 1024 until the token is alone. */
    __device__ SmPlace cross(int bin, u64 need, bool tokens)
    {
        hold(bin);
        const int tid = threadIdx.x;
        u64 lo = 0, hi = ~0ull, sum0 = bin ? s.sum[bin - 1] : 0;
        uint32_t n0 = bin ? s.n[bin - 1] : 0;
        if (s.held == bin) {
            if (tid == 0) {
                s.range[0] = ~0ull;
                s.range[1] = 0;
            }
            __syncthreads();
            if (tid < s.len) {
                atomicMin(&s.range[0], s.key[tid]);
                atomicMax(&s.range[1], s.key[tid]);
            }
            __syncthreads();
            lo = s.range[0];
            hi = s.range[1];
        }
        for (;;) {
            const int bits = 64 - __clzll((long long)((hi - lo) | 1));
            const int sh = max(0, bits - 10);
            s.mass[tid] = 0;
            s.best[tid] = 0;
            s.cnt[tid] = 0;
            if (tid == 0) s.hit.bin = -1;
            __syncthreads();
            each(bin, [&](u64 key, u64 w) {
                if (key < lo || key > hi) return;
                const int d = (int)((hi - key) >> sh);
                atomicAdd(&s.mass[d], w);
                atomicAdd(&s.cnt[d], 1u);
                atomicMax(&s.best[d], key);
            });
            __syncthreads();
            const u64 m = s.mass[tid];
            const uint32_t n = s.cnt[tid];
            u64 mi = m;
            uint32_t ni = n;
            scan(mi, ni);
            const u64 through = tokens ? n0 + ni : sum0 + mi;
            const u64 before = tokens ? n0 + ni - n : sum0 + mi - m;
            /* the split that passes it; the last one with tokens has no more behind */
            if (n && before < need && through >= need) s.hit = {s.best[tid], sum0 + mi, tid, (int)(n0 + ni)};
            __syncthreads();
            if (s.hit.bin < 0) {
                __syncthreads();
                if (n) atomicMax(&s.hit.bin, tid);
                __syncthreads();
                const int last = s.hit.bin;
                __syncthreads();
                if (tid == last) s.hit = {s.best[tid], sum0 + mi, tid, (int)(n0 + ni)};
                if (last < 0 && tid == 0) s.hit = {0, sum0, 0, (int)n0};
                __syncthreads();
            }
            const int d = s.hit.bin;
            SmPlace p = s.hit;
            const uint32_t nd = s.cnt[d];
            const u64 md = s.mass[d];
            __syncthreads();
            if (nd <= 1 || sh == 0) {
                p.bin = bin;
                return p;
            }
            n0 = p.n - nd;
            sum0 = p.sum - md;
            hi = p.key;
            const u64 end = hi > ((1ull << sh) - 1) ? hi - ((1ull << sh) - 1) : 0;
            lo = end > lo ? end : lo;
        }
    }
};

template <class T>
__global__ void __launch_bounds__(SP_THREADS) k_sample_pick(SampleJob a, int *d_pick)
{
    using Row = SmRow<T>;
    __shared__ typename Row::Lds s;
    const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
    const float temp = sm_temperature(a, row);
    Row r{a, s, (const T *)a.x + (size_t)row * a.stride, a.cmax + (size_t)row * a.nc,
          SmScale{0.0, false}, 0.0, 0.0};
    auto done = [&](int pick, float prob, int kept) {
        d_pick[row] = pick;
        if (a.prob) a.prob[row] = prob;
        if (a.kept) a.kept[row] = kept;
    };

    if (!(temp > 0.0f)) {
        /* the first chunk with the largest, and the first in it */
        u64 best = 0;
        for (int c = tid; c < a.nc; c += SP_THREADS) {
            const u64 k = r.cmax[c] > -INFINITY ? am_key(r.cmax[c], c) : 0;
            best = k > best ? k : best;
        }
        best = wave_max_u64(best);
        if (lane == 0) s.part[tid >> 6] = best;
        __syncthreads();
        if (tid >= 64) return;
        best = 0;
        for (int k = 0; k < SP_WAVES; k++) best = s.part[k] > best ? s.part[k] : best;
        if (best == 0) {
            if (tid == 0) done(-1, 0.0f, 0);
            return;
        }
        const int t = sm_token(best) * SM_CHUNK + lane;
        float v = -INFINITY;
        if (t < a.vocab) io_load<T, 1>(r.x + t, &v);
        const u64 k = wave_max_u64(v > -INFINITY ? am_key(v, t) : 0);
        if (tid == 0) done(sm_token(k), 1.0f, 1);
        return;
    }

    /* ---- the slices' bins as the row's ---- */
    const double *tops = a.top + (size_t)row * a.ns;
    double top = -INFINITY;
    for (int k = 0; k < a.ns; k++) top = fmax(top, tops[k]);
    if (top == -INFINITY) {
        if (tid == 0) done(-1, 0.0f, 0);
        return;
    }
    r.sc = SmScale{1.4426950408889634 / (double)temp, top == INFINITY};
    r.first = r.sc.inf ? 0.0 : top;
    r.e = sm_e(r.first);
    s.sum[tid] = 0;
    s.n[tid] = 0;
    if (tid == 0) s.held = -1;
    __syncthreads();
    for (int k = 0; k < a.ns; k++) {
        const double t = tops[k];
        if (t == -INFINITY) continue;
        const size_t at = ((size_t)row * a.ns + k) * SM_BINS + tid;
        const uint32_t n = a.count[at];
        if (!n) continue;
        u64 m = a.mass[at];
        int d = 0, sh = 0;
        if (t != top) {
            const double de = r.e - sm_e(t);
            d = r.sc.inf ? SM_BINS : sm_bin(top, t);
            sh = r.sc.inf || de >= 63.0 ? 63 : (int)de;
            if (sh) m = (m + (1ull << (sh - 1))) >> sh;
        }
        const int bin = tid == SM_BINS - 1 ? tid : min(tid + d, SM_BINS - 1);
        atomicAdd(&s.n[bin], n);
        atomicAdd(&s.sum[bin], m);
    }
    __syncthreads();
    const u64 m = s.sum[tid];
    const uint32_t n = s.n[tid];
    u64 mi = m;
    uint32_t ni = n;
    r.scan(mi, ni);
    s.sum[tid] = mi;
    s.n[tid] = ni;
    __syncthreads();

    /* ---- the last token left: key 0 is behind its whole bin ---- */
    SmPlace cut{0, s.sum[SM_BINS - 1], SM_BINS - 1, (int)s.n[SM_BINS - 1]};
    /* the first bin through which it is; the last, where roundings pass the sum */
    auto bin_of = [&](u64 need, bool tokens) {
        __syncthreads();
        if (tid == 0) s.hit.bin = SM_BINS - 1;
        __syncthreads();
        const u64 through = tokens ? ni : mi, before = tokens ? ni - n : mi - m;
        if (n && before < need && through >= need) s.hit.bin = tid;
        __syncthreads();
        return s.hit.bin;
    };
    const int k = a.r.top_k ? a.r.top_k[row] : 0;
    if (k > 0 && k < cut.n) cut = r.cross(bin_of((u64)k, true), (u64)k, true);
    const float p = a.r.top_p ? a.r.top_p[row] : 1.0f;
    if (p < 1.0f) {
        const u64 part = p > 0.0f ? sm_part(p, cut.sum, true) : 0;
        const u64 need = part > 1 ? part : 1;
        const int b = bin_of(need, false);
        if (b < cut.bin || (b == cut.bin && need < cut.sum)) cut = r.cross(b, need, false);
    }
    const float floor_ = a.r.min_p ? fminf(a.r.min_p[row], 1.0f) : 0.0f;
    if (floor_ > 0.0f) {
        /* tokens from z of the largest + log2(min_p) on */
        float best = -INFINITY;
        for (int c = tid; c < a.nc; c += SP_THREADS) best = fmaxf(best, r.cmax[c]);
        best = wave_max(best);
        __syncthreads();
        if (lane == 0) s.part[tid >> 6] = __float_as_uint(best);
        __syncthreads();
        for (int w = 0; w < SP_WAVES; w++) best = fmaxf(best, __uint_as_float((uint32_t)s.part[w]));
        const double zmin = r.sc.z(best) + log2((double)floor_);
        const int b = sm_bin(r.first, sm_q(zmin));
        if (b <= cut.bin) {
            r.hold(b);
            __syncthreads();
            if (tid == 0) s.hit = {~0ull, b ? s.sum[b - 1] : 0, b, (int)(b ? s.n[b - 1] : 0)};
            __syncthreads();
            const u64 last = cut.bin == b ? cut.key : 0;
            r.each(b, [&](u64 key, u64 w) {
                if (key < last || r.sc.z(sm_value(key)) < zmin) return;
                atomicMin(&s.hit.key, key);
                atomicAdd(&s.hit.sum, w);
                atomicAdd(&s.hit.n, 1);
            });
            __syncthreads();
            if (s.hit.n < cut.n) cut = s.hit;
            __syncthreads();
        }
    }

    /* ---- the pick ---- */
    float u = a.r.u[row];
    u64 t = cut.sum - 1;
    if (!(u >= 1.0f)) t = min(t, u > 0.0f ? sm_part(u, cut.sum, false) : 0);
    const int b = min(bin_of(t + 1, false), cut.bin);
    const SmPlace at = r.cross(b, t + 1, false);
    if (tid == 0) {
        /* behind the cut only by the roundings of the bins' sums */
        const u64 key = b == cut.bin && at.key < cut.key ? cut.key : at.key;
        const double w = sm_exp2(r.sc.z(sm_value(key)) - r.e) * __hiloint2double((1023 + a.sh) << 20, 0);
        done(sm_token(key), (float)(w / (double)cut.sum), cut.n);
    }
}

struct SamplePlan {
    int ns, nc, sh;
    size_t mass, count, top, cmax, bytes;         /* offsets                 */
};

SamplePlan sample_plan(int n, int vocab)
{
    SamplePlan p;
    p.ns = (vocab + SM_SLICE - 1) / SM_SLICE;
    p.nc = (vocab + SM_CHUNK - 1) / SM_CHUNK;
    /* sums stay below 2^62 */
    int bits = 0;
    while ((1ll << bits) < vocab) bits++;
    p.sh = 62 - bits < 50 ? 62 - bits : 50;
    const size_t slices = (size_t)n * p.ns;
    p.mass = 0;
    p.top = p.mass + slices * SM_BINS * sizeof(u64);
    p.count = p.top + slices * sizeof(double);
    p.cmax = p.count + slices * SM_BINS * sizeof(uint32_t);
    p.bytes = (p.cmax + (size_t)n * p.nc * sizeof(float) + 15) / 16 * 16;
    return p;
}

constexpr int SM_ROWS = 65536, SM_VOCAB = 1 << 22;

template <class T>
int sample_launch(const SampleJob &a, int *d_pick, hipStream_t st)
{
    hipLaunchKernelGGL(k_sample_slices<T>, dim3((unsigned)a.n * (unsigned)a.ns), dim3(SM_THREADS),
                       0, st, a);
    HIP_OK(hipGetLastError(), "sample slices launch");
    hipLaunchKernelGGL(k_sample_pick<T>, dim3((unsigned)a.n), dim3(SP_THREADS), 0, st, a,
                       d_pick);
    HIP_OK(hipGetLastError(), "sample pick launch");
    return 0;
}

} // namespace

extern "C" size_t dsv4_gpu_sample_scratch_bytes(int n, int vocab)
{
    if (n <= 0 || n > SM_ROWS || vocab <= 0 || vocab > SM_VOCAB) return 0;
    return sample_plan(n, vocab).bytes;
}

extern "C" int dsv4_gpu_sample_d(int *d_pick, float *d_prob, int *d_kept, const void *d_logits,
                                 int fmt, int n, int vocab, long long stride,
                                 const dsv4_gpu_sampling *s, void *d_scratch,
                                 size_t scratch_bytes, void *stream)
{
    if ((fmt != DSV4_WF32 && fmt != DSV4_WBF16) || n < 0 || n > SM_ROWS || vocab <= 0 ||
        vocab > SM_VOCAB || stride < vocab || !s) {
        DSV4_ERR("sample: bad arguments (fmt %d, n %d, vocab %d, stride %lld)", fmt, n, vocab,
                 stride);
        return -1;
    }
    if (n == 0) return 0;
    if (!d_pick || !d_logits || !s->u) {
        DSV4_ERR("sample: a missing buffer");
        return -1;
    }
    const SamplePlan p = sample_plan(n, vocab);
    if (!d_scratch || ((uintptr_t)d_scratch & 15) || scratch_bytes < p.bytes) {
        DSV4_ERR("sample: %zu bytes of workspace at %p; the call needs %zu, 16-byte aligned",
                 scratch_bytes, d_scratch, p.bytes);
        return -1;
    }
    char *base = (char *)d_scratch;
    SampleJob a{d_logits, stride, n, vocab, p.ns, p.nc, p.sh, *s, (u64 *)(base + p.mass),
                (uint32_t *)(base + p.count), (double *)(base + p.top), (float *)(base + p.cmax),
                d_kept, d_prob};
    hipStream_t st = (hipStream_t)stream;
    return fmt == DSV4_WF32 ? sample_launch<float>(a, d_pick, st)
                            : sample_launch<uint16_t>(a, d_pick, st);
}
