/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_sample.hip - a token of each row of logits by temperature, top-k, top-p
 * and min-p from a given random number, on gfx950.
 *
 * With z = x log2(e) / T a token weighs 2^z. All limits cut the order of
 * descending logits after some token, and the pick is where a running sum of that
 * order passes u times the sum of what is left; so the rows need no sort but the
 * place of a few sums. The order is cut into bins by floor(32 z): a token's weight
 * is known to 2^(1/32) by its bin, and the sums over bins say which bin a limit or
 * the pick falls into. Only those bins' tokens are put in order.
 *
 * Sums are of whole numbers, so that they do not depend on their order: of a bin the
 * count and the sum of 2^(r/32) - 1, r the rest of 32 z, to 2^-42; over bins
 * 2^(z - E) 2^sh, E an integer that no z of the row passes. The bins lie at the
 * same z for all slices of a row. z and the weights are in 64 bits: a pick that is
 * wrong by a rounding is another token.
 *
 * Two launches: slices of 8192 tokens, and a workgroup for each row. Bound: the
 * vector unit, busy 92 %, and one LDS add a token where bins are made (256 rows of 129280
 * 50 us); where they are not a slice's loads, as none are in flight while it is reduced
 * (23 us, 2.9 TB/s, the waves wait 72 % of it); and for few rows the pick's chain of scans
 * (13 us for 64 rows of top-k 200, 21 with bins) and its code's first fetch.
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

#include <type_traits>

namespace {

#include "dsv4_rows_io.h"

typedef unsigned long long u64;

constexpr int SM_THREADS = 512;
constexpr int SM_EACH = 16;                       /* tokens of a thread      */
constexpr int SM_SLICE = SM_THREADS * SM_EACH;
constexpr int SM_BINS = 1024;                     /* 32 octaves, the rest in the last */
constexpr int SM_CHUNK = 64;                      /* tokens with one maximum */
/* A bin of a slice in one word: the count from bit 50 on (8192 at most), and below
 * it the sum of (2^(r/32) - 1) 2^42, which is under 8192 x 0.0219 x 2^42 < 2^50. */
constexpr int SM_PART = 42, SM_COUNT = 50;
static_assert(SM_SLICE <= 8192, "a bin's word");
constexpr int SP_THREADS = 1024;                  /* of a row's pick         */
constexpr int SP_WAVES = SP_THREADS / 64;
constexpr int SP_LIST = SP_THREADS;               /* tokens put in order     */
constexpr int SP_QUEUE = 2 * SP_LIST;              /* and looked through      */
constexpr int SP_CHUNKS = 4096;                   /* chunks looked over at once */
constexpr int SP_K = 512;                         /* a short top-k, for which no bins are made */
constexpr int SP_DIRECT = 128;                    /* tokens compared with all others */
constexpr float SP_FLOOR = 0.0078125f;             /* a min_p for which none are made */
static_assert(SP_THREADS == SM_BINS, "a bin a thread");

struct SmTop {
    double q;                                     /* 32 z of the first bin   */
    u64 tail;                                     /* the last bin's sum      */
    uint32_t tail_n, pad;
};

struct SampleJob {
    const void *x;
    long long stride;
    int row0, vocab, ns, nc, sh;                  /* first row; slices, chunks of one */
    dsv4_gpu_sampling r;
    u64 *bins;                                    /* [n][ns][bins]           */
    SmTop *top;                                   /* [n][ns]                 */
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

/* 2^t, t <= 0; 0 below 2^-1000, which is under every min_p over 0. */
__device__ __forceinline__ double sm_exp2(double t)
{
    if (!(t > -1000.0)) return 0.0;
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

/* (2^(r/32) - 1) 2^42 of a token, r in [0, 1), as a whole number: the polynomial of
 * degree 5 through its values at Chebyshev's points, 2^-53 off at the most (its
 * constant term is 3e-4 of a unit), added to 2^52, which rounds it. sm_bin_bits: still
 * with 2^52's exponent above bit 51. */
__device__ __forceinline__ u64 sm_bin_bits(double r)
{
    static_assert(SM_PART == 42, "the coefficients' unit");
    double p = 176.66942619745828;
    p = fma(p, r, 40339.21157864393);
    p = fma(p, r, 7449636.473277472);
    p = fma(p, r, 1031764990.7605293);
    p = fma(p, r, 95265423098.24869);
    return (u64)__double_as_longlong(fma(p, r, 4503599627370496.0));
}
__device__ __forceinline__ u64 sm_bin_word(double z, double q)
{
    return sm_bin_bits(fma(z, 32.0, -q)) & ((1ull << 52) - 1);
}

/* The sum of n tokens of a bin, `edge` the weight at its lower edge. Equal tokens sum
 * to a multiple of a whole number, so that limits and picks that fall between two of
 * them do so exactly. */
__device__ __forceinline__ u64 sm_bin_sum(double edge, uint32_t n, u64 part)
{
    constexpr double ONE = 1.0 / (1ull << SM_PART);
    /* the quotient, which is below 2^37, to 2^-10 */
    const double r = __builtin_amdgcn_rcp((double)n);
    const double each = __builtin_rint((double)part * fma(fma(-(double)n, r, 1.0), r, r));
    if (n && (u64)each * n == part) return (u64)__builtin_rint(edge * (1.0 + each * ONE)) * n;
    return (u64)__builtin_rint(edge * ((double)n + (double)part * ONE));
}

/* A top-k so short that the chunks with the k largest maxima, which have the k largest
 * tokens, have hardly more that are as large (256 of 2020 chunks: 274 tokens). One row of
 * 129280 and 64 take 12 and 18 us so for top-k 8 and 21 and 27 for 512, with bins 23 and
 * 32, 31 and 40; for 800 there may be more than the list takes, 75 and 102 us for 35 and
 * 46. Where fewer than k chunks have a token, as under a mask, there is no k-th maximum
 * and all tokens are looked at. */
__device__ __forceinline__ bool sm_short(const SampleJob &a, int top_k)
{
    return top_k > 0 && top_k <= SP_K && 2 * top_k <= a.nc && a.nc <= SP_CHUNKS;
}

/* A row whose only other limit is min_p: what is under it has no part in any sum, so
 * that its tokens are all that is looked at, if they fit the list. 1 to 256 rows of 129280
 * take 11 to 36 us so and 23 to 56 with bins; with 11000 tokens over it, which make the
 * row's workgroup count the bins after all, 71 to 198 and 47 to 169. */
__device__ __forceinline__ float sm_floor(const SampleJob &a, int row)
{
    const float v = a.r.min_p ? a.r.min_p[row] : 0.0f;
    return v > 0.0f ? fminf(v, 1.0f) : 0.0f;      /* NaN: no such rule       */
}
__device__ __forceinline__ bool sm_above(const SampleJob &a, int row, float floor_)
{
    return floor_ >= SP_FLOOR && a.nc <= SP_CHUNKS && !(a.r.top_p && a.r.top_p[row] < 1.0f);
}
__device__ __forceinline__ bool sm_brief(const SampleJob &a, int row)
{
    return (a.r.top_k && sm_short(a, a.r.top_k[row])) || sm_above(a, row, sm_floor(a, row));
}

/* A slice of a row: the maxima of its chunks, and its bins. */
template <class T>
__global__ void __launch_bounds__(SM_THREADS) k_sample_slices(SampleJob a)
{
    __shared__ __attribute__((aligned(16))) u64 bins[SM_BINS];
    __shared__ float wtop[SM_THREADS / 64];
    __shared__ u64 tail;
    __shared__ uint32_t tail_n;
    const int tid = threadIdx.x;
    const int of = blockIdx.x / a.ns, slice = blockIdx.x - of * a.ns, row = a.row0 + of;
    const int v0 = slice * SM_SLICE;
    const T *x = (const T *)a.x + (size_t)row * a.stride + v0;
    const int lim = min(SM_SLICE, a.vocab - v0);
    constexpr int W = 4;                          /* tokens of a load: 8 of bf16 took 28 us for 23 */
    float v[SM_EACH];
#pragma unroll
    for (int p = 0; p < SM_EACH / W; p++) {
        const int c = (p * SM_THREADS + tid) * W;
        if (lim == SM_SLICE) {
            io_load<T, W>(x + c, v + W * p);
        } else {
#pragma unroll
            for (int k = 0; k < W; k++) {
                v[W * p + k] = -INFINITY;
                if (c + k < lim) io_load<T, 1>(x + c + k, v + W * p + k);
            }
        }
    }
    const float temp = sm_temperature(a, row);
    const bool brief = sm_brief(a, row);
    float top = -INFINITY;
#pragma unroll
    for (int p = 0; p < SM_EACH / W; p++) {
        /* (NaN: fmaxf takes the other) */
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < W; k++) m = fmaxf(m, v[W * p + k]);
        m = fmaxf(m, dpp_f<DPP_QUAD_XOR1, 0xF>(m));
        m = fmaxf(m, dpp_f<DPP_QUAD_XOR2, 0xF>(m));
        m = fmaxf(m, dpp_f<DPP_ROW_HMIRROR, 0xF>(m));
        if (W == 4) m = fmaxf(m, dpp_f<DPP_ROW_MIRROR, 0xF>(m));
        constexpr int LANES = SM_CHUNK / W;
        const int chunk = (v0 + p * SM_THREADS * W) / SM_CHUNK + tid / LANES;
        if ((tid & (LANES - 1)) == 0 && chunk < a.nc) a.cmax[(size_t)row * a.nc + chunk] = m;
        top = fmaxf(top, m);
    }
    /* the first is picked, or one of the first few */
    if (!(temp > 0.0f) || brief) return;

    for (int i = tid; i < SM_BINS; i += SM_THREADS) bins[i] = 0;
    if (tid == 0) {
        tail = 0;
        tail_n = 0;
    }
    top = wave_max(top);
    if ((tid & 63) == 0) wtop[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SM_THREADS / 64; k++) top = fmaxf(top, wtop[k]);
    const size_t at = (size_t)row * a.ns + slice;
    const SmScale sc{1.4426950408889634 / (double)temp, top == INFINITY};
    const double first = sm_q(sc.z(top)), e = sm_e(first);
    /* of the last bin, whose weights of at most 2^-32 need 2^-14 of their own */
    uint32_t rest = 0, rest_n = 0;
    const float unit = __uint_as_float((uint32_t)(127 + a.sh) << 23);
    if (sc.inf) {
#pragma unroll
        for (int k = 0; k < SM_EACH; k++) {
            if (v[k] == INFINITY) atomicAdd(&bins[0], 1ull << SM_COUNT);
            else rest_n += v[k] > -INFINITY;
        }
    } else if (top > -INFINITY) {
        const double c32 = sc.c * 32.0;           /* exact, and so is y - q   */
#pragma unroll
        for (int k = 0; k < SM_EACH; k++) {
            const double y = (double)v[k] * c32, q = floor(y), d = first - q;
            if (d < SM_BINS - 1) {
                /* 2^52's exponent becomes the count */
                constexpr uint32_t ONE = (1u << (SM_COUNT - 32)) - (0x433u << 20);
                const u64 bits = sm_bin_bits(y - q);
                atomicAdd(&bins[(int)d], (u64)((uint32_t)(bits >> 32) + ONE) << 32 | (uint32_t)bits);
            } else if (v[k] > -INFINITY) {
                rest += (uint32_t)(__builtin_amdgcn_exp2f((float)(y * (1.0 / 32.0) - e)) * unit);
                rest_n++;
            }
        }
    }
    if (rest_n) {
        atomicAdd(&tail, (u64)rest);
        atomicAdd(&tail_n, rest_n);
    }
    __syncthreads();
    for (int i = tid; i < SM_BINS / 2; i += SM_THREADS)
        *(u32x4 *)(a.bins + at * SM_BINS + 2 * i) = *(const u32x4 *)(bins + 2 * i);
    if (tid == 0)
        a.top[at] = SmTop{top == -INFINITY ? -INFINITY : sc.inf ? INFINITY : first, tail, tail_n, 0};
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

/* Inclusive sums over a wave, by moves within the vector unit. */
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t sm_dpp(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 sm_dpp(u64 v)
{
    return (u64)sm_dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | sm_dpp<CTRL, ROWS>((uint32_t)v);
}
template <class V>
__device__ __forceinline__ V sm_wave_scan(V v)
{
    v += sm_dpp<0x111, 0xF>(v);                   /* row_shr:1, 2, 4, 8      */
    v += sm_dpp<0x112, 0xF>(v);
    v += sm_dpp<0x114, 0xF>(v);
    v += sm_dpp<0x118, 0xF>(v);
    v += sm_dpp<DPP_ROW_BCAST15, 0xA>(v);
    v += sm_dpp<DPP_ROW_BCAST31, 0xC>(v);
    return v;
}

/* The largest of all lanes' v; of their pairs. */
__device__ __forceinline__ uint32_t sm_wave_top(uint32_t v)
{
    v = max(v, sm_dpp<DPP_QUAD_XOR1, 0xF>(v));
    v = max(v, sm_dpp<DPP_QUAD_XOR2, 0xF>(v));
    v = max(v, sm_dpp<DPP_ROW_HMIRROR, 0xF>(v));
    v = max(v, sm_dpp<DPP_ROW_MIRROR, 0xF>(v));
    v = max(v, sm_dpp<DPP_ROW_BCAST15, 0xA>(v));
    v = max(v, sm_dpp<DPP_ROW_BCAST31, 0xC>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ u64 sm_wave_top(u64 v)
{
    const uint32_t h = sm_wave_top((uint32_t)(v >> 32));
    return (u64)h << 32 | sm_wave_top((uint32_t)(v >> 32) == h ? (uint32_t)v : 0u);
}

/* The bins of top-k, top-p (between two), min-p, the last cut (at most) and the pick. */
struct SmWhere {
    int kb, pb0, pb1, mb, c1, ub0, ub1, need_k, whole;
};

/* The first of n <= 1024 places that pred holds for, n if none does; it holds for all
 * behind the first. Each wave looks for itself: 64 places at once, then the 16 before
 * the first of them that has it. */
template <class F>
__device__ __forceinline__ int sm_first(int n, F pred)
{
    const int lane = threadIdx.x & 63;
    const int end = min(16 * lane + 15, n - 1);
    const u64 far = __ballot(n > 0 && pred(max(end, 0)));
    if (!far) return n;
    const int at = min(16 * (int)__builtin_ctzll(far) + (lane & 15), n - 1);
    const u64 near = __ballot(pred(at));
    return __shfl(at, (int)__builtin_ctzll(near), 64);
}

/* The workgroup of a row. Its code is kept short, as all of it is fetched for a few
 * microseconds' run: loops stay loops but where loads have to be out together. */
template <class T>
struct SmRow {
    struct Lds {
        union {
            __attribute__((aligned(16))) u64 queue[SP_QUEUE];  /* tokens that may be listed */
            struct {
                u64 mass[SP_THREADS], best[SP_THREADS];   /* a split of a key range */
            };
        };
        __attribute__((aligned(16))) u64 key[SP_LIST];    /* tokens in order */
        __attribute__((aligned(16))) u64 through[SP_LIST];  /* and the sums through them */
        u64 sum[SM_BINS];                         /* through a bin           */
        uint32_t n[SM_BINS];
        int off[SM_BINS];                         /* a bin's place in the list, or -1 */
        uint32_t cur[SM_BINS];                    /* a bin's tokens so far   */
        unsigned short chunk[SP_CHUNKS];          /* chunks to read          */
        u64 part[SP_WAVES];
        uint32_t npart[SP_WAVES];
        SmPlace hit;
        SmWhere where;
        u64 tail;                                 /* the last bin's sum      */
        uint32_t tail_n;
        int len, chunks;                          /* tokens queued; to read  */
    };
    const SampleJob &a;
    Lds &s;
    const T *x;
    const float *cmax;
    SmScale sc;
    double first, e;
    double width;                                 /* of a bin, in logits     */
    float cm[SP_CHUNKS / SP_THREADS];             /* this thread's of the first chunks */

    /* Inclusive sums over the threads. */
    __device__ __forceinline__ void scan(u64 &m, uint32_t &n)
    {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        m = sm_wave_scan(m);
        n = sm_wave_scan(n);
        __syncthreads();
        if (lane == 63) {
            s.part[w] = m;
            s.npart[w] = n;
        }
        __syncthreads();
        /* lane k's sum of the waves 0 .. k, of which this wave takes those before it */
        const u64 mw = sm_wave_scan(lane < SP_WAVES ? s.part[lane & (SP_WAVES - 1)] : 0);
        const uint32_t nw = sm_wave_scan(lane < SP_WAVES ? s.npart[lane & (SP_WAVES - 1)] : 0u);
        if (w) {
            m += __shfl(mw, w - 1, 64);
            n += __shfl(nw, w - 1, 64);
        }
    }

    __device__ __forceinline__ uint32_t n_before(int bin) const { return bin ? s.n[bin - 1] : 0; }
    __device__ __forceinline__ u64 sum_before(int bin) const { return bin ? s.sum[bin - 1] : 0; }
    __device__ __forceinline__ int bin_of(float v) const { return sm_bin(first, sm_q(sc.z(v))); }
    /* The first bin through which the sum is; the last, where roundings pass it. */
    __device__ __forceinline__ int sum_bin(u64 need) const
    {
        return min(sm_first(SM_BINS, [&](int i) { return s.sum[i] >= need; }), SM_BINS - 1);
    }

    /* The weight at the lower edge of the bin of 32 z = q, and of a token in it. */
    __device__ __forceinline__ double edge(double q) const
    {
        return sm_exp2(q * (1.0 / 32.0) - e) * __hiloint2double((1023 + a.sh) << 20, 0);
    }
    __device__ __forceinline__ u64 weight(double z) const
    {
        const double q = sm_q(z);
        return first - q < SM_BINS - 1 ? sm_bin_sum(edge(q), 1, sm_bin_word(z, q))
                                       : sm_weight(z - e, a.sh);
    }

    /* Logits between which all tokens of bins [b0, b1] lie, with a margin for the roundings
     * of z and of this, in 64 bits: a width that f32 holds with few bits, as of a
     * temperature under 2^-120, would put the bins beside their tokens. */
    __device__ __forceinline__ void range_of(int b0, int b1, float *lo, float *hi) const
    {
        const double l = (first - b1) * width, h = (first - b0 + 1.0) * width;
        *lo = (float)(l - fabs(l) * 4e-6);
        *hi = (float)(h + fabs(h) * 4e-6);
        if (sc.inf || b1 == SM_BINS - 1 || !(*lo > -3.4028235e38f)) *lo = -3.4028235e38f;
        if (sc.inf || b0 == 0 || !(*hi < INFINITY)) *hi = INFINITY;
    }

    /* f(G, x [G][4], token [G]) for the row's chunks whose largest is lo or more, G times four
     * tokens of a lane at once (-infinity where there are none). The whole workgroup; 16
     * lanes a chunk, so that a load takes 1 KB of four chunks. */
    template <int G, class F>
    __device__ __forceinline__ void each_of_row(float lo, F f)
    {
        const int tid = threadIdx.x;
#pragma unroll 1
        for (int c0 = 0; c0 < a.nc; c0 += SP_CHUNKS) {
            __syncthreads();
            if (tid == 0) s.chunks = 0;
            __syncthreads();
#pragma unroll
            for (int k = tid; k < SP_CHUNKS; k += SP_THREADS) {
                const float top = c0 ? c0 + k < a.nc ? cmax[c0 + k] : -INFINITY : cm[k / SP_THREADS];
                const bool want = top >= lo;
                const u64 who = __ballot(want);
                int at = 0;
                if ((tid & 63) == 0 && who) at = atomicAdd(&s.chunks, (int)__popcll(who));
                at = __builtin_amdgcn_readfirstlane(at) +
                     (int)__popcll(who & ((1ull << (tid & 63)) - 1));
                if (want) s.chunk[at] = (unsigned short)k;
            }
            __syncthreads();
            const int n = s.chunks;
            if (n <= SP_THREADS / 16) chunks<1>(c0, n, f);
            else chunks<G>(c0, n, f);
        }
        __syncthreads();
    }

    /* The listed chunks, 16 lanes each, G of them in flight. */
    template <int G, class F>
    __device__ __forceinline__ void chunks(int c0, int n, F f)
    {
        constexpr int EACH = SP_THREADS / 16;
        const int tid = threadIdx.x, whole = a.vocab / SM_CHUNK;
#pragma unroll 1
        for (int i0 = tid / 16; i0 < n; i0 += G * EACH) {
            float v[G][4];
            int t[G];
#pragma unroll
            for (int u = 0; u < G; u++) {
                const int c = i0 + u * EACH < n ? c0 + s.chunk[i0 + u * EACH] : INT32_MAX;
                t[u] = c * SM_CHUNK + 4 * (tid & 15);
#pragma unroll
                for (int k = 0; k < 4; k++) v[u][k] = -INFINITY;
                if (c < whole) {
                    io_load<T, 4>(x + t[u], v[u]);
                } else if (c == whole) {          /* the row's last, not whole */
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (t[u] + k < a.vocab) io_load<T, 1>(x + t[u] + k, v[u] + k);
                }
            }
            f(std::integral_constant<int, G>(), v, t);
        }
    }

    /* Queue the tokens from lo to hi; how many, over SP_QUEUE: not all. One add for all
     * of a wave's. */
    __device__ __forceinline__ int queue(float lo, float hi)
    {
        const int lane = threadIdx.x & 63;
        if (threadIdx.x == 0) s.len = 0;
        each_of_row<2>(lo, [&](auto groups, float (*v)[4], const int *t) {
            constexpr int G = decltype(groups)::value;
            u64 hit[G][4];
            int many = 0;
#pragma unroll
            for (int u = 0; u < G; u++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    hit[u][k] = __ballot(__builtin_amdgcn_fmed3f(v[u][k], lo, hi) == v[u][k]);
                    many += (int)__popcll(hit[u][k]);
                }
            if (!many) return;
            int at = 0;
            if (lane == 0) at = atomicAdd(&s.len, many);
            at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
            for (int u = 0; u < G; u++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (!hit[u][k]) continue;
                    const int i = at + (int)__popcll(hit[u][k] & ((1ull << lane) - 1));
                    if (hit[u][k] >> lane & 1 && i < SP_QUEUE) s.queue[i] = am_key(v[u][k], t[u] + k);
                    at += (int)__popcll(hit[u][k]);
                }
        });
        return s.len;
    }
    /* And those from lo2 to hi2, lo <= lo2. An add for each: with all of a wave's counted
     * first a flat row's call takes 40 us and not 37. */
    __device__ __forceinline__ int queue(float lo, float hi, float lo2, float hi2)
    {
        if (threadIdx.x == 0) s.len = 0;
        each_of_row<4>(lo, [&](auto groups, float (*v)[4], const int *t) {
#pragma unroll
            for (int u = 0; u < decltype(groups)::value; u++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (__builtin_amdgcn_fmed3f(v[u][k], lo, hi) == v[u][k] ||
                        __builtin_amdgcn_fmed3f(v[u][k], lo2, hi2) == v[u][k]) {
                        const int at = atomicAdd(&s.len, 1);
                        if (at < SP_QUEUE) s.queue[at] = am_key(v[u][k], t[u] + k);
                    }
        });
        return s.len;
    }

    /* Of SP_THREADS parts of the range of the keys of threads 0 .. n - 1, which has thread
     * tid's, the largest first. */
    __device__ __forceinline__ int part_of_range(int n, u64 key)
    {
        const int tid = threadIdx.x;
        uint32_t k0 = tid < n ? (uint32_t)(key >> 32) : ~0u, k1 = tid < n ? k0 : 0;
        k0 = ~sm_wave_top(~k0);
        k1 = sm_wave_top(k1);
        __syncthreads();
        if ((tid & 63) == 0) s.part[tid >> 6] = (u64)k0 << 32 | k1;
        __syncthreads();
        const u64 v = s.part[tid & (SP_WAVES - 1)];
        k0 = ~sm_wave_top(~(uint32_t)(v >> 32));
        k1 = sm_wave_top((uint32_t)v);
        /* (a range that is not finite, or 0: all in one, as NaN becomes 0) */
        const float top = sm_value((u64)k1 << 32), by = (SP_THREADS - 1) / (top - sm_value((u64)k0 << 32));
        return (int)fminf(fmaxf((top - sm_value(key)) * by, 0.0f), SP_THREADS - 1.0f);
    }

    /* The place of thread tid's key among those of threads 0 .. n - 1, the largest first.
     * All keys read by all threads are n^2 reads of LDS; over SP_DIRECT of them each is
     * compared with those of its part d only, of SP_THREADS in the same order. One row's
     * call takes 15.7 us for 100 so and 16.7 by parts, for 200 18.7 and 17.8, for 512 29 and
     * 21. */
    __device__ __forceinline__ int order(int n, u64 key, int d)
    {
        const int tid = threadIdx.x;
        int i0 = 0, i1 = n, at = tid;
        if (n > SP_DIRECT) {
            s.cur[tid] = 0;
            __syncthreads();
            if (tid < n) at = (int)atomicAdd(&s.cur[d], 1u);
            __syncthreads();
            u64 none = 0;
            uint32_t e = s.cur[tid];
            scan(none, e);
            s.cur[tid] = e;
            __syncthreads();
            if (tid < n) {
                i0 = d ? (int)s.cur[d - 1] : 0;
                i1 = (int)s.cur[d];
                at += i0;
            }
        }
        if (tid < n) s.through[at] = key;
        __syncthreads();
        int place = i0;
        if (tid < n) {
            int i = i0;
            if (i & 1) place += s.through[i++] > key;
#pragma unroll 4
            for (; i + 2 <= i1; i += 2) {
                const ulonglong2 k = *reinterpret_cast<const ulonglong2 *>(s.through + i);
                place += (k.x > key) + (k.y > key);
            }
            if (i < i1) place += s.through[i] > key;
        }
        __syncthreads();
        return place;
    }

    /* Put the tokens of the bins that have a place (s.off), of b0 to b1 or b2 to b3, into the
     * list, in order, n in all; false where those between are too many. */
    __device__ __forceinline__ bool list(int b0, int b1, int b2, int b3, int n)
    {
        const int tid = threadIdx.x;
        float lo, hi, lo2, hi2;
        range_of(b0, b1, &lo, &hi);
        range_of(b2, b3, &lo2, &hi2);
        s.cur[tid] = 0;
        if (lo2 < lo) {
            float t = lo;
            lo = lo2;
            lo2 = t;
            t = hi;
            hi = hi2;
            hi2 = t;
        }
        const int len = hi2 <= hi ? queue(lo, hi) : queue(lo, hi, lo2, hi2);
        if (len > SP_QUEUE) return false;
#pragma unroll 1
        for (int i = tid; i < len; i += SP_THREADS) {
            const u64 key = s.queue[i];
            const int bin = bin_of(sm_value(key)), off = s.off[bin];
            if (off < 0) continue;
            const int at = off + (int)atomicAdd(&s.cur[bin], 1u);
            if (at < n) s.key[at] = key;          /* (the counts say that it is) */
        }
        __syncthreads();
        const u64 key = tid < n ? s.key[tid] : 0;
        int d = 0;
        if (tid < n) {                            /* a part for each of a bin's tokens */
            const double z = sc.z(sm_value(key)), q = sm_q(z);
            const int bin = sm_bin(first, q), many = (int)(s.n[bin] - n_before(bin));
            const float r = bin == SM_BINS - 1 ? 0.0f : 1.0f - (float)fma(z, 32.0, -q);
            d = max(0, s.off[bin] + max(0, min((int)(r * (float)many), many - 1)));
        }
        __syncthreads();
        const int at = order(n, key, d);
        if (tid < n) {
            s.key[at] = key;
            s.queue[at] = weight(sc.z(sm_value(key)));
        }
        __syncthreads();
        u64 m = tid < n ? s.queue[tid] : 0;
        const u64 w = m;
        uint32_t k = 0;
        scan(m, k);
        s.queue[SP_LIST + tid] = m - w;           /* before it in the list   */
        __syncthreads();
        if (tid < n) {
            const int bin = bin_of(sm_value(s.key[tid]));
            s.through[tid] = sum_before(bin) + m - s.queue[SP_LIST + s.off[bin]];
        }
        __syncthreads();
        return true;
    }
};

template <class T>
__global__ void __launch_bounds__(SP_THREADS) k_sample_pick(SampleJob a, int *d_pick)
{
    using Row = SmRow<T>;
    __shared__ typename Row::Lds s;
    constexpr int LAST = SM_BINS - 1;
    const int tid = threadIdx.x, lane = tid & 63, row = a.row0 + blockIdx.x;
    const float temp = sm_temperature(a, row);
    const int top_k = a.r.top_k ? a.r.top_k[row] : 0;
    const float p = a.r.top_p ? a.r.top_p[row] : 1.0f;
    const float floor_ = sm_floor(a, row);
    const bool few = sm_short(a, top_k), brief = few || sm_above(a, row, floor_);
    const float u = a.r.u[row];
    Row r{a, s, (const T *)a.x + (size_t)row * a.stride, a.cmax + (size_t)row * a.nc,
          SmScale{0.0, false}, 0.0, 0.0, (double)temp * 0.02166084939249829, {}};
    auto done = [&](int pick, float prob, int kept) {
        d_pick[row] = pick;
        if (a.prob) a.prob[row] = prob;
        if (a.kept) a.kept[row] = kept;
    };

    /* the largest logit, and the first chunk that has it; the slices' first bins on
     * their way meanwhile */
    constexpr int G = 16;
    const SmTop *tops = a.top + (size_t)row * a.ns;
    const u64 *bins = a.bins + (size_t)row * a.ns * SM_BINS;
    const bool sampled = temp > 0.0f;
    SmTop mine{-INFINITY, 0, 0, 0};
    if (sampled && !brief && (lane & (G - 1)) < a.ns) mine = tops[lane & (G - 1)];
    u64 most = 0;
#pragma unroll
    for (int k = 0; k < SP_CHUNKS / SP_THREADS; k++) {
        const int c = tid + k * SP_THREADS;
        r.cm[k] = c < a.nc ? r.cmax[c] : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < SP_CHUNKS / SP_THREADS; k++) {
        const u64 key = r.cm[k] > -INFINITY ? am_key(r.cm[k], tid + k * SP_THREADS) : 0;
        most = key > most ? key : most;
    }
#pragma unroll 1
    for (int c = SP_CHUNKS + tid; c < a.nc; c += SP_THREADS) {
        const u64 key = r.cmax[c] > -INFINITY ? am_key(r.cmax[c], c) : 0;
        most = key > most ? key : most;
    }
    /* and the least of the chunks with tokens */
    uint32_t least = ~0u;
#pragma unroll
    for (int k = 0; k < SP_CHUNKS / SP_THREADS; k++)
        if (r.cm[k] > -INFINITY) least = min(least, (uint32_t)(am_key(r.cm[k], 0) >> 32));
    most = sm_wave_top(most);
    least = ~sm_wave_top(~least);
    if (lane == 0) {
        s.part[tid >> 6] = most;
        s.npart[tid >> 6] = least;
    }
    if (tid == 0) {
        s.tail = 0;
        s.tail_n = 0;
    }
    __syncthreads();
    most = sm_wave_top(s.part[lane & (SP_WAVES - 1)]);
    if (most == 0) {
        if (tid == 0) done(-1, 0.0f, 0);
        return;
    }
    if (!sampled) {
        if (tid >= 64) return;
        const int t = sm_token(most) * SM_CHUNK + lane;
        float v = -INFINITY;
        if (t < a.vocab) io_load<T, 1>(r.x + t, &v);
        const u64 k = sm_wave_top(v > -INFINITY ? am_key(v, t) : 0);
        if (tid == 0) done(sm_token(k), 1.0f, 1);
        return;
    }

    /* ---- the slices' bins as the row's ---- */
    const float largest = sm_value(most);
    r.sc = SmScale{1.4426950408889634 / (double)temp, largest == INFINITY};
    const double zmost = r.sc.z(largest);
    r.first = sm_q(zmost);
    r.e = sm_e(r.first);
    const double edge = r.edge(r.first - tid), unit = __hiloint2double((1023 + a.sh) << 20, 0);
    auto part_of = [&](u64 total) {               /* top-p's sum             */
        const u64 v = p > 0.0f ? sm_part(p, total, true) : 0;
        return v > 1 ? v : 1;
    };
    auto place_of = [&](u64 total) {              /* the pick's              */
        u64 t = total - 1;
        if (!(u >= 1.0f)) t = min(t, u > 0.0f ? sm_part(u, total, false) : 0);
        return t + 1;
    };
    auto under = [&](u64 key) {                   /* min_p                   */
        return sm_exp2(r.sc.z(sm_value(key)) - zmost) < (double)floor_;
    };
    const bool by_p = p < 1.0f, by_floor = floor_ > 0.0f;
    auto each = [](auto f) {                      /* f(x, token) for a batch of them */
        return [f](auto groups, float (*v)[4], const int *t) {
#pragma unroll
            for (int u = 0; u < decltype(groups)::value; u++)
#pragma unroll
                for (int k = 0; k < 4; k++) f(v[u][k], t[u] + k);
        };
    };

    /* ---- a short top-k: the tokens as large as the k-th largest chunk, in order, or all
     *      where fewer chunks have any; or a min_p alone: those that it may leave ---- */
    bool fits = brief;
    float low = INFINITY;
    if (few) {
        /* that chunk's maximum, or a little less: the range of keys split by 1024 */
        uint32_t key0 = ~sm_wave_top(~s.npart[lane & (SP_WAVES - 1)]), key1 = (uint32_t)(most >> 32);
        int n0 = 0;
#pragma unroll 1
        for (;;) {
            const int sh = max(0, 22 - (int)__clz((int)((key1 - key0) | 1)));
            __syncthreads();
            s.cur[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < SP_CHUNKS / SP_THREADS; k++) {
                const uint32_t key = (uint32_t)(am_key(r.cm[k], 0) >> 32);
                if (r.cm[k] > -INFINITY && key >= key0 && key <= key1)
                    atomicAdd(&s.cur[(key1 - key) >> sh], 1u);
            }
            __syncthreads();
            u64 none = 0;
            uint32_t c = s.cur[tid];
            r.scan(none, c);
            s.cur[tid] = n0 + c;
            __syncthreads();
            const int d = sm_first(SP_THREADS, [&](int i) { return s.cur[i] >= (uint32_t)top_k; });
            if (d == SP_THREADS) {                /* fewer chunks with tokens: all of those */
                key0 = (uint32_t)(am_key(-3.4028235e38f, 0) >> 32);
                break;
            }
            const uint32_t end = key1 - (((uint32_t)d << sh) | ((1u << sh) - 1));
            n0 = d ? (int)s.cur[d - 1] : n0;
            const int through = (int)s.cur[d];
            key1 -= (uint32_t)d << sh;
            key0 = end > key0 && end <= key1 ? end : key0;
            if (sh == 0 || through <= top_k + top_k / 8 + 8) break;
        }
        low = sm_value((u64)key0 << 32);
    } else if (brief) {
        /* with a margin for the logarithm and the quotient; every chunk above has a token */
        if (!r.sc.inf) {
            low = (float)((zmost + (double)__builtin_amdgcn_logf(floor_) - 1e-5) / r.sc.c);
            low = fmaxf(low - fabsf(low) * 1e-6f, -3.4028235e38f);
        }
        int n = 0;
#pragma unroll
        for (int k = 0; k < SP_CHUNKS / SP_THREADS; k++) n += (int)__popcll(__ballot(r.cm[k] >= low));
        __syncthreads();
        if (lane == 0) s.npart[tid >> 6] = (uint32_t)n;
        __syncthreads();
        fits = sm_wave_scan(lane < SP_WAVES ? s.npart[lane & (SP_WAVES - 1)] : 0u) <= SP_LIST;
        fits = __all(fits);
    }
    if (fits) {
        const int len = r.queue(low, INFINITY);
        if (len <= SP_LIST) {
            const u64 key = tid < len ? s.queue[tid] : 0;
            const int at = r.order(len, key, len > SP_DIRECT ? r.part_of_range(len, key) : 0);
            if (tid < len) s.key[at] = key;
            __syncthreads();
            const int end = top_k > 0 ? min(top_k, len) : len;
            u64 m = tid < end ? sm_weight(r.sc.z(sm_value(s.key[tid])) - r.e, a.sh) : 0;
            uint32_t none = 0;
            r.scan(m, none);
            s.through[tid] = m;
            __syncthreads();
            if (tid >= 64) return;
            int kept = end;
            if (by_p)
                kept = min(kept, sm_first(end, [&, need = part_of(s.through[end - 1])](int i) {
                                     return s.through[i] >= need;
                                 }) + 1);
            if (by_floor)
                kept = min(kept, max(1, sm_first(end, [&](int i) { return under(s.key[i]); })));
            const u64 total = s.through[kept - 1], need = place_of(total);
            const int i = min(sm_first(kept, [&](int j) { return s.through[j] >= need; }), kept - 1);
            if (tid == 0) {
                const double v = sm_exp2(r.sc.z(sm_value(s.key[i])) - r.e) *
                                 __hiloint2double((1023 + a.sh) << 20, 0);
                done(sm_token(s.key[i]), (float)(v / (double)total), kept);
            }
            return;
        }
    }

    /* a bin a thread. A slice's bins start d behind the row's: bin `tid` is its tid - d, and
     * threads 0 .. d - 1 have its last d, which are behind the row's and join the last one */
    const double edge_rest = r.edge(r.first - LAST - tid);
    uint32_t n = 0, rest_n = 0;
    u64 part = 0, rest = 0;
#pragma unroll 1
    for (int k0 = 0; !brief && k0 < a.ns; k0 += G) {
        if (k0) {
            mine = SmTop{-INFINITY, 0, 0, 0};
            if (k0 + (lane & (G - 1)) < a.ns) mine = tops[k0 + (lane & (G - 1))];
        }
        const bool same = mine.q == (r.sc.inf ? INFINITY : r.first);
        const int mine_d = same ? 0 : r.sc.inf ? LAST : sm_bin(r.first, mine.q);
        /* how much less a slice's weights are where it starts more bins behind */
        const double mine_far =
            r.sc.inf ? 0.0 : sm_exp2(fmin((mine.q - r.first + mine_d) * (1.0 / 32.0), 0.0));
        u64 word[G];
#pragma unroll
        for (int k = 0; k < G; k++) {
            const int d = __builtin_amdgcn_readlane(mine_d, k);
            const int j = tid < d ? LAST - d + tid : tid - d;
            word[k] = k0 + k < a.ns && tid < LAST ? bins[(size_t)(k0 + k) * SM_BINS + j] : 0;
        }
#pragma unroll
        for (int k = 0; k < G; k++) {
            const int d = __builtin_amdgcn_readlane(mine_d, k);
            const double far = __hiloint2double(
                __builtin_amdgcn_readlane(__double2hiint(mine_far), k),
                __builtin_amdgcn_readlane(__double2loint(mine_far), k));
            const uint32_t wn = (uint32_t)(word[k] >> SM_COUNT);
            const u64 wp = word[k] & ((1ull << SM_COUNT) - 1);
            if (tid >= d) {
                n += wn;
                part += wp;
            } else if (wn) {
                rest_n += wn;
                rest += (u64)__builtin_rint(edge_rest * far *
                                            ((double)wn + (double)wp * (1.0 / (1ull << SM_PART))));
            }
        }
        /* the slices' last bins, in units of 2^E of their own */
        if (tid < G && mine.tail_n) {
            u64 m = mine.tail;
            if (r.sc.inf) {
                m = 0;
            } else if (!same) {
                const double de = r.e - sm_e(mine.q);
                const int sh = de >= 63.0 ? 63 : (int)de;
                if (sh) m = (m + (1ull << (sh - 1))) >> sh;
            }
            rest_n += mine.tail_n;
            rest += m;
        }
    }
    if (brief) {
        /* too many tokens: the bins from the row */
        __syncthreads();
        s.mass[tid] = 0;
        s.cur[tid] = 0;
        r.template each_of_row<2>(-3.4028235e38f, each([&](float v, int) {
            if (!(v > -INFINITY)) return;
            const double z = r.sc.z(v), q = sm_q(z);
            const int bin = sm_bin(r.first, q);
            if (bin < LAST) {
                atomicAdd(&s.cur[bin], 1u);
                atomicAdd(&s.mass[bin], sm_bin_word(z, q));
            } else {
                rest_n++;
                rest += sm_weight(z - r.e, a.sh);
            }
        }));
        n = s.cur[tid];
        part = s.mass[tid];
    }
    if (__any(rest_n != 0)) {
        rest_n = sm_wave_scan(rest_n);
        rest = sm_wave_scan(rest);
        if (lane == 63) {
            atomicAdd(&s.tail_n, rest_n);
            atomicAdd(&s.tail, rest);
        }
    }
    __syncthreads();
    if (tid == LAST) n = s.tail_n;
    const u64 m = tid == LAST ? s.tail : sm_bin_sum(edge, n, part);
    u64 mi = m;
    uint32_t ni = n;
    r.scan(mi, ni);
    s.sum[tid] = mi;
    s.n[tid] = ni;
    __syncthreads();
    const int all = (int)s.n[LAST];

    /* ---- the bins where the limits and the pick may be: what comes before them and
     *      what comes through them bounds every sum ---- */
    const bool by_k = top_k > 0 && top_k < all;
    if (tid < 64) {
        int kb = LAST, pb0 = LAST, pb1 = LAST, mb = LAST;
        if (by_k) kb = sm_first(SM_BINS, [&](int i) { return s.n[i] >= (uint32_t)top_k; });
        u64 lo = by_k ? r.sum_before(kb) : s.sum[LAST], hi = s.sum[kb];
        if (by_p) {
            pb1 = min(kb, r.sum_bin(part_of(hi)));
            pb0 = by_k ? min(kb, r.sum_bin(part_of(lo ? lo : 1))) : pb1;
        }
        /* the first bin whose lower edge is under the floor has the last that stays */
        if (by_floor)
            mb = min(sm_first(SM_BINS, [&](int i) {
                         return sm_exp2(fmin((r.first - i) * (1.0 / 32.0) - zmost, 0.0)) <
                                (double)floor_;
                     }), LAST);
        const int c0 = min(min(kb, pb0), mb), c1 = min(min(kb, pb1), mb);
        /* listed are all bins up to the last cut, if they fit, else the ones that may be
         * needed; top-k's is if it is the cut or top-p takes a part of its sum */
        const bool need_k = by_k && (by_p || kb <= c1);
        const int kn = need_k && kb > c1 ? (int)(s.n[kb] - r.n_before(kb)) : 0;
        const bool whole = (int)s.n[c1] + kn <= SP_LIST;
        int ub0 = 0, ub1 = c1;
        if (!whole) {
            if (by_k || by_p || by_floor) {
                lo = max(r.sum_before(c0), 1ull);
                hi = s.sum[c1];
            }
            ub0 = min(r.sum_bin(place_of(lo)), c1);
            ub1 = min(r.sum_bin(place_of(hi)), c1);
        }
        if (tid == 0) s.where = SmWhere{kb, pb0, pb1, mb, c1, ub0, ub1, need_k, whole};
    }
    __syncthreads();
    const SmWhere at = s.where;
    const int kb = at.kb, pb0 = at.pb0, pb1 = at.pb1, mb = at.mb, ub0 = at.ub0, ub1 = at.ub1;
    const bool need_k = at.need_k, whole = at.whole;
    /* The list has the bins of the limits and of the pick; where they are too many
     * together, of the limits first and then, as the cut is known, of the pick. */
    SmPlace cut{0, s.sum[LAST], LAST, all};       /* key 0 is behind the whole bin */
    bool limits = true, pick = true;
    int u0 = ub0, u1 = ub1;
#pragma unroll 1
    for (;;) {
        const bool in = whole ? (need_k && tid == kb) || tid <= at.c1
                              : (limits && ((need_k && tid == kb) ||
                                            (by_p && tid >= pb0 && tid <= pb1) ||
                                            (by_floor && tid == mb))) ||
                                    (pick && tid >= u0 && tid <= u1);
        /* which lie in two ranges */
        int b0 = 0, b1 = at.c1, b2 = need_k ? kb : 0, b3 = need_k ? kb : at.c1;
        if (!whole) {
            b0 = min(min(limits && need_k ? kb : LAST, limits && by_p ? pb0 : LAST),
                     limits && by_floor ? mb : LAST);
            b1 = max(max(limits && need_k ? kb : 0, limits && by_p ? pb1 : 0),
                     limits && by_floor ? mb : 0);
            if (b0 > b1) b0 = b1 = u0;
            b2 = pick ? u0 : b0;
            b3 = pick ? u1 : b1;
        }
        u64 none = 0;
        uint32_t len = in ? n : 0;
        r.scan(none, len);
        s.off[tid] = in && n ? (int)(len - n) : -1;
        if (tid == LAST) s.len = (int)len;
        __syncthreads();
        const int listed = s.len;
        __syncthreads();
        if (listed > SP_LIST) {
            if (!(limits && pick) || whole || !(by_k || by_p || by_floor)) break;
            pick = false;
            continue;
        }
        if (!r.list(b0, b1, b2, b3, listed)) break;
        if (pick && tid >= 64) return;
        auto place = [&](int b, int i) {
            return SmPlace{s.key[i], s.through[i], b, (int)r.n_before(b) + i - s.off[b] + 1};
        };
        /* the token of bin b that passes the sum, or the bin's last */
        auto token = [&](int b, u64 need) {
            const int off = s.off[b], end = off + (int)(s.n[b] - r.n_before(b)) - 1;
            const int i = sm_first(listed, [&](int j) { return s.through[j] >= need; });
            return place(b, min(max(i, off), end));
        };
        if (limits) {
            if (need_k) cut = place(kb, s.off[kb] + top_k - 1 - (int)r.n_before(kb));
            if (by_p) {
                const u64 need = part_of(cut.sum);
                const int b = min(max(r.sum_bin(need), pb0), pb1);
                if (s.off[b] >= 0) {              /* else min_p cuts before it */
                    const SmPlace c = token(b, need);
                    if (c.n < cut.n) cut = c;
                }
            }
            if (by_floor && mb <= cut.bin) {
                /* up to the first of the bin that is under it */
                SmPlace c{~0ull, r.sum_before(mb), mb, (int)r.n_before(mb)};
                const int off = s.off[mb];
                if (off >= 0) {
                    const int i = sm_first((int)(s.n[mb] - r.n_before(mb)),
                                           [&](int j) { return under(s.key[off + j]); });
                    if (i > 0) c = place(mb, off + i - 1);
                }
                if (c.n < cut.n) cut = c;
            }
        }
        const u64 need = place_of(cut.sum);
        if (!pick) {
            u0 = u1 = min(min(max(r.sum_bin(need), ub0), ub1), cut.bin);
            limits = false;
            pick = true;
            __syncthreads();
            continue;
        }
        const SmPlace got = token(min(min(max(r.sum_bin(need), u0), u1), cut.bin), need);
        if (tid == 0) {
            /* behind the cut only by the roundings of the bins' sums */
            const u64 best = got.n > cut.n ? cut.key : got.key;
            const double v = sm_exp2(r.sc.z(sm_value(best)) - r.e) * unit;
            done(sm_token(best), (float)(v / (double)cut.sum), cut.n);
        }
        return;
    }
    cut = SmPlace{0, s.sum[LAST], LAST, all};

    /* ---- more tokens than the list takes: each limit and then the pick by passes over the
     *      row. Where the order passes `need` tokens or the sum `need`, in a bin that is
     *      known: the bin's range of keys is split by 1024 until the token that does is alone,
     *      or, where roundings of the bins' sums leave the tokens short, the bin's last. ---- */
#pragma unroll 1
    for (int phase = 0; phase < 4; phase++) {     /* top-k, top-p, min-p, the pick */
        u64 need = 0;
        int b = 0;
        if (phase == 0) {
            if (!by_k) continue;
            need = (u64)top_k;
            b = kb;
        } else if (phase == 1) {
            if (!by_p) continue;
            need = part_of(cut.sum);
            b = r.sum_bin(need);
            if (b > cut.bin || need >= cut.sum) continue;
        } else if (phase == 2) {
            if (!by_floor || mb > cut.bin) continue;
            b = mb;
        } else {
            need = place_of(cut.sum);
            b = min(r.sum_bin(need), cut.bin);
        }
        float xlo, xhi;
        r.range_of(b, b, &xlo, &xhi);
        u64 key0 = am_key(xlo, INT32_MAX), key1 = am_key(xhi, 0), sum0 = r.sum_before(b);
        uint32_t n0 = r.n_before(b);
        const u64 stay = cut.bin == b ? cut.key : 0;
        SmPlace got;
#pragma unroll 1
        for (;;) {
            const int bits = 64 - __clzll((long long)((key1 - key0) | 1));
            const int sh = max(0, bits - 10);
            __syncthreads();
            s.mass[tid] = 0;
            s.best[tid] = 0;
            s.cur[tid] = 0;
            if (tid == 0) s.hit = {~0ull, sum0, phase == 2 ? b : -1, (int)n0};
            r.template each_of_row<2>(xlo, each([&](float v, int t) {
                if (__builtin_amdgcn_fmed3f(v, xlo, xhi) != v) return;
                const double z = r.sc.z(v);
                if (sm_bin(r.first, sm_q(z)) != b) return;
                const u64 key = am_key(v, t), w = r.weight(z);
                if (phase == 2) {
                    if (key < stay || under(key)) return;
                    atomicMin(&s.hit.key, key);
                    atomicAdd(&s.hit.sum, w);
                    atomicAdd(&s.hit.n, 1);
                    return;
                }
                if (key < key0 || key > key1) return;
                const int d = (int)((key1 - key) >> sh);
                atomicAdd(&s.mass[d], w);
                atomicAdd(&s.cur[d], 1u);
                atomicMax(&s.best[d], key);
            }));
            if (phase == 2) {
                got = s.hit;
                break;
            }
            const u64 dm = s.mass[tid];
            const uint32_t dn = s.cur[tid];
            u64 dmi = dm;
            uint32_t dni = dn;
            r.scan(dmi, dni);
            const u64 through = phase == 0 ? n0 + dni : sum0 + dmi;
            const u64 before = phase == 0 ? n0 + dni - dn : sum0 + dmi - dm;
            if (dn && before < need && through >= need)
                s.hit = {s.best[tid], sum0 + dmi, tid, (int)(n0 + dni)};
            __syncthreads();
            int d = s.hit.bin;
            __syncthreads();
            if (d < 0) {
                if (dn) atomicMax(&s.hit.bin, tid);
                __syncthreads();
                d = max(0, s.hit.bin);
                __syncthreads();
                if (tid == d) s.hit = {s.best[tid], sum0 + dmi, tid, (int)(n0 + dni)};
                __syncthreads();
            }
            got = s.hit;
            got.bin = b;
            const uint32_t nd = s.cur[d];
            const u64 md = s.mass[d];
            if (nd <= 1 || sh == 0) break;
            n0 = got.n - nd;
            sum0 = got.sum - md;
            key1 = got.key;
            const u64 end = key1 > ((1ull << sh) - 1) ? key1 - ((1ull << sh) - 1) : 0;
            key0 = end > key0 ? end : key0;
        }
        __syncthreads();
        if (phase == 3) {
            if (tid == 0) {
                const u64 key = b == cut.bin && got.key < cut.key ? cut.key : got.key;
                const double v = sm_exp2(r.sc.z(sm_value(key)) - r.e) * unit;
                done(sm_token(key), (float)(v / (double)cut.sum), cut.n);
            }
        } else if (got.n < cut.n) {
            cut = got;
        }
    }
}

struct SamplePlan {
    int ns, nc, sh;
    size_t top, cmax, bytes;                      /* offsets; the bins are first */
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
    p.top = slices * SM_BINS * sizeof(u64);
    p.cmax = p.top + slices * sizeof(SmTop);
    p.bytes = (p.cmax + (size_t)n * p.nc * sizeof(float) + 15) / 16 * 16;
    return p;
}

constexpr int SM_ROWS = 65536, SM_VOCAB = 1 << 22;

/* As many rows a launch as keep its threads under 2^32; one launch up to 2^23 slices. */
template <class T>
int sample_launch(SampleJob a, int n, int *d_pick, hipStream_t st)
{
    const int most = (int)(((1ll << 32) / SM_THREADS - 1) / a.ns);
    for (a.row0 = 0; a.row0 < n; a.row0 += most) {
        const unsigned rows = (unsigned)(n - a.row0 < most ? n - a.row0 : most);
        hipLaunchKernelGGL(k_sample_slices<T>, dim3(rows * (unsigned)a.ns), dim3(SM_THREADS), 0, st,
                           a);
        HIP_OK(hipGetLastError(), "sample slices launch");
        hipLaunchKernelGGL(k_sample_pick<T>, dim3(rows), dim3(SP_THREADS), 0, st, a, d_pick);
        HIP_OK(hipGetLastError(), "sample pick launch");
    }
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
    SampleJob a{d_logits, stride, 0, vocab, p.ns, p.nc, p.sh, *s, (u64 *)base,
                (SmTop *)(base + p.top), (float *)(base + p.cmax), d_kept, d_prob};
    hipStream_t st = (hipStream_t)stream;
    return fmt == DSV4_WF32 ? sample_launch<float>(a, n, d_pick, st)
                            : sample_launch<uint16_t>(a, n, d_pick, st);
}
