/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_logits.hip - a request's rules on its logits, and the greedy pick
 * under them, on gfx950.
 *
 * For a token with count > 0 in its row's text: y = x > 0 ? x / r : x * r, then y
 * -= count * f + p; then y += bias; a token that the row's grammar does not
 * allow becomes -infinity. Each step is rounded by itself. The pick is the
 * head's scan (dsv4_head.hip) over the allowed tokens: the first of them if it
 * is NaN, else the first maximum, by the same composites.
 *
 * Bound: the logits, read and written once. One pass does everything: a
 * workgroup owns a slice of the vocabulary for a group of rows, counts the
 * history's tokens of its slice in LDS (integer adds, so their order does not
 * matter), and adds and takes back the drafted tokens of each row's own path
 * between rows. It leaves the best composite and the first allowed token of its
 * part of a row, and a second launch of one wave per row picks.
 *
 * 64 rows of 129280 with every rule and 16384 ids of history: 24.6 us from HBM,
 * of which 14 are the 66 MB at a large copy's 4.6 TB/s, 3.5 the second launch
 * and some 5 the history. One row: 5.7 us, both launches' latency.
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_WAVES = LG_THREADS / 64;
/* A longer history is counted by a launch of its own, with four times the
 * threads on a slice; a shorter one each workgroup counts for itself. For 1, 8
 * and 64 rows of 129280, without that launch and with it: 7.6, 9.5, 26.0 and 7.9, 10.5, 26.0
 * us at 16384 ids, 9.9 and 8.7 us for one row of 32768, and 24, 31, 54 and 13, 17,
 * 32 us at 131072. */
constexpr int LC_HIST = 24576;
constexpr int LC_THREADS = 1024, LC_SLICE = 1024;
constexpr int LG_ROWS = 8;                       /* most rows of a workgroup */
constexpr int LG_PIECE = 4 * LG_THREADS;          /* a thread's 4 tokens each */

struct LogitJob {
    float *out;
    const float *in;
    long long stride;
    int nt, vocab, rpg;
    dsv4_gpu_logit_rules r;
    const int *count;                             /* [vocab], or NULL        */
    unsigned long long *best;                     /* [nt][slices]            */
    uint32_t *first;
};

/* Row t's word of drafted tokens it counts. */
__device__ __forceinline__ unsigned long long path_of(const LogitJob &a, int t)
{
    if (a.r.mask) return a.r.mask[t];
    return t >= 63 ? ~0ull : (2ull << t) - 1;
}

/* The history's tokens of the slice [v0, v0 + lim) into cnt. */
template <int THREADS>
__device__ __forceinline__ void count_slice(const LogitJob &a, int v0, uint32_t lim, int *cnt)
{
    const int n4 = a.r.n_hist / 4;
    constexpr int G = 4;                          /* loads in flight         */
    for (int k = threadIdx.x; k < n4; k += G * THREADS) {
        u32x4 v[G];
#pragma unroll
        for (int u = 0; u < G; u++)
            __builtin_memcpy(&v[u], a.r.hist + 4 * min(k + u * THREADS, n4 - 1), 16);
#pragma unroll
        for (int u = 0; u < G; u++)
            if (k + u * THREADS < n4)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (v[u][e] - (uint32_t)v0 < lim) atomicAdd(&cnt[v[u][e] - (uint32_t)v0], 1);
    }
    for (int i = 4 * n4 + threadIdx.x; i < a.r.n_hist; i += THREADS) {
        const uint32_t k = (uint32_t)a.r.hist[i] - (uint32_t)v0;
        if (k < lim) atomicAdd(&cnt[k], 1);
    }
}

/* The history's counts of the whole vocabulary, padded to whole pieces of 4,
 * for k_logits' many groups of rows. */
__global__ void __launch_bounds__(LC_THREADS) k_logits_count(LogitJob a, int *count)
{
    __shared__ int cnt[LC_SLICE];
    const int v0 = blockIdx.x * LC_SLICE, lim = min(LC_SLICE, a.vocab - v0);
    for (int i = threadIdx.x; i < LC_SLICE; i += LC_THREADS) cnt[i] = 0;
    __syncthreads();
    count_slice<LC_THREADS>(a, v0, (uint32_t)lim, cnt);
    __syncthreads();
    for (int i = threadIdx.x; i < (lim + 3) / 4 * 4; i += LC_THREADS) count[v0 + i] = cnt[i];
}

/* A slice of NP pieces and a group of rows. The next row's logits are on their
 * way while a row is computed, the first row's while the history is counted. */
template <int NP>
__global__ void __launch_bounds__(LG_THREADS) k_logits(LogitJob a)
{
    constexpr int SW = NP * LG_PIECE;
    extern __shared__ __attribute__((aligned(16))) int cnt[];   /* [SW] */
    __shared__ unsigned long long wbest[LG_ROWS][LG_WAVES];
    __shared__ uint32_t wfirst[LG_ROWS][LG_WAVES];
    const int tid = threadIdx.x;
    const int v0 = blockIdx.x * SW;
    const int t0 = blockIdx.y * a.rpg, t1 = min(t0 + a.rpg, a.nt);
    const bool counts = a.r.n_hist > 0 || a.r.draft;
    const bool whole = v0 + SW <= a.vocab;

    /* 4 tokens from v0 + c of a row, at any address; 0 past the vocabulary */
    auto load4 = [&](const float *x, int c) -> f32x4 {
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (whole) {
            __builtin_memcpy(&v, x + v0 + c, 16);
            return v;
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (v0 + c + k < a.vocab) v[k] = x[v0 + c + k];
        return v;
    };
    f32x4 x[NP], b[NP];
    uint32_t ok[NP];                              /* allowed, a bit a token  */
    auto row = [&](int t) {
#pragma unroll
        for (int p = 0; p < NP; p++) x[p] = load4(a.in + t * a.stride, p * LG_PIECE + 4 * tid);
        const uint32_t *allow =
            a.r.allow ? a.r.allow + (long long)t * a.r.allow_stride : nullptr;
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const int c = v0 + p * LG_PIECE + 4 * tid, n = max(0, min(4, a.vocab - c));
            ok[p] = (1u << n) - 1;
            if (allow && n) ok[p] &= allow[c >> 5] >> (c & 31);
        }
    };
    row(t0);
#pragma unroll
    for (int p = 0; p < NP; p++)
        b[p] = a.r.bias ? load4(a.r.bias, p * LG_PIECE + 4 * tid) : f32x4{0.f, 0.f, 0.f, 0.f};

    int mine = -1;                                /* this lane's draft's slot */
    if (counts) {
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const int c = p * LG_PIECE + 4 * tid;
            *reinterpret_cast<int4 *>(cnt + c) =
                a.count && v0 + c < a.vocab ? *reinterpret_cast<const int4 *>(a.count + v0 + c)
                                            : int4{0, 0, 0, 0};
        }
        __syncthreads();
        const uint32_t lim = (uint32_t)min(SW, a.vocab - v0);
        if (!a.count) count_slice<LG_THREADS>(a, v0, lim, cnt);
        if (a.r.draft && tid < a.nt) {
            const uint32_t k = (uint32_t)a.r.draft[tid] - (uint32_t)v0;
            if (k < lim) mine = (int)k;
        }
    }
    int held = 0;                                 /* counted for the last row */
    for (int t = t0; t < t1; t++) {
        if (counts) {
            if (a.r.draft) {
                if (t > t0) __syncthreads();
                if (mine >= 0) {
                    const int now = (int)(path_of(a, t) >> tid) & 1;
                    if (now != held) atomicAdd(&cnt[mine], now - held);
                    held = now;
                }
            }
            if (a.r.draft || t == t0) __syncthreads();
        }
        f32x4 v[NP];
        uint32_t may[NP];
#pragma unroll
        for (int p = 0; p < NP; p++) {
            v[p] = x[p];
            may[p] = ok[p];
        }
        if (t + 1 < t1) row(t + 1);
        /* a thread's tokens ascend, so its first maximum is kept by > */
        float top = -INFINITY;
        int at = -1;
        uint32_t first = 0xFFFFFFFFu;
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const int c = v0 + p * LG_PIECE + 4 * tid;
            if (counts) {
                const int4 m4 = *reinterpret_cast<const int4 *>(cnt + p * LG_PIECE + 4 * tid);
                const int m[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (m[k] > 0) {
                        float y = v[p][k];
                        y = y > 0.0f ? y / a.r.repetition : y * a.r.repetition;
                        v[p][k] = y - ((float)m[k] * a.r.frequency + a.r.presence);
                    }
            }
            if (a.r.bias) v[p] = v[p] + b[p];
            if (first == 0xFFFFFFFFu && (may[p] & 15u)) {
                const int k = __builtin_ctz(may[p]);
                const float f = k < 2 ? (k ? v[p].y : v[p].x) : k == 2 ? v[p].z : v[p].w;
                first = (uint32_t)(c + k) << 1 | (f != f ? 1u : 0u);
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (!(may[p] >> k & 1u)) v[p][k] = -INFINITY;
                const bool up = v[p][k] > top;
                top = up ? v[p][k] : top;
                at = up ? c + k : at;
            }
        }
        if (a.out) {
            float *y = a.out + t * a.stride + v0 + 4 * tid;
#pragma unroll
            for (int p = 0; p < NP; p++) {
                if (whole) {
                    __builtin_memcpy(y + p * LG_PIECE, &v[p], 16);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (v0 + p * LG_PIECE + 4 * tid + k < a.vocab) y[p * LG_PIECE + k] = v[p][k];
                }
            }
        }
        if (!a.best) continue;
        /* 0: nothing over -infinity */
        const unsigned long long best = wave_max_u64(at < 0 ? 0ull : am_key(top, at));
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) first = min(first, (uint32_t)__shfl_xor((int)first, o, 64));
        if ((tid & 63) == 0) {
            wbest[t - t0][tid >> 6] = best;
            wfirst[t - t0][tid >> 6] = first;
        }
    }
    if (!a.best) return;
    __syncthreads();
    if (tid < t1 - t0) {
        unsigned long long best = wbest[tid][0];
        uint32_t first = wfirst[tid][0];
#pragma unroll
        for (int k = 1; k < LG_WAVES; k++) {
            best = wbest[tid][k] > best ? wbest[tid][k] : best;
            first = min(first, wfirst[tid][k]);
        }
        const size_t at = (size_t)(t0 + tid) * gridDim.x + blockIdx.x;
        a.best[at] = best;
        a.first[at] = first;
    }
}

/* The pick of a row: its first allowed token if that is NaN or nothing is over
 * -infinity (all that are not NaN then tie, and it is the first of them), else
 * the first maximum. */
__global__ void __launch_bounds__(64)
k_logits_pick(int *__restrict__ pick, const unsigned long long *__restrict__ best,
              const uint32_t *__restrict__ first, int n)
{
    const size_t at = (size_t)blockIdx.x * n;
    unsigned long long b = 0ull;
    uint32_t f = 0xFFFFFFFFu;
    for (int i = threadIdx.x; i < n; i += 64) {
        const unsigned long long k = best[at + i];
        b = k > b ? k : b;
        f = min(f, first[at + i]);
    }
    b = wave_max_u64(b);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) f = min(f, (uint32_t)__shfl_xor((int)f, o, 64));
    if (threadIdx.x == 0)
        pick[blockIdx.x] = f == 0xFFFFFFFFu         ? -1
                         : (f & 1u) || b == 0ull    ? (int)(f >> 1)
                                                    : (int)(0xFFFFFFFFu - (uint32_t)b);
}

/* Pieces of a slice and rows of a workgroup. Few rows take short slices, so that
 * more workgroups share them (one row of 129280: 5.7 us, 6.2 with two pieces);
 * with more rows two pieces cost less than they gain (4 rows 6.4 us with one and 6.8
 * with two, 8 8.3 and 7.4, 64 23.4 and 22.2). Groups of rows are as small as the
 * card's 256 CUs hold at once, six workgroups each (64 rows and 16384 ids: 1024
 * workgroups 25.8 us, 1536 25.9, 2048 27.7, one row each 30.7). */
void plan(int nt, int vocab, int *np, int *rpg)
{
    *np = nt >= 4 ? 2 : 1;
    const int sw = *np * LG_PIECE, ns = (int)(((long long)vocab + sw - 1) / sw);
    const long long groups = ((long long)nt * ns + 1535) / 1536;
    *rpg = (int)(groups < LG_ROWS ? groups : LG_ROWS);
}

} // namespace

extern "C" size_t dsv4_gpu_logits_scratch_bytes(int nt, int vocab)
{
    if (nt <= 0 || vocab <= 0 || nt > DSV4_MAX_BATCH) return 0;
    /* slices of one piece whatever the plan takes, so that the bytes of more rows
     * are enough for fewer, whose slices may be shorter */
    const size_t n = (size_t)nt * (((size_t)vocab + LG_PIECE - 1) / LG_PIECE);
    return (n * (sizeof(unsigned long long) + sizeof(uint32_t)) + 15) / 16 * 16 +
           ((size_t)vocab + 3) / 4 * 4 * sizeof(int);
}

extern "C" int dsv4_gpu_logits_adjust_d(float *d_out, int *d_pick, const float *d_logits, int nt,
                                        int vocab, long long stride,
                                        const dsv4_gpu_logit_rules *rules, void *d_scratch,
                                        size_t scratch_bytes, void *stream)
{
    if (nt < 0 || nt > DSV4_MAX_BATCH || vocab <= 0 || vocab > (1 << 30) || stride < vocab ||
        !rules) {
        DSV4_ERR("logits_adjust: bad arguments (nt %d, vocab %d, stride %lld)", nt, vocab,
                 stride);
        return -1;
    }
    if (rules->n_hist < 0 || rules->n_hist > 1 << 30 || (rules->n_hist && !rules->hist) || !(rules->repetition > 0.0f) ||
        (rules->allow && rules->allow_stride &&
         rules->allow_stride < (int)(((long long)vocab + 31) / 32))) {
        DSV4_ERR("logits_adjust: bad rules (n_hist %d, repetition %g, allow_stride %d)",
                 rules->n_hist, (double)rules->repetition, rules->allow_stride);
        return -1;
    }
    if (nt == 0 || (!d_out && !d_pick)) return 0;
    if (!d_logits) {
        DSV4_ERR("logits_adjust: no logits");
        return -1;
    }
    const bool room = d_scratch && !((uintptr_t)d_scratch & 15) &&
                      scratch_bytes >= dsv4_gpu_logits_scratch_bytes(nt, vocab);
    if (d_pick && !room) {
        DSV4_ERR("logits_adjust: %zu bytes of workspace at %p; the call needs %zu, 16-byte "
                 "aligned", scratch_bytes, d_scratch, dsv4_gpu_logits_scratch_bytes(nt, vocab));
        return -1;
    }
    LogitJob a{};
    a.out = d_out;
    a.in = d_logits;
    a.stride = stride;
    a.nt = nt;
    a.vocab = vocab;
    int np;
    plan(nt, vocab, &np, &a.rpg);
    a.r = *rules;
    const int sw = np * LG_PIECE, ns = (int)(((long long)vocab + sw - 1) / sw);
    const size_t n = (size_t)nt * ns;
    if (d_pick) {
        a.best = (unsigned long long *)d_scratch;
        a.first = (uint32_t *)(a.best + n);
    }
    hipStream_t st = (hipStream_t)stream;
    const int groups = (nt + a.rpg - 1) / a.rpg;
    if (room && rules->n_hist > LC_HIST) {
        int *count = (int *)((char *)d_scratch +
                             (n * (sizeof(unsigned long long) + sizeof(uint32_t)) + 15) / 16 * 16);
        a.count = count;
        hipLaunchKernelGGL(k_logits_count, dim3((unsigned)((vocab + (LC_SLICE - 1ll)) / LC_SLICE)),
                           dim3(LC_THREADS), 0, st, a, count);
        HIP_OK(hipGetLastError(), "logits count launch");
    }
    const size_t lds = rules->n_hist || rules->draft ? (size_t)sw * sizeof(int) : 0;
    hipLaunchKernelGGL(np == 1 ? k_logits<1> : k_logits<2>, dim3(ns, groups),
                       dim3(LG_THREADS), lds, st, a);
    HIP_OK(hipGetLastError(), "logits launch");
    if (d_pick) {
        hipLaunchKernelGGL(k_logits_pick, dim3(nt), dim3(64), 0, st, d_pick, a.best, a.first, ns);
        HIP_OK(hipGetLastError(), "logits pick launch");
    }
    return 0;
}
