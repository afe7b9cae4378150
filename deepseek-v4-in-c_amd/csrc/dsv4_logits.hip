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
 * between rows. Each wave leaves the best composite and the first allowed
 * token of its part of a row, and a second launch of one wave per row picks.
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_PIECE = 4 * LG_THREADS;          /* tokens of one pass      */
constexpr int LG_WAVES = LG_THREADS / 64;

struct LogitJob {
    float *out;
    const float *in;
    long long stride;
    int nt, vocab, sw, rpg;
    dsv4_gpu_logit_rules r;
    int vec, hvec;                                /* 16-byte pieces          */
    unsigned long long *best;                     /* [nt][slices * LG_WAVES] */
    uint32_t *first;
};

/* Row t's word of drafted tokens it counts. */
__device__ __forceinline__ unsigned long long path_of(const LogitJob &a, int t)
{
    if (a.r.mask) return a.r.mask[t];
    return t >= 63 ? ~0ull : (2ull << t) - 1;
}

__global__ void __launch_bounds__(LG_THREADS) k_logits(LogitJob a)
{
    extern __shared__ int cnt[];                  /* [sw]                    */
    const int tid = threadIdx.x;
    const int v0 = blockIdx.x * a.sw;
    const int t0 = blockIdx.y * a.rpg, t1 = min(t0 + a.rpg, a.nt);
    const bool counts = a.r.n_hist > 0 || a.r.draft;
    int mine = -1;                                /* this lane's draft's slot */
    if (counts) {
        for (int i = tid; i < a.sw; i += LG_THREADS) cnt[i] = 0;
        __syncthreads();
        const uint32_t lim = (uint32_t)min(a.sw, a.vocab - v0);
        int i = 0;
        if (a.hvec) {
            const u32x4 *h4 = reinterpret_cast<const u32x4 *>(a.r.hist);
            const int n4 = a.r.n_hist / 4;
            for (int k = tid; k < n4; k += LG_THREADS) {
                const u32x4 v = h4[k] - (uint32_t)v0;
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (v[e] < lim) atomicAdd(&cnt[v[e]], 1);
            }
            i = 4 * n4;
        }
        for (i += tid; i < a.r.n_hist; i += LG_THREADS) {
            const uint32_t k = (uint32_t)a.r.hist[i] - (uint32_t)v0;
            if (k < lim) atomicAdd(&cnt[k], 1);
        }
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
        const float *x = a.in + t * a.stride;
        float *y = a.out ? a.out + t * a.stride : nullptr;
        const uint32_t *allow =
            a.r.allow ? a.r.allow + (long long)t * a.r.allow_stride : nullptr;
        unsigned long long best = 0ull;
        uint32_t first = 0xFFFFFFFFu;
        for (int p = 4 * tid; p < a.sw; p += LG_PIECE) {
            const int c = v0 + p;
            if (c >= a.vocab) break;
            const int n = min(4, a.vocab - c);
            const bool whole = a.vec && n == 4;
            float v[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
            if (whole) {
                const f32x4 q = ldf4(x + c);
                v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
                if (a.r.bias) {
                    const f32x4 d = ldf4(a.r.bias + c);
                    b[0] = d.x; b[1] = d.y; b[2] = d.z; b[3] = d.w;
                }
            } else {
                for (int k = 0; k < n; k++) {
                    v[k] = x[c + k];
                    if (a.r.bias) b[k] = a.r.bias[c + k];
                }
            }
            const uint32_t ok = allow ? allow[c >> 5] >> (c & 31) : 0xFu;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int m = counts ? cnt[p + k] : 0;
                if (m > 0) {
                    v[k] = v[k] > 0.0f ? v[k] / a.r.repetition : v[k] * a.r.repetition;
                    v[k] = v[k] - ((float)m * a.r.frequency + a.r.presence);
                }
                if (a.r.bias) v[k] = v[k] + b[k];
                if (!(ok >> k & 1)) {
                    v[k] = -INFINITY;
                } else if (k < n) {
                    const unsigned long long key = am_key(v[k], c + k);
                    best = key > best ? key : best;
                    const uint32_t f = (uint32_t)(c + k) << 1 | (v[k] != v[k] ? 1u : 0u);
                    first = min(first, f);
                }
            }
            if (!y) continue;
            if (whole) {
                *reinterpret_cast<f32x4 *>(y + c) = f32x4{v[0], v[1], v[2], v[3]};
            } else {
                for (int k = 0; k < n; k++) y[c + k] = v[k];
            }
        }
        if (!a.best) continue;
        best = wave_max_u64(best);
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) first = min(first, (uint32_t)__shfl_xor((int)first, o, 64));
        if ((tid & 63) == 0) {
            const size_t at = ((size_t)t * gridDim.x + blockIdx.x) * LG_WAVES + (tid >> 6);
            a.best[at] = best;
            a.first[at] = first;
        }
    }
}

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
        pick[blockIdx.x] = f == 0xFFFFFFFFu ? -1
                         : (f & 1u)        ? (int)(f >> 1)
                                           : (int)(0xFFFFFFFFu - (uint32_t)b);
}

/* Tokens of a slice and rows of a workgroup. */
void plan(int nt, int vocab, int *sw, int *rpg)
{
    *sw = nt >= 4 ? 4 * LG_PIECE : LG_PIECE;
    const int ns = (vocab + *sw - 1) / *sw;
    *rpg = (nt * ns + 1023) / 1024;
}

} // namespace

extern "C" size_t dsv4_gpu_logits_scratch_bytes(int nt, int vocab)
{
    if (nt <= 0 || vocab <= 0 || nt > DSV4_MAX_BATCH) return 0;
    int sw, rpg;
    plan(nt, vocab, &sw, &rpg);
    const size_t n = (size_t)nt * (((size_t)vocab + sw - 1) / sw) * LG_WAVES;
    return n * (sizeof(unsigned long long) + sizeof(uint32_t));
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
    if (rules->n_hist < 0 || (rules->n_hist && !rules->hist) || !(rules->repetition > 0.0f) ||
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
    if (d_pick && (!d_scratch || ((uintptr_t)d_scratch & 15) ||
                   scratch_bytes < dsv4_gpu_logits_scratch_bytes(nt, vocab))) {
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
    plan(nt, vocab, &a.sw, &a.rpg);
    a.r = *rules;
    a.vec = stride % 4 == 0 && (((uintptr_t)d_logits | (uintptr_t)d_out |
                                 (uintptr_t)rules->bias) & 15) == 0;
    a.hvec = rules->n_hist && ((uintptr_t)rules->hist & 15) == 0;
    const int ns = (int)(((long long)vocab + a.sw - 1) / a.sw);
    const size_t n = (size_t)nt * ns * LG_WAVES;
    if (d_pick) {
        a.best = (unsigned long long *)d_scratch;
        a.first = (uint32_t *)(a.best + n);
    }
    hipStream_t st = (hipStream_t)stream;
    const size_t lds = rules->n_hist || rules->draft ? (size_t)a.sw * sizeof(int) : 0;
    hipLaunchKernelGGL(k_logits, dim3(ns, (nt + a.rpg - 1) / a.rpg), dim3(LG_THREADS), lds, st,
                       a);
    HIP_OK(hipGetLastError(), "logits launch");
    if (d_pick) {
        hipLaunchKernelGGL(k_logits_pick, dim3(nt), dim3(64), 0, st, d_pick, a.best, a.first,
                           ns * LG_WAVES);
        HIP_OK(hipGetLastError(), "logits pick launch");
    }
    return 0;
}
