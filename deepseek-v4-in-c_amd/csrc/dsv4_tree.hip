/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_tree.hip - attention of a tree of drafted tokens over the latent cache
 * on gfx950.
 *
 * o = sum_r e^(s_r - m) row_r[:d_v] / (sum_r e^(s_r - m) + e^(sink - m)) over
 * the rows r a token sees, s_r = scale q . row_r[:d_qk], in one pass over the
 * rows with the running maximum m and sum. One workgroup per (token, head).
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

#include <math.h>

namespace {

#include "dsv4_rows_io.h"

constexpr int TR_THREADS = 256;
constexpr int TR_TILE = 64;
constexpr int TR_DQK = 576, TR_DV = 512;

struct TreeJob {
    void *o;
    const void *q;
    int nt, h, dqk, dv;
    const void *kv;
    const float *ks;
    int stride, rows;
    const int *pages;
    int n_pages, page, ctx;
    const uint64_t *mask;
    int window;
    const float *sink;
    float scale;
};

__device__ __forceinline__ unsigned long long seen_drafts(const TreeJob &a, int t)
{
    if (a.mask) return a.mask[t];
    return t >= 63 ? ~0ull : (2ull << t) - 1;
}

/* The drafts that token t sees beside itself: its depth. */
__device__ __forceinline__ int depth_of(unsigned long long see, int t, int nt)
{
    if (nt < 64) see &= (1ull << nt) - 1;
    return __popcll(see & ~(1ull << t));
}

/* Cache row of position p, or -1. */
__device__ __forceinline__ long long cache_row(const TreeJob &a, int p)
{
    long long r = p;
    if (a.pages) {
        const int k = p / a.page;
        if (k >= a.n_pages) return -1;
        const int pg = a.pages[k];
        if (pg < 0) return -1;
        r = (long long)pg * a.page + (p - k * a.page);
    }
    return r < a.rows ? r : -1;
}

__device__ __forceinline__ float cache_at(const TreeJob &a, int fmt, long long row, int c)
{
    const size_t at = (size_t)row * a.stride + c;
    if (fmt == DSV4_GPU_KV_F32) return ((const float *)a.kv)[at];
    if (fmt == DSV4_GPU_KV_BF16)
        return __uint_as_float((uint32_t)((const uint16_t *)a.kv)[at] << 16);
    return dec_e4m3(((const uint8_t *)a.kv)[at]) * a.ks[row];
}

template <class T>
__global__ void __launch_bounds__(TR_THREADS) k_tree(TreeJob a, int fmt)
{
    __shared__ float qs[TR_DQK], sc[TR_TILE];
    __shared__ long long row[TR_TILE];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int t = blockIdx.x / a.h, hd = blockIdx.x - t * a.h;
    for (int c = tid; c < a.dqk; c += TR_THREADS)
        io_load<T, 1>((const T *)a.q + (size_t)blockIdx.x * a.dqk + c, qs + c);
    const unsigned long long see = seen_drafts(a, t);
    const int here = a.ctx + depth_of(see, t, a.nt);
    const int lo = a.window ? max(0, here - a.window + 1) : 0;
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    const int n = a.ctx + a.nt;
    for (int p0 = lo / TR_TILE * TR_TILE; p0 < n; p0 += TR_TILE) {
        __syncthreads();
        if (tid < TR_TILE) {
            const int p = p0 + tid;
            bool ok = p >= lo && p < n;
            if (ok && p >= a.ctx) {
                const int j = p - a.ctx;
                ok = (see >> j) & 1;
                if (ok && a.window)
                    ok = here - (a.ctx + depth_of(seen_drafts(a, j), j, a.nt)) < a.window;
            }
            row[tid] = ok ? cache_row(a, p) : -1;
        }
        __syncthreads();
        for (int k = w; k < TR_TILE; k += 4) {
            const long long r = row[k];
            float s = 0.0f;
            if (r >= 0)
                for (int c = lane; c < a.dqk; c += 64) s = fmaf(qs[c], cache_at(a, fmt, r, c), s);
            s = wave_sum(s);
            if (lane == 0) sc[k] = r >= 0 ? s * a.scale : -INFINITY;
        }
        __syncthreads();
        float top = m;
        for (int k = 0; k < TR_TILE; k++) top = fmaxf(top, sc[k]);
        const float f = top == -INFINITY ? 0.0f : expf(m - top);
        l *= f;
        acc[0] *= f;
        acc[1] *= f;
        m = top;
        /* the tile's own sums first: a chain as long as the context would lose
         * bits where its terms are alike */
        float tl = 0.0f, ta[2] = {0.0f, 0.0f};
        for (int k = 0; k < TR_TILE; k++) {
            if (row[k] < 0) continue;
            const float e = m == -INFINITY && sc[k] == m ? 0.0f : expf(sc[k] - m);
            tl += e;
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int c = tid + i * TR_THREADS;
                if (c < a.dv) ta[i] = fmaf(e, cache_at(a, fmt, row[k], c), ta[i]);
            }
        }
        l += tl;
        acc[0] += ta[0];
        acc[1] += ta[1];
    }
    if (l != 0.0f && a.sink) l += expf(a.sink[hd] - m);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int c = tid + i * TR_THREADS;
        const float v = acc[i] * inv;
        if (c < a.dv) io_store<T, 1>((T *)a.o + (size_t)blockIdx.x * a.dv + c, &v);
    }
}

/* What is wrong with a call's shape, or nullptr. */
const char *tree_bad(int fmt, int nt, int h, int d_qk, int d_v, int kv_fmt, int n_ctx, int window)
{
    if (fmt != DSV4_WF32 && fmt != DSV4_WBF16) return "an unknown type of q";
    if (kv_fmt != DSV4_GPU_KV_F32 && kv_fmt != DSV4_GPU_KV_BF16 && kv_fmt != DSV4_GPU_KV_FP8)
        return "an unknown cache format";
    if (nt < 0 || nt > DSV4_MAX_BATCH) return "0 to 64 tokens are taken";
    if (h <= 0 || h > 4096) return "1 to 4096 heads are taken";
    if (d_v <= 0 || d_qk < d_v || d_qk > TR_DQK || d_v > TR_DV)
        return "widths d_v <= d_qk, at most 512 and 576, are taken";
    if (n_ctx < 0 || n_ctx > INT32_MAX - 1024 || window < 0) return "a negative or too long context";
    return nullptr;
}

} // namespace

extern "C" size_t dsv4_gpu_tree_attn_scratch_bytes(int fmt, int nt, int h, int d_qk, int d_v,
                                                   int kv_fmt, int n_ctx, int window)
{
    if (tree_bad(fmt, nt, h, d_qk, d_v, kv_fmt, n_ctx, window)) return 0;
    return 0;
}

extern "C" int dsv4_gpu_tree_attn_d(void *d_o, const void *d_q, int fmt, int nt, int h, int d_qk,
                                    int d_v, const void *d_kv, const float *d_kv_scales,
                                    int kv_fmt, int kv_stride, int kv_rows, const int *d_pages,
                                    int n_pages, int page_rows, int n_ctx, const uint64_t *d_mask,
                                    int window, const float *d_sink, float scale, void *d_scratch,
                                    size_t scratch_bytes, void *stream)
{
    if (const char *bad = tree_bad(fmt, nt, h, d_qk, d_v, kv_fmt, n_ctx, window)) {
        DSV4_ERR("tree_attn: %s (fmt %d, nt %d, h %d, d_qk %d, d_v %d, cache %d, n_ctx %d, window "
                 "%d)", bad, fmt, nt, h, d_qk, d_v, kv_fmt, n_ctx, window);
        return -1;
    }
    if (kv_stride < d_qk || kv_rows <= 0 || (d_pages && (page_rows <= 0 || n_pages < 0))) {
        DSV4_ERR("tree_attn: bad cache shape (stride %d, rows %d, %d pages of %d)", kv_stride,
                 kv_rows, n_pages, page_rows);
        return -1;
    }
    if (nt == 0) return 0;
    if (!d_o || !d_q || !d_kv || (kv_fmt == DSV4_GPU_KV_FP8 && !d_kv_scales)) {
        DSV4_ERR("tree_attn: a missing buffer");
        return -1;
    }
    TreeJob a{d_o, d_q, nt, h, d_qk, d_v, d_kv, d_kv_scales, kv_stride, kv_rows, d_pages,
              n_pages, page_rows, n_ctx, d_mask, window, d_sink, scale};
    hipStream_t st = (hipStream_t)stream;
    if (fmt == DSV4_WF32)
        hipLaunchKernelGGL(k_tree<float>, dim3(nt * h), dim3(TR_THREADS), 0, st, a, kv_fmt);
    else
        hipLaunchKernelGGL(k_tree<uint16_t>, dim3(nt * h), dim3(TR_THREADS), 0, st, a, kv_fmt);
    HIP_OK(hipGetLastError(), "tree attn launch");
    return 0;
}
