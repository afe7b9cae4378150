/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_kvrows.hip - rows of the latent cache written from f32 or bf16 rows
 * on the device, and read back, on gfx950.
 *
 * APPEND. A row goes to its cache format by one wave: rotated if asked (the
 * arithmetic of dsv4_rope.hip), then stored as f32, as bf16 (to nearest even)
 * or as e4m3(x / s). s is the least power of two with max |x| <= 448 s over
 * the finite elements, so x / s is exact and each element is rounded once;
 * it comes from the maximum's bits alone: 448 is 1.75 * 2^8, so s has the
 * maximum's exponent less 8, one more where the significand is over 1.75.
 * A row read back as code * s has a maximum of 224 s (then it gets s / 2 and
 * every code doubles, which e4m3 holds exactly) or more (then it gets s
 * again), so writing it again keeps its values.
 * Bound: x read once (twice past 768 elements), the codes written once. One
 * row per wave keeps the maximum in registers: no LDS, no second launch.
 * Where two tokens name one row the later is written. A workgroup compares the
 * later entries of a short list with its four tokens' rows; with a long one it
 * hashes its tokens' rows into LDS and looks the entries up there, so that one
 * costs an LDS read however many tokens the workgroup has, and it takes more
 * of them, 256 at most, as the list grows: of rows of 512 f32 to FP8, 2000 take
 * 4.3 us compared and looked up, 6000 7.4 and 6.3, 60000 245 and 42 (27 where they
 * follow row0); of rows of 32, 118000 take 817 and 70.
 *
 * READ. A thread makes 16 bytes of output at a time, so that stores, the
 * larger stream from an FP8 cache, are whole lines, and two of them: 131072
 * rows of 576 from FP8 to f32 take 69.2 us (5.5 TB/s), with four pieces a thread
 * 69.7 and with one 71.7; 2048 rows 3.0, 3.4 and 2.7.
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

namespace {

#include "dsv4_rows_io.h"

constexpr int KR_THREADS = 256;
constexpr int KR_ROWS = KR_THREADS / 64;          /* rows per workgroup      */
constexpr int KR_DIM = 16384;                     /* the longest row         */
constexpr int KR_MOST = 1 << 30;                  /* most rows of a call     */

struct AppendJob {
    void *kv;
    float *scales;
    int kv_stride, kv_rows;
    const void *x;
    long long xs;
    int n, dim;
    const int *rows;
    int row0;
    const int *pos;                               /* nullptr: not rotated    */
    dsv4_gpu_rope rp;
    int tok;                                      /* tokens of a workgroup   */
};

constexpr int AP_WAVES = 16;                      /* of a workgroup with a list */
constexpr int AP_TOK = 256;                       /* its most tokens         */
constexpr int AP_BITS = 12;                       /* slots, 16 a token at least */
constexpr int AP_SHORT = 4096;                    /* lists that are compared */
/* Most tokens of a launch. Of a list's launches a later one writes over the rows of
 * those before it, so each looks for later tokens among its own only and a list's
 * cost grows with its length, not its square; without a list 64 threads a token
 * stay below a launch's 2^32. */
constexpr int AP_LIST = 1 << 17, AP_RUN = 1 << 25;
enum { AP_NONE, AP_COMPARE, AP_HASH };            /* what a list takes       */

__device__ __forceinline__ uint32_t row_slot(int row)
{
    return ((uint32_t)row * 2654435761u) >> (32 - AP_BITS);
}

/* late[k] for tokens t0 + k of a workgroup, k < tok: a later token of the list
 * names the same row. The table holds the last of the workgroup's tokens for
 * each row. */
__device__ __forceinline__ void find_late(const int *list, int n, int kv_rows, int t0, int tok,
                                          int *row, int *late, int *tbl)
{
    const int tid = threadIdx.x, nth = blockDim.x;
    for (int i = tid; i < 1 << AP_BITS; i += nth) tbl[i] = -1;
    for (int k = tid; k < tok; k += nth) {
        row[k] = t0 + k < n ? list[t0 + k] : -1;
        late[k] = 0;
    }
    __syncthreads();
    for (int k = tid; k < tok; k += nth) {
        const int r = row[k];
        if (r < 0 || r >= kv_rows) continue;
        /* a slot's row does not change once it is taken, and at most 256 of the
         * 4096 are, so this ends */
        for (uint32_t s = row_slot(r);; s = (s + 1) & ((1 << AP_BITS) - 1)) {
            const int was = atomicCAS(&tbl[s], -1, k);
            if (was == -1) break;
            if (row[was] != r) continue;
            late[min(k, atomicMax(&tbl[s], k))] = 1;
            break;
        }
    }
    __syncthreads();
    constexpr int G = 4;                          /* loads in flight         */
    for (int j = t0 + tok + tid; j < n; j += G * nth) {
        int r[G];
#pragma unroll
        for (int u = 0; u < G; u++) r[u] = list[min(j + u * nth, n - 1)];
#pragma unroll
        for (int u = 0; u < G; u++) {             /* the last entry again: no harm */
            uint32_t s = row_slot(r[u]);
            for (int k; (k = tbl[s]) >= 0; s = (s + 1) & ((1 << AP_BITS) - 1))
                if (row[k] == r[u]) {
                    late[k] = 1;
                    break;
                }
        }
    }
    __syncthreads();
}

/* Elements c .. c + V - 1 of a row, rotated by the table row r (nullptr
 * tables: a position outside them). */
template <class T, int V>
__device__ __forceinline__ void row_values(const AppendJob &a, const T *x, int c,
                                           const float *cs, const float *sn, float *v)
{
    io_load<T, V>(x + c, v);
    const int rc = c - a.rp.offset;
    if (!a.pos || rc < 0 || rc >= a.rp.dim) return;
    const int half = a.rp.dim / 2;
    if (!cs) {
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = __uint_as_float(0x7FC00000u);
        return;
    }
    if (a.rp.layout == DSV4_GPU_ROPE_PAIRS) {
        if constexpr (V == 1) {
            float o;
            io_load<T, 1>(x + (a.rp.offset + (rc ^ 1)), &o);
            const float cc = cs[rc >> 1], ss = sn[rc >> 1];
            v[0] = (rc & 1) ? o * ss + v[0] * cc : v[0] * cc - o * ss;
        } else {
#pragma unroll
            for (int k = 0; k < V; k += 2) {
                const float cc = cs[(rc + k) >> 1], ss = sn[(rc + k) >> 1];
                const float x0 = v[k], x1 = v[k + 1];
                v[k] = x0 * cc - x1 * ss;
                v[k + 1] = x0 * ss + x1 * cc;
            }
        }
        return;
    }
    const bool second = rc >= half;
    const int p = second ? rc - half : rc;
    float o[V];
    io_load<T, V>(x + (second ? c - half : c + half), o);
#pragma unroll
    for (int k = 0; k < V; k++) {
        const float cc = cs[p + k], ss = sn[p + k];
        v[k] = second ? o[k] * ss + v[k] * cc : v[k] * cc - o[k] * ss;
    }
}

__device__ __forceinline__ bool finite_f(float v)
{
    return (__float_as_uint(v) & 0x7F800000u) != 0x7F800000u;
}

/* The row's scale and its inverse, both powers of two, from its largest
 * finite magnitude. */
__device__ __forceinline__ void row_scale(float top, float *s, float *inv)
{
    const uint32_t b = __float_as_uint(top);
    int e = (int)(b >> 23) - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    if (e < 1) e = 1;
    if (b == 0u) e = 127;
    *s = __uint_as_float((uint32_t)e << 23);
    *inv = __uint_as_float((uint32_t)(254 - e) << 23);
}

/* Four e4m3 codes of four values at or below 448 in magnitude; what is not
 * finite becomes NaN. */
__device__ __forceinline__ uint32_t codes4(const float *v)
{
    float t[4];
#pragma unroll
    for (int k = 0; k < 4; k++) t[k] = finite_f(v[k]) ? v[k] : __uint_as_float(0x7FC00000u);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(t[0], t[1], 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(t[2], t[3], r, true);
    return (uint32_t)r;
}

template <int KVF, int V>
__device__ __forceinline__ void row_store(const AppendJob &a, size_t at, const float *v,
                                          float inv)
{
    if constexpr (KVF == DSV4_GPU_KV_F32) {
        io_store<float, V>((float *)a.kv + at, v);
    } else if constexpr (KVF == DSV4_GPU_KV_BF16) {
        io_store<uint16_t, V>((uint16_t *)a.kv + at, v);
    } else {
        float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < V; k++) t[k] = v[k] * inv;
        const uint32_t c = codes4(t);
        if constexpr (V == 4) __builtin_memcpy((uint8_t *)a.kv + at, &c, 4);
        else ((uint8_t *)a.kv)[at] = (uint8_t)c;
    }
}

/* Pieces of V from element c, the last moved back to end with the row: what it
 * shares with the one before it is computed and written twice, the same. NC
 * pieces per lane kept in registers between the maximum and the
 * store (the row is no longer than 64 V NC); NC 0: read again. */
template <class T, int KVF, int V, int NC, int LIST>
__global__ void __launch_bounds__(LIST == AP_HASH ? 64 * AP_WAVES : KR_THREADS)
k_append(AppendJob a)
{
    constexpr int WV = LIST == AP_HASH ? AP_WAVES : KR_ROWS;
    __shared__ int late[LIST == AP_HASH ? AP_TOK : KR_ROWS];
    __shared__ int lrow[LIST == AP_HASH ? AP_TOK : 1];
    __shared__ int tbl[LIST == AP_HASH ? 1 << AP_BITS : 1];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int t0 = blockIdx.x * (LIST == AP_HASH ? a.tok : KR_ROWS);
    constexpr int KEEP = NC > 0 ? NC : 1;
    float v[KEEP][V];
    const float *cs, *sn;
    auto load = [&](int t) {
        cs = sn = nullptr;
        if (a.pos) {
            const int p = a.pos[t];
            if (p >= 0 && p < a.rp.max_pos) {
                cs = a.rp.cos + (size_t)p * (a.rp.dim / 2);
                sn = a.rp.sin + (size_t)p * (a.rp.dim / 2);
            }
        }
        if constexpr (NC > 0) {
            const T *x = (const T *)a.x + t * a.xs;
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const int c = (i * 64 + lane) * V;
                if (c < a.dim) {
                    row_values<T, V>(a, x, min(c, a.dim - V), cs, sn, v[i]);
                } else {
#pragma unroll
                    for (int k = 0; k < V; k++) v[i][k] = 0.0f;
                }
            }
        }
    };
    auto store = [&](int t, int row) {
        const T *x = (const T *)a.x + t * a.xs;
        const size_t at = (size_t)row * a.kv_stride;
        float inv = 1.0f;
        if constexpr (KVF == DSV4_GPU_KV_FP8) {
            float top = 0.0f;
            if constexpr (NC > 0) {
#pragma unroll
                for (int i = 0; i < NC; i++)
#pragma unroll
                    for (int k = 0; k < V; k++)
                        if (finite_f(v[i][k])) top = fmaxf(top, fabsf(v[i][k]));
            } else {
                for (int c = lane * V; c < a.dim; c += 64 * V) {
                    row_values<T, V>(a, x, min(c, a.dim - V), cs, sn, v[0]);
#pragma unroll
                    for (int k = 0; k < V; k++)
                        if (finite_f(v[0][k])) top = fmaxf(top, fabsf(v[0][k]));
                }
            }
            top = wave_max(top);
            float s;
            row_scale(top, &s, &inv);
            if (lane == 0) a.scales[row] = s;
        }
        if constexpr (NC > 0) {
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const int c = (i * 64 + lane) * V;
                if (c < a.dim) row_store<KVF, V>(a, at + min(c, a.dim - V), v[i], inv);
            }
        } else {
            for (int c = lane * V; c < a.dim; c += 64 * V) {
                row_values<T, V>(a, x, min(c, a.dim - V), cs, sn, v[0]);
                row_store<KVF, V>(a, at + min(c, a.dim - V), v[0], inv);
            }
        }
    };
    /* the first row's loads are out while the list is looked through */
    const int t = t0 + w;
    if (t < a.n) load(t);
    if constexpr (LIST == AP_HASH) {
        find_late(a.rows, a.n, a.kv_rows, t0, a.tok, lrow, late, tbl);
        for (int k = w; k < a.tok && t0 + k < a.n; k += WV) {
            const int row = lrow[k];
            if (row < 0 || row >= a.kv_rows || late[k]) continue;
            if (k != w) load(t0 + k);
            store(t0 + k, row);
        }
        return;
    }
    if constexpr (LIST == AP_COMPARE) {
        if (threadIdx.x < KR_ROWS) late[threadIdx.x] = 0;
        __syncthreads();
        int mine[KR_ROWS];
#pragma unroll
        for (int k = 0; k < KR_ROWS; k++) mine[k] = a.rows[min(t0 + k, a.n - 1)];
        for (int j = t0 + 1 + (int)threadIdx.x; j < a.n; j += KR_THREADS) {
            const int r = a.rows[j];
#pragma unroll
            for (int k = 0; k < KR_ROWS; k++)
                if (r == mine[k] && j > t0 + k) late[k] = 1;
        }
        __syncthreads();
        if (late[w]) return;
    }
    if (t >= a.n) return;
    const int row = LIST == AP_NONE ? a.row0 + t : a.rows[t];
    if (row >= 0 && row < a.kv_rows) store(t, row);
}

struct ReadJob {
    void *out;
    long long os;
    const void *kv;
    const float *scales;
    int kv_stride, kv_rows;
    const int *rows;
    int row0, dim, items;
    IoDiv units;
};

constexpr int RD_IL = 2;                          /* pieces per thread       */

template <class T, int KVF, int V>
__global__ void __launch_bounds__(KR_THREADS) k_read(ReadJob a)
{
    const uint32_t i0 = blockIdx.x * (KR_THREADS * RD_IL) + threadIdx.x;
    float v[RD_IL][V];
    T *o[RD_IL];
#pragma unroll
    for (int u = 0; u < RD_IL; u++) {
        const uint32_t i = i0 + u * KR_THREADS;
        o[u] = nullptr;
#pragma unroll
        for (int k = 0; k < V; k++) v[u][k] = 0.0f;
        if (i >= (uint32_t)a.items) continue;
        const uint32_t t = a.units.div(i);
        const int c = min((int)(i - t * a.units.d) * V, a.dim - V);
        o[u] = (T *)a.out + (long long)t * a.os + c;
        const int row = a.rows ? a.rows[t] : a.row0 + (int)t;
        if (row < 0 || row >= a.kv_rows) continue;
        const size_t at = (size_t)row * a.kv_stride + c;
        if constexpr (KVF == DSV4_GPU_KV_F32) {
            io_load<float, V>((const float *)a.kv + at, v[u]);
        } else if constexpr (KVF == DSV4_GPU_KV_BF16) {
            io_load<uint16_t, V>((const uint16_t *)a.kv + at, v[u]);
        } else {
            const uint8_t *p = (const uint8_t *)a.kv + at;
            const float s = a.scales[row];
            if constexpr (V == 1) {
                v[u][0] = dec_e4m3(p[0]) * s;
            } else {
#pragma unroll
                for (int k = 0; k < V; k += 4) {
                    uint32_t w;
                    __builtin_memcpy(&w, p + k, 4);
                    dec_e4m3x4(w, v[u] + k);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[u][k + e] *= s;
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < RD_IL; u++)
        if (o[u]) io_store<T, V>(o[u], v[u]);
}

/* -1 with a message unless the cache's own description holds, for a call of n
 * rows. */
int cache_ok(const char *what, const void *kv, const float *scales, int fmt, int stride, int rows,
             int dim, int n)
{
    if (fmt != DSV4_GPU_KV_F32 && fmt != DSV4_GPU_KV_BF16 && fmt != DSV4_GPU_KV_FP8) {
        DSV4_ERR("%s: unknown cache format %d", what, fmt);
        return -1;
    }
    if (dim <= 0 || stride < dim || rows <= 0) {
        DSV4_ERR("%s: bad cache shape (rows %d of %d, stride %d)", what, rows, dim, stride);
        return -1;
    }
    if (n && (!kv || (fmt == DSV4_GPU_KV_FP8 && !scales))) {
        DSV4_ERR("%s: no cache, or an FP8 cache without row scales", what);
        return -1;
    }
    return 0;
}

template <class T, int KVF, int LIST>
void append_launch(const AppendJob &a, int V, hipStream_t st)
{
    const int tok = LIST == AP_HASH ? a.tok : KR_ROWS;
    const dim3 g((unsigned)(((long long)a.n + tok - 1) / tok));
    const dim3 b(LIST == AP_HASH ? 64 * AP_WAVES : KR_THREADS);
    if (V == 1)
        hipLaunchKernelGGL((k_append<T, KVF, 1, 0, LIST>), g, b, 0, st, a);
    else if (a.dim <= 64 * 4 * 3)
        hipLaunchKernelGGL((k_append<T, KVF, 4, 3, LIST>), g, b, 0, st, a);
    else
        hipLaunchKernelGGL((k_append<T, KVF, 4, 0, LIST>), g, b, 0, st, a);
}

template <class T, int KVF>
void append_list(const AppendJob &a, int V, hipStream_t st)
{
    if (!a.rows) append_launch<T, KVF, AP_NONE>(a, V, st);
    else if (a.n <= AP_SHORT) append_launch<T, KVF, AP_COMPARE>(a, V, st);
    else append_launch<T, KVF, AP_HASH>(a, V, st);
}

template <class T>
void append_fmt(const AppendJob &a, int fmt, int V, hipStream_t st)
{
    if (fmt == DSV4_GPU_KV_F32) append_list<T, DSV4_GPU_KV_F32>(a, V, st);
    else if (fmt == DSV4_GPU_KV_BF16) append_list<T, DSV4_GPU_KV_BF16>(a, V, st);
    else append_list<T, DSV4_GPU_KV_FP8>(a, V, st);
}

template <class T, int V>
void read_fmt(const ReadJob &a, int fmt, hipStream_t st)
{
    const int per = KR_THREADS * RD_IL;
    const dim3 g((a.items + per - 1) / per), b(KR_THREADS);
    if (fmt == DSV4_GPU_KV_F32)
        hipLaunchKernelGGL((k_read<T, DSV4_GPU_KV_F32, V>), g, b, 0, st, a);
    else if (fmt == DSV4_GPU_KV_BF16)
        hipLaunchKernelGGL((k_read<T, DSV4_GPU_KV_BF16, V>), g, b, 0, st, a);
    else
        hipLaunchKernelGGL((k_read<T, DSV4_GPU_KV_FP8, V>), g, b, 0, st, a);
}

} // namespace

extern "C" int dsv4_gpu_kv_append_d(void *d_kv, float *d_kv_scales, int kv_fmt, int kv_stride,
                                    int kv_rows, const void *d_x, int x_fmt, long long x_stride,
                                    int n, int row_dim, const int *d_rows, int row0,
                                    const dsv4_gpu_rope *rope, const int *d_pos, void *stream)
{
    if (cache_ok("kv_append", d_kv, d_kv_scales, kv_fmt, kv_stride, kv_rows, row_dim, n) != 0)
        return -1;
    if (n < 0 || n > KR_MOST || row_dim > KR_DIM || x_stride < row_dim ||
        (x_fmt != DSV4_WF32 && x_fmt != DSV4_WBF16) || (n && !d_x)) {
        DSV4_ERR("kv_append: bad arguments (n %d, row_dim %d, x_fmt %d, x_stride %lld)", n,
                 row_dim, x_fmt, x_stride);
        return -1;
    }
    if (!d_rows && (row0 < 0 || (long long)row0 + n > kv_rows)) {
        DSV4_ERR("kv_append: rows %d .. %lld of a cache of %d", row0, (long long)row0 + n - 1,
                 kv_rows);
        return -1;
    }
    if (rope) {
        const char *bad = dsv4_rope_bad(rope, row_dim);
        if (!bad && n && !d_pos) bad = "no positions";
        if (bad) {
            DSV4_ERR("kv_append: rope: %s", bad);
            return -1;
        }
    }
    if (n == 0) return 0;
    /* pieces of four elements, the last one moved back to the row's end; one by
     * one in rows of less, and where the rotation's pairs do not fall into pieces */
    int V = row_dim < 4 ? 1 : 4;
    if (rope && (row_dim % 4 || rope->offset % 4 || rope->dim % 4 ||
                 (rope->layout == DSV4_GPU_ROPE_HALVES && rope->dim % 8)))
        V = 1;
    const int es = x_fmt == DSV4_WBF16 ? 2 : 4;
    const int most = d_rows ? AP_LIST : AP_RUN;
    for (int t0 = 0; t0 < n; t0 += most) {
        const int m = n - t0 < most ? n - t0 : most;
        AppendJob a{d_kv, d_kv_scales, kv_stride, kv_rows,
                    (const char *)d_x + (size_t)t0 * x_stride * es, x_stride, m, row_dim,
                    d_rows ? d_rows + t0 : nullptr, row0 + (d_rows ? 0 : t0),
                    rope ? d_pos + t0 : nullptr, rope ? *rope : dsv4_gpu_rope{}, 0};
        /* a long list's workgroups: 512 of them fill the card's waves */
        const int per = m / (AP_WAVES * 512) + 1;
        a.tok = AP_WAVES * (per < AP_TOK / AP_WAVES ? per : AP_TOK / AP_WAVES);
        if (x_fmt == DSV4_WF32) append_fmt<float>(a, kv_fmt, V, (hipStream_t)stream);
        else append_fmt<uint16_t>(a, kv_fmt, V, (hipStream_t)stream);
        HIP_OK(hipGetLastError(), "kv_append launch");
    }
    return 0;
}

extern "C" int dsv4_gpu_kv_read_d(void *d_out, int out_fmt, long long out_stride,
                                  const void *d_kv, const float *d_kv_scales, int kv_fmt,
                                  int kv_stride, int kv_rows, const int *d_rows, int row0, int n,
                                  int row_dim, void *stream)
{
    if (cache_ok("kv_read", d_kv, d_kv_scales, kv_fmt, kv_stride, kv_rows, row_dim, n) != 0)
        return -1;
    if (n < 0 || n > KR_MOST || row_dim > KR_DIM || out_stride < row_dim ||
        (out_fmt != DSV4_WF32 && out_fmt != DSV4_WBF16) || (n && !d_out)) {
        DSV4_ERR("kv_read: bad arguments (n %d, row_dim %d, out_fmt %d, out_stride %lld)", n,
                 row_dim, out_fmt, out_stride);
        return -1;
    }
    if (!d_rows && (row0 < 0 || (long long)row0 + n > kv_rows)) {
        DSV4_ERR("kv_read: rows %d .. %lld of a cache of %d", row0, (long long)row0 + n - 1,
                 kv_rows);
        return -1;
    }
    if (d_rows) row0 = 0;
    /* 16 bytes of output, the last piece moved back to the row's end; one by one
     * in rows of less */
    const int es = out_fmt == DSV4_WBF16 ? 2 : 4;
    const int V = row_dim < 16 / es ? 1 : 16 / es;
    const int units = (row_dim + V - 1) / V;
    const int most = (1 << 30) / units;           /* rows of a launch         */
    for (int t0 = 0; t0 < n; t0 += most) {
        const int m = n - t0 < most ? n - t0 : most;
        ReadJob a{(char *)d_out + (size_t)t0 * out_stride * es, out_stride, d_kv, d_kv_scales,
                  kv_stride, kv_rows, d_rows ? d_rows + t0 : nullptr, row0 + t0, row_dim, m * units,
                  IoDiv((uint32_t)units)};
        hipStream_t st = (hipStream_t)stream;
        if (es == 4) {
            if (V > 1) read_fmt<float, 4>(a, kv_fmt, st);
            else read_fmt<float, 1>(a, kv_fmt, st);
        } else {
            if (V > 1) read_fmt<uint16_t, 8>(a, kv_fmt, st);
            else read_fmt<uint16_t, 1>(a, kv_fmt, st);
        }
        HIP_OK(hipGetLastError(), "kv_read launch");
    }
    return 0;
}
