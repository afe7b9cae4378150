/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_tree.hip - attention of a tree of drafted tokens over the latent cache
 * on gfx950: the plan, the join and the entry point (the kernel: dsv4_tree.h).
 *
 * For a row of q (token, head) and the cache rows r that the token sees,
 *   s_r = scale q . row_r[:d_qk],  o = sum e^(s_r - m) row_r[:d_v] / (sum e^(s_r
 *   - m) + e^(sink - m)),
 * in one pass over the cache with the running maximum m and sum. The rows of q
 * of all tokens and heads read the same cache, so they are cut into blocks of
 * 16 to 128 that share each tile of the cache; where the blocks do not fill
 * the card the cache is cut into splits, whose sums a second launch adds with
 * weights e^(m_split - m).
 */
#include "dsv4_tree.h"

#include <math.h>

namespace {

#include "dsv4_rows_io.h"

constexpr int TJ_THREADS = 256;
constexpr int TJ_COLS = 64;                       /* columns of a workgroup  */
constexpr int TJ_GROUPS = TJ_THREADS / (TJ_COLS / 4);
constexpr int TJ_SPLITS = 512;                    /* most splits of a call   */

/* 1 / (a row's sum with its sink), 0 where the row saw nothing. */
__device__ __forceinline__ float join_scale(const Dsv4TreeJob &a, int r, float m, float l)
{
    if (a.sink && l != 0.0f)
        l += __builtin_amdgcn_exp2f(a.sink[r % a.h] * 1.44269504088896340736f - m);
    return l != 0.0f ? 1.0f / l : 0.0f;
}

template <class T>
__device__ __forceinline__ void join_store(const Dsv4TreeJob &a, T *o, int r, int c, f32x4 v)
{
    if (c >= a.dv) return;
    const float y[4] = {v.x, v.y, v.z, v.w};
    T *d = o + (size_t)r * a.dv + c;
    if (a.ovec) {
        io_store<T, 4>(d, y);
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (c + e < a.dv) io_store<T, 1>(d + e, y + e);
    }
}

/* o of one row of q and 64 columns: thread (group of splits, 4 columns), the
 * groups' sums added in order through LDS. Each wave weighs all splits for
 * itself, and the first 64 splits' sums are on their way meanwhile. */
template <class T>
__global__ void __launch_bounds__(TJ_THREADS) k_tree_join(Dsv4TreeJob a, T *o)
{
    constexpr int NK = TJ_SPLITS / 64, NI = 64 / TJ_GROUPS;
    __shared__ f32x4 sum[TJ_GROUPS][TJ_COLS / 4];
    const int tid = threadIdx.x, lane = tid & 63, r = blockIdx.x, R = a.nt * a.h;
    const int c4 = tid & (TJ_COLS / 4 - 1), gr = tid / (TJ_COLS / 4);
    const int c = blockIdx.y * TJ_COLS + 4 * c4;
    auto part = [&](int s) {
        return s < a.ns && c < a.dvp ? ldf4(a.part + ((size_t)s * R + r) * a.dvp + c)
                                     : f32x4{0.f, 0.f, 0.f, 0.f};
    };
    float ms[NK], ls[NK], m = -INFINITY;
#pragma unroll
    for (int k = 0; k < NK; k++) {
        const int s = 64 * k + lane;
        ms[k] = -INFINITY;
        ls[k] = 0.0f;
        if (64 * k < a.ns && s < a.ns) {
            ms[k] = a.pm[(size_t)s * R + r];
            ls[k] = a.pl[(size_t)s * R + r];
        }
    }
    f32x4 x[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) x[i] = part(gr + TJ_GROUPS * i);
#pragma unroll
    for (int k = 0; k < NK; k++) m = fmaxf(m, ms[k]);
    m = wave_max(m);
    float l = 0.0f;
#pragma unroll
    for (int k = 0; k < NK; k++) {
        if (64 * k >= a.ns) break;
        ms[k] = tree_join_weight(ms[k], ls[k], m);
        l += ms[k] * ls[k];
    }
    l = wave_sum(l);
    f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NK; k++) {
        if (64 * k >= a.ns) break;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int s = gr + TJ_GROUPS * i;
            v += __shfl(ms[k], s, 64) * (k == 0 ? x[i] : part(64 * k + s));
        }
    }
    sum[gr][c4] = v;
    __syncthreads();
    if (gr != 0) return;
    for (int k = 1; k < TJ_GROUPS; k++) v += sum[k][c4];
    join_store(a, o, r, c, v * join_scale(a, r, m, l));
}

/* The same by one wave for a row, where the rows alone fill the card: lane s has
 * split s's weight, and each lane up to eight columns. */
template <class T>
__global__ void __launch_bounds__(TJ_THREADS) k_tree_join_rows(Dsv4TreeJob a, T *o)
{
    const int lane = threadIdx.x & 63, R = a.nt * a.h;
    const int r = blockIdx.x * (TJ_THREADS / 64) +
                  __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (r >= R) return;
    const float ms = lane < a.ns ? a.pm[(size_t)lane * R + r] : -INFINITY;
    const float ls = lane < a.ns ? a.pl[(size_t)lane * R + r] : 0.0f;
    const float m = wave_max(ms), wt = tree_join_weight(ms, ls, m);
    const float inv = join_scale(a, r, m, wave_sum(wt * ls));
    f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    const float *p = a.part + (size_t)r * a.dvp + 4 * lane;
    for (int s = 0; s < a.ns; s++, p += (size_t)R * a.dvp) {
        const float e = __shfl(wt, s, 64);
#pragma unroll
        for (int k = 0; k < 2; k++)
            if (256 * k + 4 * lane < a.dvp) v[k] += e * ldf4(p + 256 * k);
    }
#pragma unroll
    for (int k = 0; k < 2; k++) join_store(a, o, r, 256 * k + 4 * lane, v[k] * inv);
}

/* A wave for a row from 2048 rows on, eight waves a CU; the plan then leaves 32
 * splits at most. 8192 rows of 4 splits: 13.3 us, 64.8 by 64 columns a workgroup. */
template <class T>
void join_launch(const Dsv4TreeJob &a, hipStream_t st)
{
    const int R = a.nt * a.h;
    if (R >= 2048)
        hipLaunchKernelGGL(k_tree_join_rows<T>, dim3((R + TJ_THREADS / 64 - 1) / (TJ_THREADS / 64)),
                           dim3(TJ_THREADS), 0, st, a, (T *)a.o);
    else
        hipLaunchKernelGGL(k_tree_join<T>, dim3(R, (a.dv + TJ_COLS - 1) / TJ_COLS),
                           dim3(TJ_THREADS), 0, st, a, (T *)a.o);
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

struct TreePlan {
    int kc, tile0, tile1, nb, br, cap, ns, dvp;
    size_t bytes;
};

/* Rows of q of a workgroup and splits of the cache, by what a workgroup takes, in
 * halves of the time of a tile on a lone wave (0.55 us for bf16 q over 576
 * columns, 0.8 for f32 q): 2 a tile for up to four waves with rows of q and 3 for
 * eight; 8 for the start and 2 for each such wave's q and sums; 5 for the join's
 * launch and 1 for each 4 MB of its sums. A workgroup has a CU to itself but for
 * the narrowest rows, so beyond 256 they come in rounds. Few rows are thus spread over workgroups of 16
 * of them and read the cache through L2 as often, until the splits fill the
 * card; then wider ones win. Measured, one token's 64 heads of f32 q over a bf16
 * cache, at the best split for 16, 32 and 64 rows a workgroup: 16.0, 17.8 and 23.4 us
 * at 1500 rows of cache (and 14.1 with a tile a split where these had two), 21.4,
 * 23.2 and 28.7 at 8192, 41.9, 34.3 and 39.0 at 32768, 122, 77 and 74 at 131072.
 * A tile has that price at every width and format, though those of narrower rows
 * take less: such calls may take more splits than are best for them.
 * The narrowest rows with bf16 q share a CU by two workgroups, whose tiles then
 * take 1.6 times as long each (1920 rows over 65536 of 128 FP8: 139 us in 256
 * workgroups of 128 rows, 110 in 512). */
TreePlan tree_plan(int fmt, int nt, int h, int d_qk, int d_v, int kv_fmt, int n_ctx, int window)
{
    TreePlan p;
    p.kc = dsv4_tree_chunks(d_qk, d_v);
    const int lo = window && n_ctx >= window ? n_ctx - window + 1 : 0;
    p.tile0 = lo / TR_TILE;
    p.tile1 = (n_ctx + nt + TR_TILE - 1) / TR_TILE;
    const int tiles = p.tile1 - p.tile0, br = dsv4_tree_block_rows(fmt, kv_fmt, p.kc);
    const int wide = (nt * h + br - 1) / br;
    p.dvp = (d_v + 15) / 16 * 16;
    /* the most tiles that any context up to this length can have: the tiles of this
     * one go up and down by one as its window's start passes a tile's edge */
    const long long most = window ? ((long long)window + nt) / TR_TILE + 2 : p.tile1;
    const int up = p.tile1 < most ? p.tile1 : (int)most;
    p.cap = up < TJ_SPLITS / wide ? up : TJ_SPLITS / wide;
    if (p.cap < 1) p.cap = 1;
    long long best = -1;
    for (int r = 16; r <= br; r *= 2) {
        const int nb = (nt * h + r - 1) / r, waves = r / 16 * tree_split(fmt, kv_fmt, p.kc);
        for (int k = 0; k < 5; k++) {             /* one split, or k rounds and more */
            long long ns = k ? 256ll * ((nb + 255) / 256 + k - 1) / nb : 1;
            if (ns > p.cap) ns = p.cap;
            if (ns > tiles) ns = tiles;
            const long long each = (tiles + ns - 1) / ns;
            ns = (tiles + each - 1) / each;
            /* rounds in fifths: two that share the CUs take eight */
            const long long full = (nb * ns + 255) / 256;
            const long long fifths = tree_per_cu(fmt, p.kc) == 2 ? full / 2 * 8 + full % 2 * 5
                                                                 : full * 5;
            const long long cost = fifths * (each * (waves > 4 ? 3 : 2) + 8 + 2 * waves) / 5 +
                                   (ns > 1 ? 5 + ((ns * nt * h * p.dvp) >> 20) : 0);
            if (best >= 0 && cost >= best) continue;
            best = cost;
            p.br = r;
            p.nb = nb;
            p.ns = (int)ns;
        }
    }
    /* the workspace: not what this plan writes, whose splits fall in steps as the
     * rows of q grow, but the least that holds it and never falls with a size */
    const long long all = (long long)(up < TJ_SPLITS ? up : TJ_SPLITS) * nt * h;
    const long long most_rows = (long long)TJ_SPLITS * br;
    p.bytes = up > 1 ? (size_t)(all < most_rows ? all : most_rows) * (p.dvp + 2) * sizeof(float)
                     : 0;
    return p;
}

} // namespace

int dsv4_tree_chunks(int d_qk, int d_v)
{
    if (d_qk <= 128) return 4;
    if (d_qk <= 256) return 8;
    return d_qk <= 512 ? 16 : 18;
}

int dsv4_tree_block_rows(int fmt, int kv_fmt, int kc)
{
    return 16 * TR_WAVES / tree_split(fmt, kv_fmt, kc);
}

extern "C" size_t dsv4_gpu_tree_attn_scratch_bytes(int fmt, int nt, int h, int d_qk, int d_v,
                                                   int kv_fmt, int n_ctx, int window)
{
    if (nt == 0 || tree_bad(fmt, nt, h, d_qk, d_v, kv_fmt, n_ctx, window)) return 0;
    return tree_plan(fmt, nt, h, d_qk, d_v, kv_fmt, n_ctx, window).bytes;
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
    const TreePlan p = tree_plan(fmt, nt, h, d_qk, d_v, kv_fmt, n_ctx, window);
    if (p.ns > 1 && (!d_scratch || ((uintptr_t)d_scratch & 15) || scratch_bytes < p.bytes)) {
        DSV4_ERR("tree_attn: %zu bytes of workspace at %p; the call needs %zu, 16-byte aligned",
                 scratch_bytes, d_scratch, p.bytes);
        return -1;
    }
    const IoDiv pd((uint32_t)(d_pages ? page_rows : 1));
    const int es = fmt == DSV4_WBF16 ? 2 : 4;
    Dsv4TreeJob a{};
    a.o = d_o;
    a.q = d_q;
    a.nt = nt;
    a.h = h;
    a.dqk = d_qk;
    a.dv = d_v;
    a.kv = d_kv;
    a.ks = d_kv_scales;
    a.stride = kv_stride;
    a.rows = kv_rows;
    a.pages = d_pages;
    a.n_pages = n_pages;
    a.page = page_rows;
    a.page_m = pd.m;
    a.page_s = pd.s;
    a.ctx = n_ctx;
    a.mask = d_mask;
    a.window = window;
    a.sink = d_sink;
    a.scale = scale;
    a.tile0 = p.tile0;
    a.tile1 = p.tile1;
    a.ns = p.ns;
    a.nb = p.nb;
    a.br = p.br;
    a.dvp = p.dvp;
    a.part = (float *)d_scratch;
    a.pm = a.part + (size_t)p.ns * nt * h * p.dvp;
    a.pl = a.pm + (size_t)p.ns * nt * h;
    a.vec = d_qk % 8 == 0 && kv_stride % 8 == 0 && ((uintptr_t)d_kv & 15) == 0;
    a.qvec = d_qk % 8 == 0 && ((uintptr_t)d_q & 15) == 0;
    a.ovec = d_v % 4 == 0 && (uintptr_t)d_o % (4 * es) == 0;
    hipStream_t st = (hipStream_t)stream;
    const int rc = kv_fmt == DSV4_GPU_KV_F32    ? dsv4_tree_f32_launch(a, fmt, p.kc, st)
                 : kv_fmt == DSV4_GPU_KV_BF16 ? dsv4_tree_bf16_launch(a, fmt, p.kc, st)
                                              : dsv4_tree_fp8_launch(a, fmt, p.kc, st);
    if (rc != 0 || p.ns == 1) return rc;
    if (fmt == DSV4_WF32) join_launch<float>(a, st);
    else join_launch<uint16_t>(a, st);
    HIP_OK(hipGetLastError(), "tree attn join launch");
    return 0;
}
