/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_tree.h - the attention of drafted tokens over a latent cache: the job
 * that dsv4_tree.hip plans, and the kernel, instantiated per cache format in
 * dsv4_tree_f32.hip, dsv4_tree_bf16.hip and dsv4_tree_fp8.hip. */
#pragma once

#include "dsv4_dev.h"
#include "dsv4_internal.h"

constexpr int TR_THREADS = 256;
constexpr int TR_WAVES = TR_THREADS / 64;
constexpr int TR_TILE = 32;                       /* cache rows of a step    */
constexpr int TR_DQK = 576, TR_DV = 512;

struct Dsv4TreeJob {
    void *o;
    const void *q;
    int nt, h, dqk, dv;
    const void *kv;
    const float *ks;
    int stride, rows;
    const int *pages;
    int n_pages, page;
    uint32_t page_m, page_s;                      /* division by page        */
    int ctx;
    const uint64_t *mask;
    int window;
    const float *sink;
    float scale;
    /* set by the plan: tiles [tile0, tile1) in ns splits of the rows of q's nb
     * blocks; part [ns][nt h][dvp] and its maxima and sums [ns][nt h] */
    int tile0, tile1, ns, nb, dvp;
    float *part, *pm, *pl;
    int vec, qvec, ovec;                          /* whole pieces            */
};

/* The width class of a call (32-element chunks of d_qk that the kernel holds),
 * the rows of q that one workgroup takes and its launch; 0 / -1. */
int dsv4_tree_chunks(int d_qk, int d_v);
int dsv4_tree_block_rows(int fmt, int kv_fmt, int kc);
int dsv4_tree_f32_launch(const Dsv4TreeJob &a, int fmt, int kc, hipStream_t st);
int dsv4_tree_bf16_launch(const Dsv4TreeJob &a, int fmt, int kc, hipStream_t st);
int dsv4_tree_fp8_launch(const Dsv4TreeJob &a, int fmt, int kc, hipStream_t st);

/* bf16 terms that carry an f32 value exactly. */
constexpr int TR_TERMS = 3;
constexpr int tree_terms(int fmt) { return fmt == DSV4_WF32 ? TR_TERMS : 1; }
constexpr int tree_planes(int kv_fmt) { return kv_fmt == DSV4_GPU_KV_F32 ? TR_TERMS : 1; }
constexpr int tree_vtiles(int kc) { return kc >= 16 ? 32 : 2 * kc; }
/* Blocks of 16 rows of q per wave. A wave reads every row of a tile from LDS
 * for each of its blocks' products: with one term of q two blocks share the
 * read, with three the terms do. */
constexpr int tree_qblocks(int fmt, int kv_fmt, int kc)
{
    return tree_terms(fmt) * tree_planes(kv_fmt) == 1 && kc <= 4 ? 2 : 1;
}

#ifdef DSV4_TREE_KERNEL

namespace {

#include "dsv4_rows_io.h"

typedef __bf16 tr_bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 tr_bf2 __attribute__((ext_vector_type(2)));
typedef short tr_s4 __attribute__((ext_vector_type(4)));
typedef short tr_s8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) tr_s4 tr_lds_s4;

/* Eight f32 -> N bf16 vectors whose sum is the values: exactly with three (a
 * residual of a rounding to 8 bits has 16 left, then 8), rounded once with
 * one. */
template <int N>
__device__ __forceinline__ void tr_terms(const float *v, tr_bf8 *t)
{
    u32x4 w[N];
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = v[i];
#pragma unroll
    for (int n = 0; n < N; n++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t b = io_bf2(r[2 * i], r[2 * i + 1]);
            w[n][i] = b;
            r[2 * i] -= __uint_as_float(b << 16);
            r[2 * i + 1] -= __uint_as_float(b & 0xFFFF0000u);
        }
        t[n] = __builtin_bit_cast(tr_bf8, w[n]);
    }
}

__device__ __forceinline__ f32x4 tr_mfma(tr_bf8 a, tr_bf8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

/* LDS of a workgroup: NBUF tiles of [planes][TR_TILE][pitch] bytes, then per
 * buffer the rows' scales and two words of row bits. */
template <int KVF, int KC>
struct TreeLds {
    static constexpr int KT = tree_planes(KVF);
    static constexpr int PITCH = KC * 64 + 16;        /* + 16: spreads the banks */
    static constexpr int PLANE = TR_TILE * PITCH;
    static constexpr int NBUF = KT == 1 ? 2 : 1;
    static constexpr int META = NBUF * KT * PLANE;
    static constexpr int MSIZE = TR_TILE * 4 + 16;
    static constexpr int BYTES = META + NBUF * MSIZE;
};

/* Workgroup (split, block of q's rows): wave w holds 16 QB rows of q as the
 * B operands of S^T = K Q^T (a row of q per column), in bf16 terms.
 *
 * Per tile of 32 cache rows: S^T for two tiles of 16 keys; a lane then has
 * eight scores of its own column's row of q, which become that column's
 * weights; those eight, in the order they lie in, are the K slots 8 g .. 8 g +
 * 7 of the B operand of O^T = V^T P^T when V^T's slots name the same keys (rows
 * 4 g + j and 16 + 4 g + j of the tile), so the weights never leave their
 * lane. V is the same LDS tile read transposed (ds_read_b64_tr_b16). The sums
 * O^T stay in registers, the row's maximum and sum in the row's lanes; the
 * maximum follows only when it grows by 2^8, as the weights may be that much
 * over 1 without loss.
 *
 * The next tile's rows are loaded into registers while this one is used. A
 * tile with drafts, a window's edge or rows outside the cache is masked by a
 * word of 32 bits per row of q; in such a tile a cache row that holds NaN or
 * infinity is stored as zeros, which a weight of 0 leaves at 0, and gives NaN
 * scores to the rows of q that see it. */
template <class T, int KVF, int KC>
__global__ void __launch_bounds__(TR_THREADS, KC >= 16 ? 1 : 2)
k_tree(Dsv4TreeJob a)
{
    using L = TreeLds<KVF, KC>;
    constexpr int FMT = sizeof(T) == 2 ? DSV4_WBF16 : DSV4_WF32;
    constexpr int NT = tree_terms(FMT), KT = L::KT, NV = tree_vtiles(KC);
    constexpr int QB = tree_qblocks(FMT, KVF, KC);
    constexpr int NP = KC / 2;                         /* pieces of 8 per thread */
    constexpr int PT = NT > KT ? NT : KT;              /* term pairs i + j < PT  */
    constexpr int RAW = KVF == DSV4_GPU_KV_F32 ? 8 : KVF == DSV4_GPU_KV_BF16 ? 4 : 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, g = lane >> 4;

    /* Workgroup i runs on XCD i mod 8: each XCD takes a run of (split, block)
     * in split order, so blocks that read the same rows share its L2. */
    int split, blk;
    {
        const int all = gridDim.x, id = blockIdx.x, k = id & 7;
        const int at = k * (all >> 3) + min(k, all & 7) + (id >> 3);
        split = at / a.nb;
        blk = at - split * a.nb;
    }
    const int tiles = a.tile1 - a.tile0;
    const int i0 = a.tile0 + (int)((long long)tiles * split / a.ns);
    const int i1 = a.tile0 + (int)((long long)tiles * (split + 1) / a.ns);
    const int R = a.nt * a.h;

    /* this lane's rows of q: their tokens' drafts and first positions */
    int rq[QB], lo[QB];
    unsigned long long see[QB];
    tr_bf8 q[QB][NT][KC];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        rq[b] = ((blk * TR_WAVES + w) * QB + b) * 16 + l16;
        const int r = min(rq[b], R - 1), t = r / a.h;
        const unsigned long long all = a.nt >= 64 ? ~0ull : (1ull << a.nt) - 1;
        const unsigned long long own = a.mask ? a.mask[t] : (t >= 63 ? ~0ull : (2ull << t) - 1);
        const int depth = __popcll(own & all & ~(1ull << t));
        see[b] = own & all;
        lo[b] = a.window ? max(0, a.ctx + depth - a.window + 1) : 0;
        if (a.window && a.window < a.nt)
            for (int j = 0; j < a.nt; j++) {
                const unsigned long long oj = a.mask ? a.mask[j] : (2ull << j) - 1;
                if (depth - __popcll(oj & all & ~(1ull << j)) >= a.window) see[b] &= ~(1ull << j);
            }
    }
    /* elements past the row are zeroed by a mask in a register: the many lane
     * masks of comparisons would crowd out the scalar registers */
#pragma unroll
    for (int kc = 0; kc < KC; kc++)
#pragma unroll
        for (int b = 0; b < QB; b++) {
            const T *qr = (const T *)a.q + (size_t)min(rq[b], R - 1) * a.dqk;
            const int c = 32 * kc + 8 * g;
            float v[8];
            if (a.qvec) {
                io_load<T, 8>(qr + min(c, a.dqk - 8), v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) io_load<T, 1>(qr + min(c + e, a.dqk - 1), v + e);
            }
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = __int_as_float(__float_as_int(v[e]) & ((c + e - a.dqk) >> 31));
            tr_bf8 tm[NT];
            tr_terms<NT>(v, tm);
#pragma unroll
            for (int n = 0; n < NT; n++) q[b][n][kc] = tm[n];
            __builtin_amdgcn_sched_barrier(0);     /* few of q's loads at a time */
        }
    f32x4 o[QB][NV];
    float m[QB], l[QB];
#pragma unroll
    for (int b = 0; b < QB; b++) {
        m[b] = -INFINITY;
        l[b] = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; v++) o[b][v] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    /* ---- staging: thread tid has row tid / 8 of a tile and its pieces tid % 8
     *      + 8 i ---- */
    const int sr = tid >> 3, sp = tid & 7;
    const int end = a.ctx + a.nt;
    /* the cache row of tile i's row, -1 where there is none */
    auto find = [&](int i) -> int {
        const int p = i * TR_TILE + sr;
        if (p >= end || i >= i1) return -1;
        if (!a.pages) return p < a.rows ? p : -1;
        const int k = (int)((__umulhi(a.page_m, (uint32_t)p) + (uint32_t)p) >> a.page_s);
        if (k >= a.n_pages) return -1;
        const long long r = (long long)a.pages[k] * a.page + (p - k * a.page);
        return r >= 0 && r < a.rows ? (int)r : -1;
    };
    /* Pieces past the row repeat its last one: q is zero there. */
    uint32_t raw[NP][RAW];
    float rks = 1.0f;
    auto fetch = [&](int row) {
        const size_t at = (size_t)max(row, 0) * a.stride;
        if (KVF == DSV4_GPU_KV_FP8) rks = a.ks[max(row, 0)];
        if (!a.vec) return;
        constexpr int ES = KVF == DSV4_GPU_KV_F32 ? 4 : KVF == DSV4_GPU_KV_BF16 ? 2 : 1;
        const unsigned char *p = (const unsigned char *)a.kv + at * ES;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int c = min(8 * (sp + 8 * i), a.dqk - 8);
            if constexpr (ES == 1) {
                const uint2 v = *(const uint2 *)(p + c);
                raw[i][0] = v.x;
                raw[i][1] = v.y;
            } else {
#pragma unroll
                for (int k = 0; k < RAW; k += 4) {
                    const u32x4 v = ld16(p + c * ES + 4 * k);
#pragma unroll
                    for (int e = 0; e < 4; e++) raw[i][k + e] = v[e];
                }
            }
        }
    };
    /* the same for one piece of a row that is not in whole pieces */
    auto fetch1 = [&](int row, int i, uint32_t *r) {
        const size_t at = (size_t)max(row, 0) * a.stride;
#pragma unroll
        for (int k = 0; k < RAW; k++) r[k] = 0u;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const size_t c = at + min(8 * (sp + 8 * i) + e, a.dqk - 1);
            if constexpr (KVF == DSV4_GPU_KV_F32) r[e] = ((const uint32_t *)a.kv)[c];
            else if constexpr (KVF == DSV4_GPU_KV_BF16)
                r[e / 2] |= (uint32_t)((const uint16_t *)a.kv)[c] << (16 * (e & 1));
            else r[e / 4] |= (uint32_t)((const uint8_t *)a.kv)[c] << (8 * (e & 3));
        }
    };
    auto wild = [&](const uint32_t *r) {
        bool bad = false;
#pragma unroll
        for (int k = 0; k < RAW; k++) {
            if constexpr (KVF == DSV4_GPU_KV_F32) {
                bad |= (r[k] & 0x7F800000u) == 0x7F800000u;
            } else if constexpr (KVF == DSV4_GPU_KV_BF16) {
                bad |= (r[k] & 0x7F80u) == 0x7F80u || (r[k] & 0x7F800000u) == 0x7F800000u;
            } else {
#pragma unroll
                for (int e = 0; e < 32; e += 8) bad |= (r[k] >> e & 0x7Fu) == 0x7Fu;
            }
        }
        return bad;
    };
    auto put = [&](unsigned char *d, const uint32_t *r, bool zero) {
        if constexpr (KVF == DSV4_GPU_KV_F32) {
            float v[8];
            tr_bf8 tm[KT];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = zero ? 0.0f : __uint_as_float(r[e]);
            tr_terms<KT>(v, tm);
#pragma unroll
            for (int n = 0; n < KT; n++) *(tr_bf8 *)(d + n * L::PLANE) = tm[n];
        } else {
            u32x4 v;
            if constexpr (KVF == DSV4_GPU_KV_BF16) {
                v = u32x4{r[0], r[1], r[2], r[3]};
            } else {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    v[2 * e] = __builtin_bit_cast(uint32_t,
                        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[e], 1.0f, false));
                    v[2 * e + 1] = __builtin_bit_cast(uint32_t,
                        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[e], 1.0f, true));
                }
            }
            *(u32x4 *)d = zero ? u32x4{0u, 0u, 0u, 0u} : v;
        }
    };
    /* some row of q may not see some row of tile i */
    auto partial = [&](int i) {
        return (i + 1) * TR_TILE > a.ctx ||
               (a.window && i * TR_TILE < a.ctx + a.nt - a.window);
    };
    auto store = [&](int i, int row, int buf) {
        unsigned char *t = lds + (size_t)buf * KT * L::PLANE + sr * L::PITCH;
        bool bad = false;
        if (partial(i)) {
            if (a.vec) {
#pragma unroll
                for (int k = 0; k < NP; k++) bad |= wild(raw[k]);
            } else {
#pragma unroll 1
                for (int k = 0; k < NP; k++) {
                    uint32_t r[RAW];
                    fetch1(row, k, r);
                    bad |= wild(r);
                }
            }
            if (KVF == DSV4_GPU_KV_FP8)
                bad |= (__float_as_uint(rks) & 0x7F800000u) == 0x7F800000u;
        }
        /* the eight threads of a row, rows 8 w .. 8 w + 7 of the tile */
        const unsigned long long vb = __ballot(bad), vr = __ballot(row >= 0);
        bad = (vb >> (lane & 56) & 0xFFull) != 0;
        unsigned char *meta = lds + L::META + buf * L::MSIZE;
        if (lane == 0) {
            uint32_t ok = 0, no = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                ok |= (uint32_t)(vr >> (8 * k) & 1) << k;
                no |= (uint32_t)((vb >> (8 * k) & 0xFFull) != 0) << k;
            }
            meta[TR_TILE * 4 + w] = (unsigned char)ok;
            meta[TR_TILE * 4 + 4 + w] = (unsigned char)(no & ok);
        }
        if (KVF == DSV4_GPU_KV_FP8 && sp == 0) ((float *)meta)[sr] = bad || row < 0 ? 0.0f : rks;
        const bool zero = bad || row < 0;
        if (a.vec) {
#pragma unroll
            for (int k = 0; k < NP; k++) put(t + 16 * (sp + 8 * k), raw[k], zero);
        } else {
#pragma unroll 1
            for (int k = 0; k < NP; k++) {
                uint32_t r[RAW];
                fetch1(row, k, r);
                put(t + 16 * (sp + 8 * k), r, zero);
            }
        }
    };

    const float c2 = a.scale * 1.44269504088896340736f;       /* to powers of two */
    auto use = [&](int i, int buf) {
        const unsigned char *t = lds + (size_t)buf * KT * L::PLANE;
        const unsigned char *meta = lds + L::META + buf * L::MSIZE;
        /* one sum per order of the terms: the small ones do not round at the
         * size of the large */
        f32x4 s[QB][2], so[QB][2][PT];
#pragma unroll
        for (int b = 0; b < QB; b++)
#pragma unroll
            for (int n = 0; n < PT; n++) so[b][0][n] = so[b][1][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kc = 0; kc < KC; kc++) {
#pragma unroll
            for (int p = 0; p < KT; p++)
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const tr_bf8 row = *(const tr_bf8 *)(t + p * L::PLANE +
                                                         (16 * k + l16) * L::PITCH + 64 * kc +
                                                         16 * g);
#pragma unroll
                    for (int n = 0; n < NT; n++)
                        if (n + p < PT)
#pragma unroll
                            for (int b = 0; b < QB; b++)
                                so[b][k][n + p] = tr_mfma(row, q[b][n][kc], so[b][k][n + p]);
                }
        }
#pragma unroll
        for (int b = 0; b < QB; b++)
#pragma unroll
            for (int k = 0; k < 2; k++) {
                s[b][k] = so[b][k][PT - 1];
#pragma unroll
                for (int n = PT - 2; n >= 0; n--) s[b][k] += so[b][k][n];
            }
        const uint32_t ok = *(const uint32_t *)(meta + TR_TILE * 4);
        const bool masked = partial(i) || ok != 0xFFFFFFFFu;
        f32x4 ks[2];
        if (KVF == DSV4_GPU_KV_FP8) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                ks[k] = *(const f32x4 *)(meta + 4 * (16 * k + 4 * g));
#pragma unroll
                for (int b = 0; b < QB; b++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[b][k][j] *= ks[k][j];
            }
        }
        uint32_t vis[QB];
#pragma unroll
        for (int b = 0; b < QB; b++) vis[b] = ~0u;
        if (masked) {
            const uint32_t no = *(const uint32_t *)(meta + TR_TILE * 4 + 4);
            const int p0 = i * TR_TILE;
#pragma unroll
            for (int b = 0; b < QB; b++) {
                /* positions [lo, ctx) of the context, then the drafts' bits */
                vis[b] = 0u;
                const int f = max(lo[b] - p0, 0), e = min(a.ctx - p0, TR_TILE);
                if (f < e) vis[b] = (e >= 32 ? ~0u : (1u << e) - 1u) & ~((1u << f) - 1u);
                const int d = p0 - a.ctx;
                if (d > -TR_TILE && d < 64)
                    vis[b] |= d >= 0 ? (uint32_t)(see[b] >> d) : (uint32_t)(see[b] << -d);
                vis[b] &= ok;
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (no >> (16 * k + 4 * g + j) & 1u)
                            s[b][k][j] = __uint_as_float(0x7FC00000u);
            }
        }
        tr_bf8 pw[QB][PT];
#pragma unroll
        for (int b = 0; b < QB; b++) {
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float x = s[b][k][j] * c2;
                    if (masked) x = vis[b] >> (16 * k + 4 * g + j) & 1u ? x : -INFINITY;
                    top = fmaxf(top, x);
                }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const bool grow = top > m[b] + 8.0f;
            if (__any(grow)) {
                const float f = grow ? __builtin_amdgcn_exp2f(m[b] - top) : 1.0f;
                m[b] = grow ? top : m[b];
                l[b] *= f;
#pragma unroll
                for (int v = 0; v < NV; v++) o[b][v] *= f;
            }
            const float mm = m[b] == -INFINITY ? 0.0f : m[b];
            float e[8], sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float x = __builtin_amdgcn_exp2f(fmaf(s[b][k][j], c2, -mm));
                    if (masked) x = vis[b] >> (16 * k + 4 * g + j) & 1u ? x : 0.0f;
                    sum += x;
                    e[4 * k + j] = KVF == DSV4_GPU_KV_FP8 ? x * ks[k][j] : x;
                }
            l[b] += sum;
            tr_terms<NT>(e, pw[b]);
        }
#pragma unroll
        for (int v = 0; v < NV; v++) {
#pragma unroll
            for (int p = 0; p < KT; p++) {
                const unsigned char *at = t + p * L::PLANE + (4 * g + (l16 >> 2)) * L::PITCH +
                                          2 * (16 * v + 4 * (l16 & 3));
                const tr_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_lds_s4 *)at);
                const tr_s4 y =
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_lds_s4 *)(at + 16 * L::PITCH));
                const tr_bf8 col = __builtin_bit_cast(
                    tr_bf8, (tr_s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int n = 0; n < NT; n++)
                    if (n + p < PT)
#pragma unroll
                        for (int b = 0; b < QB; b++) o[b][v] = tr_mfma(col, pw[b][n], o[b][v]);
            }
        }
    };

    if (i0 < i1) {
        int row = find(i0), next = find(i0 + 1);
        fetch(row);
        store(i0, row, 0);
        __syncthreads();
        for (int i = i0; i < i1; i++) {
            const int buf = L::NBUF == 2 ? (i - i0) & 1 : 0;
            const bool more = i + 1 < i1;
            row = next;
            if (more) {
                fetch(row);
                next = find(i + 2);
            }
            use(i, buf);
            if (more) {
                if (L::NBUF == 1) __syncthreads();
                store(i + 1, row, L::NBUF == 2 ? buf ^ 1 : 0);
                __syncthreads();
            }
        }
    }

    /* ---- the split's sums, or the result ---- */
#pragma unroll
    for (int b = 0; b < QB; b++) {
        l[b] += __shfl_xor(l[b], 16, 64);
        l[b] += __shfl_xor(l[b], 32, 64);
        if (rq[b] >= R) continue;
        if (a.ns > 1) {
            const size_t at = (size_t)split * R + rq[b];
            if (g == 0) {
                a.pm[at] = m[b];
                a.pl[at] = l[b];
            }
            float *d = a.part + at * a.dvp + 4 * g;
#pragma unroll
            for (int v = 0; v < NV; v++)
                if (16 * v < a.dvp) *(f32x4 *)(d + 16 * v) = o[b][v];
            continue;
        }
        float den = l[b];
        if (a.sink && den != 0.0f)
            den += __builtin_amdgcn_exp2f(a.sink[rq[b] % a.h] * 1.44269504088896340736f - m[b]);
        const float inv = den != 0.0f ? 1.0f / den : 0.0f;
        T *d = (T *)a.o + (size_t)rq[b] * a.dv + 4 * g;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const f32x4 x = o[b][v] * inv;
            const float y[4] = {x.x, x.y, x.z, x.w};
            const int c = 16 * v + 4 * g;
            if (a.ovec) {
                if (c < a.dv) io_store<T, 4>(d + 16 * v, y);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (c + e < a.dv) io_store<T, 1>(d + 16 * v + e, y + e);
            }
        }
    }
}

template <class T, int KVF, int KC>
int tree_launch(const Dsv4TreeJob &a, hipStream_t st)
{
    using L = TreeLds<KVF, KC>;
    if (L::BYTES > 64 * 1024) {
        /* once per device, as the attribute is the device's */
        static bool asked[64];
        int dev = 0;
        HIP_OK(hipGetDevice(&dev), "hipGetDevice");
        if (dev < 0 || dev >= 64 || !asked[dev]) {
            (void)dsv4_lds_optin((const void *)k_tree<T, KVF, KC>, L::BYTES, "tree attention");
            if (dev >= 0 && dev < 64) asked[dev] = true;
        }
    }
    hipLaunchKernelGGL((k_tree<T, KVF, KC>), dim3((unsigned)(a.ns * a.nb)), dim3(TR_THREADS),
                       L::BYTES, st, a);
    HIP_OK(hipGetLastError(), "tree attn launch");
    return 0;
}

template <class T, int KVF>
int tree_width(const Dsv4TreeJob &a, int kc, hipStream_t st)
{
    switch (kc) {
    case 4: return tree_launch<T, KVF, 4>(a, st);
    case 8: return tree_launch<T, KVF, 8>(a, st);
    case 16: return tree_launch<T, KVF, 16>(a, st);
    default: return tree_launch<T, KVF, 18>(a, st);
    }
}

template <int KVF>
int tree_format(const Dsv4TreeJob &a, int fmt, int kc, hipStream_t st)
{
    return fmt == DSV4_WF32 ? tree_width<float, KVF>(a, kc, st)
                            : tree_width<uint16_t, KVF>(a, kc, st);
}

} // namespace

#endif
