/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_tree.h - the attention of drafted tokens over a latent cache: the job
 * that dsv4_tree.hip plans, and the kernel, instantiated per cache format in
 * dsv4_tree_f32.hip, dsv4_tree_bf16.hip and dsv4_tree_fp8.hip. */
#pragma once

#include "dsv4_dev.h"
#include "dsv4_internal.h"

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
    int tile0, tile1, ns, nb, br, dvp;
    float *part, *pm, *pl;
    int vec, qvec, ovec;                          /* the bf16 cache, q and o: whole
                                                   * and aligned pieces of 8, 8, 4 */
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
/* bf16 q's weights in one, as a second would double the second product's matrix
 * instructions for an error that is at most the output's own rounding. */
constexpr int tree_terms(int fmt) { return fmt == DSV4_WF32 ? TR_TERMS : 1; }
/* An F32 cache's elements in as many for f32 q, and in two, to 2^-17 of each, for
 * bf16 q, whose weights are rounded to 2^-8 (2048 rows of q over 16384 of 512: 195
 * us, 265 with three). */
constexpr int tree_planes(int fmt, int kv_fmt)
{
    return kv_fmt != DSV4_GPU_KV_F32 ? 1 : fmt == DSV4_WF32 ? TR_TERMS : 2;
}
constexpr int tree_vtiles(int kc) { return kc >= 16 ? 32 : 2 * kc; }
/* A workgroup is eight waves, two per SIMD. A wave holds 16 rows of q and their
 * sums, or, where with all terms that is more than half the registers, two
 * waves share 16 rows: each takes half of the d_qk columns of the scores, adds
 * the other's half through LDS, and sums half of the d_v columns. */
constexpr int TR_WAVES = 8;
constexpr int tree_split(int fmt, int kv_fmt, int kc)
{
    return kc >= 16 && tree_terms(fmt) * tree_planes(fmt, kv_fmt) > 1 ? 2 : 1;
}

/* Workgroups that a CU holds: two of the narrowest rows with bf16 q, whose waves
 * need no more than 128 registers (f32 q spills in so few and is slower: 1920
 * rows over 65536 of 128 bf16 188 us, and 207 so). */
constexpr int tree_per_cu(int fmt, int kc) { return fmt == DSV4_WBF16 && kc == 4 ? 2 : 1; }

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

/* The sum of eight f32, each rounded to bf16 (v_dot2_f32_bf16 with ones, of the pairs
 * as they are rounded: of the words of a vector of eight this compiler takes the
 * first four times). */
__device__ __forceinline__ float tr_sum8(const float *v)
{
    const tr_bf2 one = __builtin_bit_cast(tr_bf2, 0x3F803F80u);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        s = __builtin_amdgcn_fdot2_f32_bf16(
            __builtin_bit_cast(tr_bf2, io_bf2(v[i], v[i + 1])), one, s, false);
    return s;
}

__device__ __forceinline__ f32x4 tr_mfma(tr_bf8 a, tr_bf8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

/* LDS of a workgroup: NBUF tiles of [planes][slabs of 64 columns][TR_TILE][128
 * bytes], then per buffer the rows' scales and whether they may not be used,
 * then what q's rows see (kept out of the registers, as only masked tiles ask)
 * and the halves of scores. Piece p (16 bytes) of a slab's row r is at p ^ (r &
 * 7). Then the reads of the scores (eight rows' same piece at a time) and of
 * the values (two pieces of rows 0 .. 7, even and odd ones in different halves
 * of the 64 banks) take each bank once: SQ_LDS_BANK_CONFLICT counts none, and 4
 * cycles for each read of the values with p ^ (0, 2, 4, 6, 1, 3, 5, 7). */
template <int KVF, int KC, int SPLIT, int PLANES>
struct TreeLds {
    static constexpr int KT = PLANES;
    static constexpr int SLABS = KC / 2;
    static constexpr int SLAB = TR_TILE * 128;
    static constexpr int PLANE = SLABS * SLAB;
    static constexpr int NBUF = KT * KC > 32 || KT > 2 ? 1 : KVF == DSV4_GPU_KV_BF16 ? 3 : 2;
    static constexpr int META = NBUF * KT * PLANE;
    static constexpr int MSIZE = 2 * TR_TILE * 4;
    static constexpr int ROWS = META + NBUF * MSIZE;   /* q's rows: see, lo      */
    static constexpr int HALF = ROWS + 16 * 16 * TR_WAVES;
    static constexpr int BYTES = HALF + (SPLIT == 2 ? 2048 * TR_WAVES : 0);
    static_assert(BYTES <= 160 * 1024, "a CU's LDS");
};

__device__ __forceinline__ int tr_swz(int r) { return r & 7; }

template <int N>
__device__ __forceinline__ void tr_vm_wait()
{
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

/* 16 bytes per lane from p to LDS byte dst + 16 lane (dst the same in every
 * lane). As the builtin the compiler would wait for it before each later
 * transposed read of LDS; this way nothing waits but tr_vm_wait. Its addresses
 * are read as it issues, and it writes no register but M0. That cannot be named as
 * clobbered; k_tree has no other use of it (no LDS-direct builtin, no indexed
 * register, no message), as its assembly shows, and must not get one. */
__device__ __forceinline__ void tr_to_lds(const void *p, uint32_t dst)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 ::"s"(dst), "v"(p) : "memory");
}

/* Every wave's LDS reads and writes so far are done; loads stay in flight. */
__device__ __forceinline__ void tr_sync()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

/* The largest of the four lanes l16, l16 + 16, + 32 and + 48, in each of them
 * (exchanges within the vector unit: no trip through LDS). */
__device__ __forceinline__ float tr_max4(float v)
{
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

/* v, so that what is computed from it in a loop is not kept across the loop. */
__device__ __forceinline__ int tr_fresh(int v)
{
    asm volatile("" : "+v"(v));
    return v;
}

template <class T>
constexpr int tr_fmt() { return sizeof(T) == 2 ? DSV4_WBF16 : DSV4_WF32; }

/* Workgroup (split, block of q's rows): a wave holds 16 rows of q (or half of
 * their columns) as the B operands of S^T = K Q^T, a row of q per column, in
 * bf16 terms.
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
 * Tiles of a bf16 cache go to LDS by global_load_lds_dwordx4, two tiles ahead
 * and through no register; the other formats' next tile is loaded into
 * registers while this one is used. Operands are read from LDS a few products
 * ahead of the matrix core. What a thread can make from its lane's number again
 * is made again (place(), tr_fresh): the registers are full of q and the sums.
 *
 * A tile with drafts, a window's edge or rows outside the cache is masked by a
 * word of 32 bits per row of q; its cache rows that hold NaN or infinity, or
 * are not there, become zeros in LDS first, which a weight of 0 leaves at 0,
 * and the former give NaN scores to the rows of q that see them.
 *
 * Bound: the matrix core where there are rows of q enough, and the start (q's
 * loads and terms, one tile's trip from HBM, about 4 us) where there are not.
 * 8192 rows of q in bf16 over 131072 cache rows in bf16 (d_qk 576, d_v 512): 2053
 * to 2290 us with the clock of the card, 1.02 to 1.14 PFLOP/s, where a library
 * product of 8192^3 reaches 1.20. Per tile and SIMD the products take 2176 cycles
 * of some 4000; the rest is the softmax's vector instructions (1000 cycles for two
 * waves) and the loads' issue, of which the other wave's products hide the most.
 * 1024 rows of f32 q over 32768 of FP8: 186 to 196 us, 1.05 to 1.11 PFLOP/s of bf16
 * terms. Waves half a tile apart, deeper reads ahead, wave priorities and loads issued between
 * products measured the same or slower; 32 rows of q a wave do not fit the
 * registers. */
template <class T, int KVF, int KC>
__global__ void __launch_bounds__(64 * TR_WAVES, TR_WAVES / 4 * tree_per_cu(tr_fmt<T>(), KC))
k_tree(Dsv4TreeJob a)
{
    constexpr int SPLIT = tree_split(tr_fmt<T>(), KVF, KC);
    using L = TreeLds<KVF, KC, SPLIT, tree_planes(tr_fmt<T>(), KVF)>;
    constexpr int NT = tree_terms(tr_fmt<T>()), KT = L::KT, NV = tree_vtiles(KC);
    constexpr int PT = NT > KT ? NT : KT;              /* term pairs i + j < PT  */
    constexpr int W = TR_WAVES, WS = W / 4;
    constexpr int KC1 = KC / SPLIT, NV1 = NV / SPLIT;  /* this wave's part       */
    constexpr int NP = (L::SLABS + WS - 1) / WS;       /* pieces of 8 per thread */
    constexpr int RAW = KVF == DSV4_GPU_KV_F32 ? 8 : 2;
    constexpr int ES = KVF == DSV4_GPU_KV_F32 ? 4 : KVF == DSV4_GPU_KV_BF16 ? 2 : 1;
    constexpr bool DMA = KVF == DSV4_GPU_KV_BF16;
    /* where the next tile and all of q are in registers, few are left: with operands
     * six ahead spills took 1052 us where two ahead take 734 (8192 rows of bf16 q over
     * 32768 of FP8); with the widest rows the scales are read twice as well (687 us,
     * and 639 so; narrower rows lose 2 % by it) */
    constexpr bool SHALLOW = NT == 1 && KVF == DSV4_GPU_KV_FP8 && KC >= 16;
    constexpr bool AGAIN = SHALLOW && KC > 16;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    const int lane0 = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int ws = w >> 2;
    const int qb = w / SPLIT, half = w % SPLIT;

    /* Workgroup i runs on XCD i mod 8: each XCD takes a run of (split, block)
     * in split order, so blocks that read the same rows share its L2. */
    int i0, i1, blk, split;
    {
        const int all = gridDim.x, id = blockIdx.x, k = id & 7;
        const int at = k * (all >> 3) + min(k, all & 7) + (id >> 3);
        split = __builtin_amdgcn_readfirstlane(at / a.nb);
        blk = at - split * a.nb;
        const int tiles = a.tile1 - a.tile0;
        i0 = a.tile0 + (int)((long long)tiles * split / a.ns);
        i1 = a.tile0 + (int)((long long)tiles * (split + 1) / a.ns);
    }
    const int R = a.nt * a.h, end = a.ctx + a.nt;
    const int row0 = blk * a.br + qb * 16;             /* this wave's rows of q  */
    const bool live = 16 * qb < a.br && row0 < R;

    /* ---- staging: a thread has place (lane % 8) of row sr of slabs ws, ws + WS,
     *      ... of a tile, which is piece (lane % 8) ^ (sr & 7) of 64 columns.
     *      Pieces past the cache row repeat its last one: q is zero there. ---- */
    struct Place {
        int sr, pc, home;                              /* pc: the piece's first column */
    };
    auto place = [&]() {
        const int ln = tr_fresh(lane0), sr = 8 * (w & 3) + (ln >> 3);
        return Place{sr, 8 * ((ln & 7) ^ tr_swz(sr)), sr * 128 + 16 * (ln & 7)};
    };
    auto slot = [&](int i) { return (int)((uint32_t)(i - i0) % (uint32_t)L::NBUF); };
    auto plane = [&](int buf) { return lds + buf * KT * L::PLANE; };
    auto meta = [&](int buf) { return lds + L::META + buf * L::MSIZE; };
    const uint32_t lds0 = (uint32_t)__builtin_amdgcn_readfirstlane(
        (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)lds);
    /* the cache row of row r of tile i, -1 where there is none */
    auto find = [&](int i, int r) -> int {
        const int p = i * TR_TILE + r;
        if (!a.pages) return p < min(end, a.rows) ? p : -1;
        if (p >= end) return -1;
        const int k = (int)((__umulhi(a.page_m, (uint32_t)p) + (uint32_t)p) >> a.page_s);
        if (k >= a.n_pages) return -1;
        const long long c = (long long)a.pages[k] * a.page + (p - k * a.page);
        return c >= 0 && c < a.rows ? (int)c : -1;
    };
    /* a page's entry is asked for a tile before it is needed: lane l has row l % 32
     * of the tile to be loaded next, and `there` says which of its rows exist */
    int ahead = -1;
    auto ask = [&](int i) {
        if (a.pages && i < i1) ahead = find(i, tr_fresh(lane0) & 31);
    };
    auto there = [&](int i) -> uint32_t {
        if (a.pages) return (uint32_t)__ballot(ahead >= 0);
        const int n = min(end, a.rows) - i * TR_TILE;
        return n >= TR_TILE ? ~0u : n > 0 ? (1u << n) - 1u : 0u;
    };
    /* (__shfl's lane number is a register that the widest rows lack with DMA, and
     * its reload would wait for all loads; the other formats measure better so) */
    auto my_row = [&](int i, const Place &h) {
        if constexpr (DMA)
            return max(0, a.pages ? __builtin_amdgcn_ds_bpermute(4 * h.sr, ahead) : find(i, h.sr));
        else
            return max(0, a.pages ? __shfl(ahead, h.sr, 64) : find(i, h.sr));
    };
    /* the eight elements from column c of a row: where they are all there, in one
     * or two loads that need no alignment (the target's own; the LDS-direct ones
     * need it), else one by one */
    auto piece = [&](size_t at, int c, uint32_t *r) {
        const unsigned char *p = (const unsigned char *)a.kv + at * ES;
        if (c + 8 <= a.dqk) {
            __builtin_memcpy(r, p + c * ES, 8 * ES);
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int k = min(c + e, a.dqk - 1);
            if constexpr (ES == 4) r[e] = ((const uint32_t *)p)[k];
            else if constexpr (ES == 2)
                r[e / 2] = (e & 1 ? r[e / 2] : 0u) | (uint32_t)((const uint16_t *)p)[k]
                                                         << (16 * (e & 1));
            else r[e / 4] = (e & 3 ? r[e / 4] : 0u) | (uint32_t)p[k] << (8 * (e & 3));
        }
    };
    auto put = [&](unsigned char *d, const uint32_t *r) {
        if constexpr (KVF == DSV4_GPU_KV_F32) {
            float v[8];
            tr_bf8 tm[KT];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __uint_as_float(r[e]);
            tr_terms<KT>(v, tm);
#pragma unroll
            for (int n = 0; n < KT; n++) *(tr_bf8 *)(d + n * L::PLANE) = tm[n];
        } else if constexpr (DMA) {
            *(u32x4 *)d = u32x4{r[0], r[1], r[2], r[3]};
        } else {
            u32x4 v;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                v[2 * e] = __builtin_bit_cast(uint32_t,
                    __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[e], 1.0f, false));
                v[2 * e + 1] = __builtin_bit_cast(uint32_t,
                    __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(r[e], 1.0f, true));
            }
            *(u32x4 *)d = v;
        }
    };
    /* the bf16 cache: tile i into LDS directly */
    auto dma = [&](int i, int buf) {
        const Place h = place();
        const int row = my_row(i, h);
        if (!a.vec) {                                  /* at once, two pieces at a time */
#pragma unroll 1
            for (int s = ws; s < L::SLABS; s += 2 * WS) {
                const int s2 = min(s + WS, L::SLABS - 1);  /* or again, the same    */
                uint32_t r[2][4];
                piece((size_t)row * a.stride, 64 * s + h.pc, r[0]);
                piece((size_t)row * a.stride, 64 * s2 + h.pc, r[1]);
                put(plane(buf) + s * L::SLAB + h.home, r[0]);
                put(plane(buf) + s2 * L::SLAB + h.home, r[1]);
            }
            return;
        }
        const uint16_t *p = (const uint16_t *)a.kv + (size_t)row * a.stride;
        const uint32_t d = lds0 + buf * L::PLANE + 1024 * (w & 3) + ws * L::SLAB;
#pragma unroll
        for (int k = 0; k < NP; k++)
            if (L::SLABS % WS == 0 || ws + WS * k < L::SLABS)
                tr_to_lds(p + min(64 * (ws + WS * k) + h.pc, a.dqk - 8), d + WS * k * L::SLAB);
    };
    /* this wave's loads but those of the newest tile are done, or all */
    auto dma_wait = [&](bool newest) {
        if (!newest) tr_vm_wait<0>();
        else if (L::SLABS % WS == 0 || ws == 0) tr_vm_wait<NP>();
        else tr_vm_wait<NP - 1>();
    };
    /* the other formats: through registers. The piece that holds the row's last
     * elements, if it is not whole, is loaded as the last eight and moved down
     * when it is stored; a row of less than eight is loaded then. */
    uint32_t raw[NP][RAW];
    float rks = 1.0f;
    int held = 0;                                      /* the short row         */
    auto fetch = [&](int i) {
        const Place h = place();
        const int row = my_row(i, h);
        if (KVF == DSV4_GPU_KV_FP8) rks = a.ks[row];
        if (KC == 4 && a.dqk < 8) {
            held = row;
            return;
        }
        const unsigned char *p = (const unsigned char *)a.kv + (size_t)row * a.stride * ES;
#pragma unroll
        for (int k = 0; k < NP; k++)
            __builtin_memcpy(raw[k], p + min(64 * (ws + WS * k) + h.pc, a.dqk - 8) * ES, 8 * ES);
    };
    auto move_down = [&](uint32_t *r, bool mine) {
#pragma unroll 1
        for (int u = a.dqk & 7; u < 8; u++)
#pragma unroll
            for (int e = 0; e < RAW; e++) {
                const uint32_t up = r[e + 1 < RAW ? e + 1 : e];
                const uint32_t v = ES == 4 ? up : e + 1 < RAW ? r[e] >> (8 * ES) | up << (32 - 8 * ES)
                                 : (r[e] >> (8 * ES)) | (r[e] & ~0u << (32 - 8 * ES));
                r[e] = mine ? v : r[e];
            }
    };
    auto store = [&](int buf) {
        const Place h = place();
        if (KVF == DSV4_GPU_KV_FP8 && ws == 0 && (h.home & 112) == 0) ((float *)meta(buf))[h.sr] = rks;
        if (KC == 4 && a.dqk < 8) piece((size_t)held * a.stride, h.pc, raw[0]);
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int s = ws + WS * k;
            if ((a.dqk & 7) && a.dqk > 8 && s == a.dqk >> 6)
                move_down(raw[k], 64 * s + h.pc == (a.dqk & ~7));
            if (L::SLABS % WS == 0 || s < L::SLABS)
                put(plane(buf) + s * L::SLAB + h.home, raw[k]);
        }
    };
    /* a masked tile's rows that are not there (ok) or hold what is not finite (in
     * the first plane, which has f32's infinities and NaN too) to zeros; the
     * eight threads of a row are lanes 8 k .. 8 k + 7 of two waves, and all look
     * at the whole row */
    auto mend = [&](int buf, uint32_t ok) {
        int *mi = (int *)meta(buf);
        const Place h = place();
        bool bad = false;
#pragma unroll 1
        for (int s = 0; s < L::SLABS; s++) {
            const u32x4 v = *(const u32x4 *)(plane(buf) + s * L::SLAB + h.home);
#pragma unroll
            for (int e = 0; e < 4; e++)
                bad |= (v[e] & 0x7F80u) == 0x7F80u || (v[e] & 0x7F800000u) == 0x7F800000u;
        }
        const bool gone = !(ok >> h.sr & 1u);
        if (KVF == DSV4_GPU_KV_FP8)
            bad |= (((const uint32_t *)mi)[h.sr] & 0x7F800000u) == 0x7F800000u;
        bad = (__ballot(bad) >> (lane0 & 56) & 0xFFull) != 0;
        tr_sync();                                     /* all have looked        */
        if (ws == 0 && (h.home & 112) == 0) {
            mi[TR_TILE + h.sr] = bad && !gone;
            if (KVF == DSV4_GPU_KV_FP8 && (bad || gone)) ((float *)mi)[h.sr] = 0.0f;
        }
        if (bad || gone)
            for (int s = ws; s < L::SLABS; s += WS)
                for (int n = 0; n < KT; n++)
                    *(u32x4 *)(plane(buf) + n * L::PLANE + s * L::SLAB + h.home) =
                        u32x4{0u, 0u, 0u, 0u};
        tr_sync();
    };

    /* the first tiles' loads go out before q's */
    uint32_t ok = 0u, ok1 = 0u, ok2 = 0u;              /* of tiles i, i + 1, i + 2 */
    if (i0 < i1) {
        ask(i0);
        ok = there(i0);
        if constexpr (DMA) {
            dma(i0, 0);
            ask(i0 + 1);
            if (i0 + 1 < i1) {
                ok1 = there(i0 + 1);
                dma(i0 + 1, 1);
            }
            ask(i0 + 2);
        } else {
            fetch(i0);
            ask(i0 + 1);
        }
    }

    /* ---- q, its loads all on their way at once, or a few chunks' where the first
     *      tile's f32 rows are in registers; elements past the row are zeroed by
     *      a mask in a register, as the many lane masks of comparisons would
     *      crowd out the scalar registers ---- */
    tr_bf8 q[NT][KC1];
    if (live) {
        const int l16 = lane0 & 15, g = lane0 >> 4;
        const T *qr = (const T *)a.q + (size_t)min(row0 + l16, R - 1) * a.dqk;
        constexpr int G = KVF != DSV4_GPU_KV_F32 ? KC1 : KC1 % 3 == 0 ? KC1 / 3 : 4;
        static_assert(KC1 % G == 0, "whole groups");
        const int c0 = 32 * KC1 * half + 8 * g;
        if (a.qvec) {
#pragma unroll
            for (int k0 = 0; k0 < KC1; k0 += G) {
                u32x4 v[G][sizeof(T) / 2];
#pragma unroll
                for (int u = 0; u < G; u++)
#pragma unroll
                    for (int h = 0; h < (int)sizeof(T) / 2; h++)
                        v[u][h] = ld16((const unsigned char *)(qr + min(c0 + 32 * (k0 + u),
                                                                         a.dqk - 8)) + 16 * h);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int u = 0; u < G; u++) {
                    const uint32_t in = (uint32_t)((c0 + 32 * (k0 + u) - a.dqk) >> 31);
                    if constexpr (sizeof(T) == 2) {
                        q[0][k0 + u] = __builtin_bit_cast(tr_bf8, v[u][0] & in);
                    } else {
                        float f[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) f[e] = __uint_as_float(v[u][e / 4][e % 4] & in);
                        tr_bf8 tm[NT];
                        tr_terms<NT>(f, tm);
#pragma unroll
                        for (int n = 0; n < NT; n++) q[n][k0 + u] = tm[n];
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int kc = 0; kc < KC1; kc++) {
                const int c = c0 + 32 * kc;
                float f[8];
                if (c + 8 <= a.dqk) {                  /* loads that need no alignment */
                    T v[8];
                    __builtin_memcpy(v, qr + c, sizeof(v));
#pragma unroll
                    for (int e = 0; e < 8; e++) io_load<T, 1>(v + e, f + e);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        io_load<T, 1>(qr + min(c + e, a.dqk - 1), f + e);
                        f[e] = __int_as_float(__float_as_int(f[e]) & ((c + e - a.dqk) >> 31));
                    }
                }
                tr_bf8 tm[NT];
                tr_terms<NT>(f, tm);
#pragma unroll
                for (int n = 0; n < NT; n++) q[n][kc] = tm[n];
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    /* ---- the drafts that the token of each row of q sees, and the first
     *      position ---- */
    if (lane0 < 16) {
        const int t = min(row0 + lane0, R - 1) / a.h;
        const unsigned long long all = a.nt >= 64 ? ~0ull : (1ull << a.nt) - 1;
        unsigned long long see = (a.mask ? a.mask[t] : (t >= 63 ? ~0ull : (2ull << t) - 1)) & all;
        const int depth = __popcll(see & ~(1ull << t));
        if (a.window && a.window < a.nt)
            for (int j = 0; j < a.nt; j++) {
                const unsigned long long oj = a.mask ? a.mask[j] : (2ull << j) - 1;
                /* signed: a token may see one that is further on */
                const int back = depth - (int)__popcll(oj & all & ~(1ull << j));
                if (back >= a.window) see &= ~(1ull << j);
            }
        unsigned char *d = lds + L::ROWS + 16 * (16 * w + lane0);
        *(unsigned long long *)d = see;
        *(int *)(d + 8) = a.window ? max(0, a.ctx + depth - a.window + 1) : 0;
    }

    f32x4 o[NV1];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int v = 0; v < NV1; v++) o[v] = f32x4{0.f, 0.f, 0.f, 0.f};
    /* to powers of two; a scale of 0 becomes one that still turns the infinity of
     * a masked score into a weight of 0 */
    const float c2 = (a.scale != 0.0f ? a.scale : 1e-38f) * 1.44269504088896340736f;
    const float blank = c2 > 0.0f ? -INFINITY : INFINITY;

    f32x4 s[2];                                        /* the scores of a tile   */
    auto score = [&](int buf) {
        const unsigned char *t = plane(buf);
        /* row l16's piece g of a slab, and its other half's at ^ 64 */
        const int ln = tr_fresh(lane0), l16 = ln & 15, g = ln >> 4;
        const int ka = l16 * 128 + 16 * (g ^ tr_swz(l16));
        /* one sum per order of the terms, so that the small ones do not round at
         * the size of the large */
        f32x4 so[2][PT];
#pragma unroll
        for (int n = 0; n < PT; n++) so[0][n] = so[1][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        /* chunk kc of this wave's: the second half's first is chunk KC1 of the
         * row, in the upper half of a slab where KC1 is odd */
        const unsigned char *tk = t + half * (KC1 >> 1) * L::SLAB;
        const int kb = ka ^ (KC1 & 1 & half) * 64;
        const int up = (KC1 & 1 & half) * L::SLAB;
        /* reads of 16 keys' piece of a chunk, KD of them ahead of the products */
        constexpr int KU = 2 * KC1, KD = KT > 1 || SHALLOW ? 2 : KU < 6 ? KU : 6;
        tr_bf8 row[KD][KT];
        auto rows_of = [&](int u) {
            const int kc = u >> 1;
#pragma unroll
            for (int p = 0; p < KT; p++)
                row[u % KD][p] = *(const tr_bf8 *)(tk + p * L::PLANE + (kc >> 1) * L::SLAB +
                                                   (kc & 1 ? up : 0) + (u & 1) * 2048 +
                                                   (kb ^ (kc & 1) * 64));
        };
#pragma unroll
        for (int u = 0; u < KD; u++) rows_of(u);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < KU; u++) {
#pragma unroll
            for (int p = 0; p < KT; p++)
#pragma unroll
                for (int n = 0; n < NT; n++)
                    if (n + p < PT)
                        so[u & 1][n + p] = tr_mfma(row[u % KD][p], q[n][u >> 1], so[u & 1][n + p]);
            __builtin_amdgcn_sched_barrier(0);
            if (u + KD < KU) rows_of(u + KD);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            s[k] = so[k][PT - 1];
#pragma unroll
            for (int n = PT - 2; n >= 0; n--) s[k] += so[k][n];
        }
        if constexpr (SPLIT == 2) {
            unsigned char *x = lds + L::HALF + 16 * ln;
#pragma unroll
            for (int k = 0; k < 2; k++) *(f32x4 *)(x + 1024 * (2 * w + k)) = s[k];
        }
    };
    auto value = [&](int i, int buf, bool masked) {
        const unsigned char *t = plane(buf);
        const int ln = tr_fresh(lane0), l16 = ln & 15, g = ln >> 4;
        /* row 4 g + l16 / 4's columns 4 (l16 % 4) of a slab, and its other tiles of
         * 16 columns at ^ 32, 64 and 96 */
        const int vr = 4 * g + (l16 >> 2);
        const int va = vr * 128 + 8 * (l16 & 1) + 16 * ((l16 >> 1 & 1) ^ tr_swz(vr));
        const int *mi = (const int *)meta(buf);
        if constexpr (SPLIT == 2) {
            const unsigned char *x = lds + L::HALF + 16 * ln;
#pragma unroll
            for (int k = 0; k < 2; k++) s[k] += *(const f32x4 *)(x + 1024 * (2 * (w ^ 1) + k));
        }
        /* the first columns of V, while the weights are computed */
        constexpr int VD = KT > 1 || SHALLOW ? 2 : NV1 < 5 ? NV1 : 5;
        const unsigned char *tv = t + half * (NV1 / 4) * L::SLAB;
        tr_bf8 col[VD][KT];
        auto cols_of = [&](int v) {
#pragma unroll
            for (int p = 0; p < KT; p++) {
                const unsigned char *at =
                    tv + p * L::PLANE + (v >> 2) * L::SLAB + (va ^ (v & 3) * 32);
                const tr_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_lds_s4 *)at);
                const tr_s4 y =
                    __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_lds_s4 *)(at + 2048));
                col[v % VD][p] = __builtin_bit_cast(
                    tr_bf8, (tr_s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        };
#pragma unroll
        for (int v = 0; v < VD; v++) cols_of(v);
        __builtin_amdgcn_sched_barrier(0);

        /* ---- the weights ---- */
        f32x4 ks[2];
        if (KVF == DSV4_GPU_KV_FP8) {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                ks[k] = *(const f32x4 *)(mi + 16 * k + 4 * g);
                s[k] *= ks[k];
            }
        }
        if (masked) {
            const uint32_t no = (uint32_t)__ballot(mi[TR_TILE + (ln & 31)] != 0);
            const unsigned char *rs = lds + L::ROWS + 16 * (16 * w + l16);
            const unsigned long long see = *(const unsigned long long *)rs;
            const int lo = *(const int *)(rs + 8), p0 = i * TR_TILE;
            /* positions [lo, ctx) of the context, then the drafts' bits */
            uint32_t vis = 0u;
            const int f = max(lo - p0, 0), e = min(a.ctx - p0, TR_TILE);
            if (f < e) vis = (e >= 32 ? ~0u : (1u << e) - 1u) & ~((1u << f) - 1u);
            const int d = p0 - a.ctx;
            if (d > -TR_TILE && d < 64) vis |= d >= 0 ? (uint32_t)(see >> d) : (uint32_t)(see << -d);
            vis &= ok;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int key = 16 * k + 4 * g + j;
                    const float x = no >> key & 1u ? __uint_as_float(0x7FC00000u) : s[k][j];
                    s[k][j] = vis >> key & 1u ? x : blank;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                top = fmaxf(top, s[k][j] * c2);
            }
        top = tr_max4(top);
        const bool grow = top > m + 8.0f;
        if (__any(grow)) {
            const float f = grow ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            m = grow ? top : m;
            l *= f;
#pragma unroll
            for (int v = 0; v < NV1; v++) o[v] *= f;
        }
        const float mm = m == -INFINITY ? 0.0f : m;
        float e[8], sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[k][j], c2, -mm));
                if (NT > 1) sum += x;
                e[4 * k + j] = x;
            }
        /* weights that are rounded are divided by the sum of the rounded ones, so that
         * o stays a mean of the rows (an FP8 row's scale, a power of two as the
         * append writes it, does not change how its weight rounds). 0 to 2 % slower
         * than the sum of the unrounded ones; by a product with ones 8 % at 512
         * columns and more */
        if constexpr (NT == 1) sum = tr_sum8(e);
        l += sum;
        if (KVF == DSV4_GPU_KV_FP8) {
            int at = 0;
            if constexpr (AGAIN) at = 4 * (tr_fresh(lane0) >> 4);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                if constexpr (AGAIN) ks[k] = *(const f32x4 *)(mi + 16 * k + at);
#pragma unroll
                for (int j = 0; j < 4; j++) e[4 * k + j] *= ks[k][j];
            }
        }
        tr_bf8 pw[NT];
        tr_terms<NT>(e, pw);

        /* ---- O^T ---- */
#pragma unroll
        for (int v = 0; v < NV1; v++) {
#pragma unroll
            for (int p = 0; p < KT; p++)
#pragma unroll
                for (int n = 0; n < NT; n++)
                    if (n + p < PT) o[v] = tr_mfma(col[v % VD][p], pw[n], o[v]);
            __builtin_amdgcn_sched_barrier(0);
            if (v + VD < NV1) cols_of(v + VD);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    /* every token sees every position of tiles [ic0, ic1) */
    const int ic0 = a.window ? (max(0, a.ctx + a.nt - a.window) + TR_TILE - 1) / TR_TILE : 0;
    const int ic1 = a.ctx / TR_TILE;
    if (!DMA && L::NBUF > 1 && i0 < i1) {
        store(0);
        if (i0 + 1 < i1) {
            ok1 = there(i0 + 1);
            fetch(i0 + 1);
            ask(i0 + 2);
        }
    }
    /* a later tile's loads out, and for formats that pass registers the next one
     * to LDS. Of the two waves of a SIMD one does so before its scores and one
     * after them, while the other's products run. */
    auto next = [&](int i, int buf) {
        if constexpr (DMA) {
            if (i + 2 >= i1) return;
            dma(i + 2, buf == 0 ? 2 : buf - 1);
            ask(i + 3);
        } else {
            if (i + 1 < i1) store(buf ^ 1);
            if (i + 2 >= i1) return;
            fetch(i + 2);
            ask(i + 3);
        }
    };
    for (int i = i0; i < i1; i++) {
        const int buf = slot(i);
        if constexpr (L::NBUF > 1) {
            if (DMA) dma_wait(i + 1 < i1);
            tr_sync();                                 /* tile i there, i - 1 used */
            if (i + 2 < i1) ok2 = there(i + 2);
            if (ws == 0) next(i, buf);
        } else {
            store(0);
            if (i + 1 < i1) {
                ok1 = there(i + 1);
                fetch(i + 1);
                ask(i + 2);
            }
            tr_sync();
        }
        const bool masked = i < ic0 || i >= ic1 || ok != ~0u;
        if (masked) mend(buf, ok);
        if (live) score(buf);
        if (L::NBUF > 1 && ws == 1) next(i, buf);
        if (SPLIT == 2) tr_sync();
        if (live) value(i, buf, masked);
        if (L::NBUF == 1) tr_sync();
        ok = ok1;
        ok1 = ok2;
    }

    /* ---- the split's sums, or the result ---- */
    const int ln = tr_fresh(lane0), g = ln >> 4, rq = row0 + (ln & 15);
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (!live || rq >= R) return;
    if (a.ns > 1) {
        const size_t at = (size_t)split * R + rq;
        if (g == 0 && half == 0) {
            a.pm[at] = m;
            a.pl[at] = l;
        }
        float *d = a.part + at * a.dvp + 16 * NV1 * half + 4 * g;
#pragma unroll
        for (int v = 0; v < NV1; v++)
            if (16 * (NV1 * half + v) < a.dvp) *(f32x4 *)(d + 16 * v) = o[v];
        return;
    }
    if (a.sink && l != 0.0f)
        l += __builtin_amdgcn_exp2f(a.sink[rq % a.h] * 1.44269504088896340736f - m);
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
    T *d = (T *)a.o + (size_t)rq * a.dv + 16 * NV1 * half + 4 * g;
#pragma unroll
    for (int v = 0; v < NV1; v++) {
        const f32x4 x = o[v] * inv;
        const float y[4] = {x.x, x.y, x.z, x.w};
        const int c = 16 * (NV1 * half + v) + 4 * g;
        if (a.ovec) {
            if (c < a.dv) io_store<T, 4>(d + 16 * v, y);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c + e < a.dv) io_store<T, 1>(d + 16 * v + e, y + e);
        }
    }
}

template <class T, int KVF, int KC>
int tree_launch(const Dsv4TreeJob &a, hipStream_t st)
{
    using L = TreeLds<KVF, KC, tree_split(tr_fmt<T>(), KVF, KC), tree_planes(tr_fmt<T>(), KVF)>;
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
    hipLaunchKernelGGL((k_tree<T, KVF, KC>), dim3((unsigned)(a.ns * a.nb)),
                       dim3(64 * TR_WAVES), L::BYTES, st, a);
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
