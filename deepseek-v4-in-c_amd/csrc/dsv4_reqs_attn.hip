/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_reqs_attn.hip - attention of a batch's requests over their pages of the
 * latent cache on gfx950: the plan, the join and the entry points (the kernel:
 * dsv4_tree.h).
 *
 * A token at position p of its request sees the request's positions up to p (the
 * last `window` of them), and every head of it reads the same rows:
 *   s_r = scale q . row_r[:d_qk],  o = sum e^(s_r - m) row_r[:d_v] / (sum e^(s_r
 *   - m) + e^(sink - m)).
 * Rows of q that read the same cache rows share each tile of them in a workgroup:
 * those of one request, and over the prefix those of all requests together, so
 * that it is read once for every 128 rows of q and not once for every request.
 * The lengths lie on the device, so a plan made there once a step, for all
 * layers, cuts both into items of about the same length, one a workgroup; sums of rows
 * that several items share are joined with weights e^(m_item - m).
 */
#include "dsv4_tree.h"

#include <math.h>
#include <type_traits>

namespace {

#include "dsv4_rows_io.h"

constexpr int RP_THREADS = 1024;
constexpr int RP_SPLITS = 255;                    /* most of a request's, or of the prefix */
constexpr int RP_KINDS = DSV4_REQS_KINDS - 1;      /* of the requests' items, by length */
constexpr int RP_EXTRA = 1024, RP_PREFIX = 4096;  /* items for splits; blocks of the prefix */
constexpr int RP_ROWS = 65536, RP_PREFIX_ROWS = 262144;  /* rows of sums      */

/* What a batch's plan and workspace have room for. */
struct ReqsRoom {
    long long rows, items, parts;
};
ReqsRoom reqs_room(int n_req, int max_tok, int h)
{
    ReqsRoom m;
    m.rows = (long long)max_tok * h;
    /* blocks of 64 rows, the fewest that a workgroup takes at most, of the requests and
     * of the prefix */
    m.items = 2 * (m.rows / 64) + n_req + 1 + RP_EXTRA;
    m.parts = RP_ROWS + (2 * m.rows < RP_PREFIX_ROWS ? 2 * m.rows : RP_PREFIX_ROWS);
    return m;
}

/* The items of a plan whose blocks have up to br rows, as many as are launched: all
 * requests' whole blocks, the prefix's, which few rows of each request make worth it, and
 * some for splits. A workgroup without one ends at once, 256 of them in a microsecond. */
int reqs_items(const ReqsRoom &m, int n_req, int br)
{
    const long long blocks = m.rows / br;
    return (int)(blocks + (blocks < RP_PREFIX ? blocks : RP_PREFIX) + n_req + 1 + RP_EXTRA);
}

struct PlanJob {
    Dsv4ReqsHead *head;
    Dsv4ReqsItem *items;
    Dsv4ReqsReq *req;
    const int *len, *first;
    int n_req, max_tok, h, window, prefix, room;  /* room: positions of a table */
    IoDiv by_h;
    int br, br_split, per_cu, dvp;                /* most rows, waves a block of 16 */
    float by_slots, inv_h, tile_us, wave_more;    /* a tile's time, and how a wave of rows adds */
    int max_items, max_parts;
    uint64_t sig;
};

/* A request's step: tokens, the position of the first, tiles behind the prefix's. */
struct PlanReq {
    int n, pos, tile0, tile1;
};

/* The sum of lanes 0 to this one's, by moves within the vector unit. */
template <int CTRL, int ROWS>
__device__ __forceinline__ int moved(int v)
{
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v)
{
    v += moved<0x111, 0xF>(v);                    /* row_shr:1, 2, 4, 8      */
    v += moved<0x112, 0xF>(v);
    v += moved<0x114, 0xF>(v);
    v += moved<0x118, 0xF>(v);
    v += moved<DPP_ROW_BCAST15, 0xA>(v);
    v += moved<DPP_ROW_BCAST31, 0xC>(v);
    return v;
}

/* The largest of all lanes' v, a whole number not negative. */
__device__ __forceinline__ int wave_top(int v)
{
    v = max(v, moved<DPP_QUAD_XOR1, 0xF>(v));
    v = max(v, moved<DPP_QUAD_XOR2, 0xF>(v));
    v = max(v, moved<DPP_ROW_HMIRROR, 0xF>(v));
    v = max(v, moved<DPP_ROW_MIRROR, 0xF>(v));
    v = max(v, moved<DPP_ROW_BCAST15, 0xA>(v));
    v = max(v, moved<DPP_ROW_BCAST31, 0xC>(v));
    return __builtin_amdgcn_readlane(v, 63);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float top_with(float v)
{
    const int i = __float_as_int(v);              /* itself where no lane is moved */
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, ROWS, 0xF, false)));
}
__device__ __forceinline__ float wave_top(float v)
{
    v = top_with<DPP_QUAD_XOR1, 0xF>(v);
    v = top_with<DPP_QUAD_XOR2, 0xF>(v);
    v = top_with<DPP_ROW_HMIRROR, 0xF>(v);
    v = top_with<DPP_ROW_MIRROR, 0xF>(v);
    v = top_with<DPP_ROW_BCAST15, 0xA>(v);
    v = top_with<DPP_ROW_BCAST31, 0xC>(v);
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
/* The sum over 16 lanes. */
__device__ __forceinline__ float row_sum(float v)
{
    v += dpp_f<DPP_QUAD_XOR1, 0xF>(v);
    v += dpp_f<DPP_QUAD_XOR2, 0xF>(v);
    v += dpp_f<DPP_ROW_HMIRROR, 0xF>(v);
    return v + dpp_f<DPP_ROW_MIRROR, 0xF>(v);
}

/* Tiles cut into items of about `each`: how many, to RP_SPLITS. A quotient of floats
 * may be one off, which makes an item a little longer or shorter. */
struct PlanCut {
    float by;
    __device__ __forceinline__ explicit PlanCut(int each) : by(__builtin_amdgcn_rcpf((float)each)) {}
    __device__ __forceinline__ int splits(int tiles) const
    {
        return tiles ? max(1, min((int)ceilf((float)tiles * by - 1e-3f), RP_SPLITS)) : 0;
    }
};

/* One workgroup. A plan is: with the prefix apart or not, the rows of a block and the
 * tiles of an item. 64 of them are priced in microseconds: a tile takes what its loads and
 * the waits between them take, whatever rows of q it serves (1.65 us for 16, 32 and 64 rows
 * of bf16, 576 columns), 2.2 and half a microsecond a wave of 16 rows are an item's start,
 * and then come the sums that are joined. Workgroups begin in their order, and those of
 * one XCD go to its four engines in turn, so the longest items come first and the short ones
 * fill what the last round of these leaves free, if every engine has a free CU: items by
 * request took 420 us for 64 requests behind 32768 positions and these 364, 128 ragged
 * ones 240 and 201, 570 tokens of prompts 125 and 73.
 *
 * Bound: the chain of a load, five reductions and two scans, and the fetch of code that
 * runs once: 8 us for 8 requests, 12 for 128. Sums that are only compared are floats,
 * lanes add up within the vector unit (through LDS 10 and 13), loops that could be unrolled
 * are not (20 us unrolled, in whole numbers). */
__global__ void __launch_bounds__(RP_THREADS) k_reqs_plan(PlanJob a)
{
    extern __shared__ __align__(16) int lds[];
    __shared__ unsigned long long best, owner;
    __shared__ float work[2 * 8];
    __shared__ int bad, active, hi_min, lo_max, lo_min, longest[8];
    __shared__ int part_w[RP_THREADS / 64][2 + RP_KINDS];
    __shared__ int rows_each, tiles_each, tiles_from, longest_own;
    const int tid = threadIdx.x, lane = tid & 63, nr = a.n_req;
    int *s_first = lds, *s_len = lds + nr + 1, *s_item = s_len + nr,
        *s_to = lds + ((3 * nr + 2 + 3) & ~3),    /* four a request */
        *s_part = s_to + RP_KINDS * nr;
    if (tid == 0) {
        best = ~0ull;
        owner = 0;
        bad = active = lo_max = 0;
        hi_min = lo_min = INT32_MAX;
    }
    if (tid < 8) longest[tid] = 0;
    for (int b = tid; b <= nr; b += RP_THREADS) {
        s_first[b] = nr ? a.first[b] : 0;
        if (b < nr) s_len[b] = a.len[b];
    }
    __syncthreads();
    const int tok0 = s_first[0], tok1 = s_first[nr];
    auto lo_of = [&](int pos) { return a.window ? max(0, pos - a.window + 1) : 0; };
    auto request = [&](int b, int prefix_tiles) {
        PlanReq r;
        r.n = s_first[b + 1] - s_first[b];
        r.pos = s_len[b] - r.n;
        r.tile0 = max(prefix_tiles, lo_of(r.pos) / TR_TILE);
        r.tile1 = max(r.tile0, (s_len[b] + TR_TILE - 1) / TR_TILE);
        return r;
    };
    /* tiles of a request's block on average: an earlier one ends earlier, and with a window
     * one of more rows begins earlier */
    const float tiles_less = a.window ? 1.0f / TR_TILE : 0.5f / TR_TILE;
    auto mean_tiles = [&](int n, int t, float toks) {
        return t ? fmaxf((float)t - fmaxf((float)n - toks, 0.0f) * tiles_less, 1.0f) : 0.0f;
    };
    {
        int b_bad = tok0 < 0 || tok1 > a.max_tok, n_act = 0, hmin = INT32_MAX, lmax = 0,
            lmin = INT32_MAX;
        unsigned long long own = 0;
        for (int b = tid; b < nr; b += RP_THREADS) {
            const int f0 = s_first[b], f1 = s_first[b + 1], len = s_len[b], n = f1 - f0;
            if (f0 < 0 || f1 < f0 || f1 > a.max_tok || (n && (len < n || len > a.room))) {
                b_bad = 1;
                continue;
            }
            if (!n) continue;
            n_act++;
            hmin = min(hmin, len - n + 1);
            lmax = max(lmax, lo_of(len - 1));
            lmin = min(lmin, lo_of(len - n));
            const unsigned long long o = (unsigned long long)len << 32 | (uint32_t)b;
            own = o > own ? o : own;
        }
        if ((tid & ~63) < nr) {                   /* a wave, whole or not at all */
            b_bad = wave_top(b_bad);
            n_act = __builtin_amdgcn_readlane(wave_scan(n_act), 63);
            hmin = INT32_MAX - wave_top(INT32_MAX - hmin);
            lmax = wave_top(lmax);
            lmin = INT32_MAX - wave_top(INT32_MAX - lmin);
            const int len = wave_top((int)(own >> 32));
            own = (unsigned long long)len << 32 |
                  (uint32_t)wave_top((int)(own >> 32) == len ? (int)own : 0);
            if (lane == 0) {
                if (b_bad) bad = 1;
                atomicAdd(&active, n_act);
                atomicMin(&hi_min, hmin);
                atomicMax(&lo_max, lmax);
                atomicMin(&lo_min, lmin);
                atomicMax(&owner, own);
            }
        }
    }
    __syncthreads();
    const int R0 = tok0 * a.h, R = (tok1 - tok0) * a.h;
    if (bad || active == 0) {
        if (tid == 0) *a.head = Dsv4ReqsHead{bad ? ~a.sig : a.sig, {}, 0, 0, 0};
        return;
    }
    /* whole tiles of the prefix, as far as the longest request has it */
    const int max_len = (int)(owner >> 32);
    const int pt1 = min(a.prefix, max_len) / TR_TILE, pt0 = min(pt1, lo_min / TR_TILE);
    const bool may = active > 1 && pt1 > pt0;
    /* a request's tokens, rows, tiles and tiles behind the prefix, where s_to will be */
    for (int b = tid; b < nr; b += RP_THREADS) {
        const PlanReq q = request(b, 0), p = request(b, pt1);
        s_to[4 * b] = q.n;
        s_to[4 * b + 1] = q.n * a.h;
        s_to[4 * b + 2] = q.n ? q.tile1 - q.tile0 : 0;
        s_to[4 * b + 3] = q.n ? p.tile1 - p.tile0 : 0;
    }
    __syncthreads();

    /* group g (two waves): the prefix apart (g & 1), blocks of 1 << rs rows */
    const int g = tid >> 7, gt = tid & 127, rs = 4 + (g >> 1), r = 1 << rs;
    const bool apart = g & 1, on = r <= a.br && (!apart || may);
    const int from = apart ? pt1 : 0, ptiles = apart ? pt1 - pt0 : 0;
    const int pblocks = apart ? (R + r - 1) >> rs : 0;
    const float toks = (float)r * a.inv_h;
    if (on) {
        float w = 0.0f;
        int l = ptiles;
        for (int b = gt; b < nr; b += 128) {
            const int n = s_to[4 * b], rows = s_to[4 * b + 1], t = s_to[4 * b + 2 + apart];
            w += (float)((rows + r - 1) >> rs) * mean_tiles(n, t, toks);
            l = max(l, t);
        }
        w = wave_sum(w);
        l = wave_top(l);
        if (lane == 0) {
            work[tid >> 6] = w;
            atomicMax(&longest[g], l);
        }
    }
    __syncthreads();
    {
        /* tiles of an item, so that they are about so many workgroups' worth of the card */
        const int c = gt >> 4, cl = gt & 15;
        constexpr float SHARE[8] = {1.0f / 112, 1.0f / 208, 1.0f / 224, 1.0f / 256,
                                    1.0f / 448, 1.0f / 480, 1.0f / 704, 0.0f};
        const float w = work[2 * g] + work[2 * g + 1] + (float)pblocks * (float)ptiles;
        const int each = c < 7 ? max(1, (int)ceilf(fminf(w * SHARE[c], 1e9f))) : 1 << 30;
        const int most = min(each, longest[g]), ps = PlanCut(each).splits(ptiles);
        const PlanCut cut(each);
        const float half = 0.5f * (float)most;
        float items = 0.0f, parts = 0.0f;
        float big = 0.0f, big_tiles = 0.0f;       /* of half the longest or more */
        if (on) {
            for (int b = cl; b < nr; b += 16) {
                const int toks_b = s_to[4 * b], rows = s_to[4 * b + 1], t = s_to[4 * b + 2 + apart];
                const int ns = max(cut.splits(t), apart || !toks_b ? 0 : 1);
                const float n = (float)((rows + r - 1) >> rs) * (float)ns;
                items += n;
                parts += apart || ns > 1 ? (float)ns * (float)rows : 0.0f;
                /* blocks' tiles lie about evenly from 2 mean - t to t */
                const float least = fmaxf(2.0f * mean_tiles(toks_b, t, toks) - (float)t, 0.0f);
                const float of_item = half * (float)ns, spread = fmaxf((float)t - least, 1e-3f);
                const float longer = n * fminf(fmaxf(((float)t - of_item) * __builtin_amdgcn_rcpf(spread),
                                                     0.0f), 1.0f);
                big += longer;
                big_tiles += longer * 0.5f * ((float)t + fmaxf(of_item, least)) *
                             __builtin_amdgcn_rcpf((float)max(ns, 1));
            }
        }
        items = row_sum(items);
        parts = row_sum(parts);
        big = row_sum(big);
        big_tiles = row_sum(big_tiles);
        items += (float)pblocks * (float)ps;
        parts += (float)ps * (float)R;
        /* Sums of at most 4096 floats: 2^-12 off at most. The largest blocks, whole, are
         * what the plan's and the sums' rooms are made for. */
        const bool whole = c == 7 && !apart && r == a.br;
        unsigned long long price = ~0ull;
        if (on && (whole || (items * 1.001f <= (float)a.max_items &&
                             parts * 1.001f <= (float)a.max_parts))) {
            const int waves = (r >> 4) * a.br_split;
            const float slots = 256.0f * a.per_cu, by = a.by_slots, n = items;
            const float tile = a.tile_us * (1.0f + a.wave_more * waves);
            const float start = 2.2f + 0.55f * waves;
            if (ps && (float)ptiles >= half * ps) {
                big += (float)pblocks * ps;
                big_tiles += (float)pblocks * (float)ptiles;
            }
            const float one = (float)most * tile + start, all = w * tile + n * start;
            const float rounds = fmaxf(ceilf(big * by), 1.0f);
            const float flow = all * by + 0.6f * one;
            const float rest = (w - big_tiles) * tile + (n - big) * start;
            const float spare = rounds * slots - big;
            const bool fits = big >= n || (spare >= 0.125f * slots && rest <= 0.9f * spare * one);
            float cost = fmaxf(fits ? big >= n ? fminf(rounds * one, flow) : rounds * one : flow, one);
            cost += (parts > 0.0f ? 1.4f : 0.0f) + parts * (float)a.dvp * 0.92e-6f;
            /* a price over 0 orders as its bits do */
            price = (unsigned long long)__float_as_uint(cost) << 32 | (uint32_t)(g << 3 | c);
        }
#pragma unroll
        for (int o = 32; o >= 16; o >>= 1) {
            const unsigned long long v = __shfl_xor(price, o, 64);
            price = v < price ? v : price;
        }
        if (lane == 0 && price != ~0ull) atomicMin(&best, price);
        __syncthreads();
        if ((int)(best & 63) == (g << 3 | c) && cl == 0) {
            rows_each = rs;
            tiles_each = each;
            tiles_from = from;
            longest_own = max(1, longest[g]);
        }
        __syncthreads();
    }
    const int bs = rows_each, br = 1 << bs, start = tiles_from;
    const PlanCut cut(tiles_each);
    const int ps = start ? cut.splits(pt1 - pt0) : 0;
    const int pb = start ? (R + br - 1) >> bs : 0, pitems = ps * pb;

    /* where each request's items and sums begin */
    const int per = (nr + RP_THREADS - 1) / RP_THREADS;
    const int b0 = min(nr, tid * per), b1 = min(nr, b0 + per);
    auto splits = [&](const PlanReq &q) {
        const int ns = cut.splits(q.tile1 - q.tile0);
        return start ? ns : max(ns, 1);
    };
    /* Items by their length, in quarters of the longest: the first block with three of
     * them or more, with two and with one. Without a window a block's last row decides. */
    const int most = min(tiles_each, longest_own);
    auto quarters = [&](const PlanReq &q, int nb, int ns, int *from) {
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const int need = min(((most * (3 - k) + 3) / 4) * ns, q.tile1 - q.tile0 + 1);
            const int tok = (int)((uint32_t)(need + q.tile0 - 1) * TR_TILE - (uint32_t)q.pos);
            from[k] = a.window ? need <= q.tile1 - q.tile0 ? 0 : nb
                               : tok >= q.n ? nb : (max(tok, 0) * a.h) >> bs;
        }
    };
    constexpr int NX = 2 + RP_KINDS;              /* items, rows of sums, items by length */
    int sum[NX] = {};
    for (int b = b0; b < b1; b++) {
        const PlanReq q = request(b, start);
        const int rows = q.n * a.h, ns = q.n ? splits(q) : 0, nb = (rows + br - 1) >> bs;
        int f[3];
        quarters(q, nb, ns, f);
        sum[0] += nb * ns;
        sum[1] += start || ns > 1 ? ns * rows : 0;
        sum[2] += (nb - f[0]) * ns;
        sum[3] += (f[0] - f[1]) * ns;
        sum[4] += (f[1] - f[2]) * ns;
        sum[5] += f[2] * ns;
    }
    int x[NX];
#pragma unroll
    for (int k = 0; k < NX; k++) x[k] = wave_scan(sum[k]);
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < NX; k++) part_w[tid >> 6][k] = x[k];
    __syncthreads();
    Dsv4ReqsHead head{a.sig, {pitems}, ps, R0, R};
    int all[NX] = {};
    const int waves = ((nr + per - 1) / per + 63) / 64;
#pragma unroll 1
    for (int w = 0; w < waves; w++)
#pragma unroll
        for (int k = 0; k < NX; k++) {
            const int v = part_w[w][k];
            x[k] += w < tid >> 6 ? v : 0;
            all[k] += v;
        }
#pragma unroll
    for (int k = 0; k < NX; k++) {
        x[k] -= sum[k];
        if (k >= 2) {
            x[k] += head.end[k - 2];
            head.end[k - 1] = head.end[k - 2] + all[k];
        }
    }
    x[1] += ps * R;
    for (int b = b0; b < b1; b++) {
        const PlanReq q = request(b, start);
        const int rows = q.n * a.h, ns = q.n ? splits(q) : 0, nb = (rows + br - 1) >> bs;
        const bool direct = !start && ns <= 1;
        int f[3];
        quarters(q, nb, ns, f);
        s_item[b] = x[0];
        for (int k = 0; k < RP_KINDS; k++) s_to[RP_KINDS * b + k] = x[2 + k];
        s_part[b] = direct ? -1 : x[1];
        a.req[b] = Dsv4ReqsReq{s_first[b], q.pos, s_part[b], q.n << 8 | ns};
        x[0] += nb * ns;
        x[1] += direct ? 0 : ns * rows;
        x[2] += (nb - f[0]) * ns;
        x[3] += (f[0] - f[1]) * ns;
        x[4] += (f[1] - f[2]) * ns;
        x[5] += f[2] * ns;
    }
    if (b0 < b1 && b1 == nr) s_item[b1] = x[0];
    __syncthreads();
    const int items = s_item[nr];
    if (tid == 0) *a.head = head;
    const bool all_see = hi_min >= pt1 * TR_TILE && lo_max == 0;
    for (int i = tid; i < pitems; i += RP_THREADS) {
        const int s = i / pb, blk = i - s * pb;
        Dsv4ReqsItem it{};
        it.row0 = R0 + (blk << bs);
        it.rows = min(br, R - (blk << bs));
        it.req = (int)(uint32_t)owner;
        it.tile0 = pt0 + (int)((long long)(pt1 - pt0) * s / ps);
        it.tile1 = pt0 + (int)((long long)(pt1 - pt0) * (s + 1) / ps);
        it.end = pt1 * TR_TILE;
        it.lo = all_see ? 0 : lo_max;
        it.hi = all_see ? INT32_MAX : hi_min;
        it.kind = all_see ? 0 : 2;
        it.part = s * R + (blk << bs);
        a.items[i] = it;
    }
    for (int i = tid; i < items; i += RP_THREADS) {
        int b = 0, end = nr;                      /* the last request that starts here or
                                                   * before (one without items has the
                                                   * next one's number) */
        while (end - b > 1) {
            const int mid = (b + end) >> 1;
            if (s_item[mid] <= i) b = mid;
            else end = mid;
        }
        const PlanReq q = request(b, start);
        const int rows = q.n * a.h, nb = (rows + br - 1) >> bs, ns = splits(q);
        const int k = i - s_item[b], s = nb == 1 ? k : k / nb, blk = k - s * nb, r0 = blk << bs;
        int f[3];
        quarters(q, nb, ns, f);
        /* of its quarter, the last block first */
        const int c = blk >= f[0] ? 0 : blk >= f[1] ? 1 : blk >= f[2] ? 2 : 3;
        const int c1 = c == 0 ? nb : c == 1 ? f[0] : c == 2 ? f[1] : f[2];
        const int c0 = c == 0 ? f[0] : c == 1 ? f[1] : c == 2 ? f[2] : 0;
        const int to = s_to[RP_KINDS * b + c] + s * (c1 - c0) + c1 - 1 - blk;
        Dsv4ReqsItem it{};
        it.rows = min(br, rows - r0);
        it.row0 = s_first[b] * a.h + r0;
        it.req = b;
        /* a block's first and last tokens bound what its rows see */
        const int p0 = q.pos + (int)a.by_h.div((uint32_t)r0);
        const int p1 = q.pos + (int)a.by_h.div((uint32_t)(r0 + it.rows - 1));
        const int t0 = max(q.tile0, lo_of(p0) / TR_TILE), t1 = max(t0, p1 / TR_TILE + 1);
        it.tile0 = t0 + (int)((long long)(t1 - t0) * s / ns);
        it.tile1 = t0 + (int)((long long)(t1 - t0) * (s + 1) / ns);
        it.end = p1 + 1;
        it.lo = lo_of(p1);
        it.hi = p0 + 1;
        it.kind = 1;
        it.pos0 = p0;
        it.part = s_part[b] < 0 ? -1 : s_part[b] + s * rows + r0;
        a.items[to] = it;
    }
}

constexpr int RJ_THREADS = 256, RJ_WAVES = RJ_THREADS / 64;
constexpr int RJ_ROWS = 2048;                     /* from here on a wave a row */
constexpr int RJ_GROUPS = 4096;

struct JoinJob {
    const Dsv4ReqsHead *head;
    const Dsv4ReqsReq *req;
    const float *part, *pm, *pl, *sink;
    int n_req, h, dv, dvp, ovec;
    long long rows;                               /* of the whole buffer     */
    IoDiv by_h;
    uint64_t sig;
};

/* Rows whose sums lie in several places: the prefix's splits and then the request's.
 * WAVES waves a row: each has the weights, and adds every WAVES-th place. Few rows have
 * their workgroups' four (16 rows of 125 places 10 us, a wave a row 30; 512 of 4 6 and 7;
 * 2048 the same), many a wave each (4096 of 4 places 9 us, with four waves 11; of 128
 * columns 5 and 10). Bound: the places' bytes, 6 TB/s from L2 for many rows, and for few
 * a chain of the head, the request, the maxima and the sums. */
template <class T>
__global__ void __launch_bounds__(RJ_THREADS) k_reqs_join(JoinJob a, T *o)
{
    __shared__ f32x4 sum[RJ_WAVES][TR_DV / 4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Dsv4ReqsHead hd = *a.head;
    if (hd.sig != a.sig) {                        /* not this call's plan    */
        const float nan = __uint_as_float(0x7FC00000u);
        const long long n = a.rows * a.dv, step = (long long)gridDim.x * RJ_THREADS;
        for (long long i = (long long)blockIdx.x * RJ_THREADS + tid; i < n; i += step)
            io_store<T, 1>(o + i, &nan);
        return;
    }
    auto row = [&](int i, auto waves) {
        constexpr int WAVES = decltype(waves)::value;
        const int w = WAVES > 1 ? wave : 0;
        const int r = hd.row0 + i, t = (int)a.by_h.div((uint32_t)r);
        /* the last request whose first token is t or before it: of every step-th one, then
         * of those behind it */
        const int step = (a.n_req + 63) / 64;
        int b = 0;
        for (int s = step; s >= 1; s = s > 1 ? 1 : 0) {
            const int k = b + lane * s;
            const unsigned long long before =
                __ballot(lane < (s > 1 ? 64 : step > 1 ? step : 64) && k < a.n_req &&
                         a.req[min(k, a.n_req - 1)].first <= t);
            b += (63 - (int)__builtin_clzll(before | 1)) * s;
        }
        const Dsv4ReqsReq q = a.req[b];
        if (q.part < 0) return;
        const int ps = hd.prefix_splits, n = ps + (q.cut & 255), rows = (q.cut >> 8) * a.h;
        const size_t own = (size_t)q.part + (r - q.first * a.h);
        auto place = [&](int s) {
            return s < ps ? (size_t)s * hd.rows + i : own + (size_t)(s - ps) * rows;
        };
        constexpr int NK = (2 * RP_SPLITS + 63) / 64;
        float ms[NK], ls[NK], m = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            const int s = 64 * k + lane;
            ms[k] = -INFINITY;
            ls[k] = 0.0f;
            if (64 * k < n && s < n) {
                ms[k] = a.pm[place(s)];
                ls[k] = a.pl[place(s)];
            }
            m = fmaxf(m, ms[k]);
        }
        m = wave_top(m);
#pragma unroll
        for (int k = 0; k < NK; k++) {
            if (64 * k >= n) break;
            ms[k] = tree_join_weight(ms[k], ls[k], m);
            l += ms[k] * ls[k];
        }
        l = wave_sum(l);
        if (a.sink && l != 0.0f)
            l += __builtin_amdgcn_exp2f(a.sink[r - t * a.h] * 1.44269504088896340736f - m);
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
        constexpr int G = 4;                          /* places in flight        */
#pragma unroll
        for (int k = 0; k < NK; k++) {
            if (64 * k >= n) break;
            const int end = min(n, 64 * k + 64);
            for (int s0 = 64 * k + w; s0 < end; s0 += G * WAVES) {
                f32x4 x[G][2];
#pragma unroll
                for (int u = 0; u < G; u++) {
                    const float *p = a.part + place(min(s0 + u * WAVES, n - 1)) * a.dvp + 4 * lane;
#pragma unroll
                    for (int c = 0; c < 2; c++)
                        x[u][c] = 256 * c + 4 * lane < a.dvp ? ldf4(p + 256 * c)
                                                             : f32x4{0.f, 0.f, 0.f, 0.f};
                }
#pragma unroll
                for (int u = 0; u < G; u++) {
                    const int s = s0 + u * WAVES;
                    const float e = __shfl(ms[k], s & 63, 64);
                    if (s < end)
#pragma unroll
                        for (int c = 0; c < 2; c++) v[c] += e * x[u][c];
                }
            }
        }
        auto store = [&](int c, f32x4 y4) {
            if (c >= a.dv) return;
            y4 = y4 * inv;
            const float y[4] = {y4.x, y4.y, y4.z, y4.w};
            T *d = o + (size_t)r * a.dv + c;
            if (a.ovec) {
                io_store<T, 4>(d, y);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (c + e < a.dv) io_store<T, 1>(d + e, y + e);
            }
        };
        if constexpr (WAVES == 1) {
            store(4 * lane, v[0]);
            store(256 + 4 * lane, v[1]);
        } else {
            sum[w][lane] = v[0];
            sum[w][64 + lane] = v[1];
            __syncthreads();
            if (tid < TR_DV / 4) {
                f32x4 y = sum[0][tid];
#pragma unroll
                for (int k = 1; k < WAVES; k++) y += sum[k][tid];
                store(4 * tid, y);
            }
        }
    };
    if (hd.rows < RJ_ROWS) {                      /* a workgroup for each at least */
        if ((int)blockIdx.x < hd.rows) row(blockIdx.x, std::integral_constant<int, RJ_WAVES>());
    } else {
        for (int i = (int)blockIdx.x * RJ_WAVES + wave; i < hd.rows; i += (int)gridDim.x * RJ_WAVES)
            row(i, std::integral_constant<int, 1>());
    }
}

template <class T>
void join_launch(const JoinJob &a, T *o, hipStream_t st)
{
    const long long waves = (a.rows + RJ_WAVES - 1) / RJ_WAVES, some = a.rows < RJ_ROWS ? a.rows : RJ_ROWS;
    const long long groups = waves < some ? some : waves < RJ_GROUPS ? waves : RJ_GROUPS;
    hipLaunchKernelGGL(k_reqs_join<T>, dim3((unsigned)groups), dim3(RJ_THREADS), 0, st, a, o);
}

/* What is wrong with a call's shape, or nullptr. */
const char *reqs_bad(const dsv4_gpu_reqs *r, int fmt, int h, int d_qk, int d_v, int kv_fmt,
                     int window)
{
    if (const char *bad = dsv4_reqs_bad(r)) return bad;
    if (fmt != DSV4_WF32 && fmt != DSV4_WBF16) return "an unknown type of q";
    if (kv_fmt != DSV4_GPU_KV_F32 && kv_fmt != DSV4_GPU_KV_BF16 && kv_fmt != DSV4_GPU_KV_FP8)
        return "an unknown cache format";
    if (h <= 0 || h > 4096) return "1 to 4096 heads are taken";
    if ((long long)h * r->max_tok > 1 << 28) return "at most 2^28 rows of q are taken";
    if (d_v <= 0 || d_qk < d_v || d_qk > TR_DQK || d_v > TR_DV)
        return "widths d_v <= d_qk, at most 512 and 576, are taken";
    if (window < 0) return "a negative window";
    return nullptr;
}

/* A plan's arguments in 64 bits, which others have by a chance of 2^-64 only (32 would do
 * for mistakes, but a plan of other sizes may pass a buffer's end; all of the arguments,
 * compared word by word, cost 0.7 to 1.2 us in each pass). */
uint64_t reqs_sig(const dsv4_gpu_reqs *r, int fmt, int h, int d_qk, int d_v, int kv_fmt,
                  int window)
{
    const int v[] = {r->n_req, r->max_pages, r->page_rows, r->max_tok, r->n_prefix, fmt, h, d_qk,
                     d_v, kv_fmt, window};
    uint64_t x = 0x9E3779B97F4A7C15ull;
    for (const int k : v) {
        x = (x ^ (uint32_t)k) * 0xD6E8FEB86659FD93ull;
        x ^= x >> 32;
    }
    return x;
}

struct PlanParts {
    size_t items, req, bytes;
};
PlanParts plan_parts(int n_req, int max_tok, int h)
{
    const ReqsRoom m = reqs_room(n_req, max_tok, h);
    PlanParts p;
    p.items = 64;
    p.req = p.items + (size_t)m.items * sizeof(Dsv4ReqsItem);
    p.bytes = p.req + (size_t)n_req * sizeof(Dsv4ReqsReq);
    return p;
}
static_assert(sizeof(Dsv4ReqsHead) <= 64, "the plan's head");

bool reqs_sizes(int n_req, int max_tok, int h)
{
    return n_req >= 0 && n_req <= 4096 && max_tok >= 0 && max_tok <= 1 << 20 && h > 0 &&
           h <= 4096 && (long long)h * max_tok <= 1 << 28;
}

} // namespace

extern "C" size_t dsv4_gpu_reqs_plan_bytes(int n_req, int max_tok, int h)
{
    return reqs_sizes(n_req, max_tok, h) ? plan_parts(n_req, max_tok, h).bytes : 0;
}

extern "C" size_t dsv4_gpu_reqs_attn_scratch_bytes(int fmt, int h, int d_qk, int d_v, int kv_fmt,
                                                   int n_req, int max_tok)
{
    const dsv4_gpu_reqs r{nullptr, nullptr, nullptr, n_req, 1, 1, max_tok, 0};
    if (reqs_bad(&r, fmt, h, d_qk, d_v, kv_fmt, 0)) return 0;
    const size_t dvp = (size_t)(d_v + 15) / 16 * 16;
    return (size_t)reqs_room(n_req, max_tok, h).parts * (dvp + 2) * sizeof(float);
}

extern "C" int dsv4_gpu_reqs_plan_d(void *d_plan, size_t plan_bytes, const dsv4_gpu_reqs *r,
                                    int fmt, int h, int d_qk, int d_v, int kv_fmt, int window,
                                    void *stream)
{
    const char *bad = reqs_bad(r, fmt, h, d_qk, d_v, kv_fmt, window);
    if (!bad && (!r->first || (r->n_req && !r->len))) bad = "a missing buffer";
    if (bad) {
        DSV4_ERR("reqs_plan: %s", bad);
        return -1;
    }
    const PlanParts pp = plan_parts(r->n_req, r->max_tok, h);
    if (!d_plan || ((uintptr_t)d_plan & 15) || plan_bytes < pp.bytes) {
        DSV4_ERR("reqs_plan: %zu bytes at %p; the plan needs %zu, 16-byte aligned", plan_bytes,
                 d_plan, pp.bytes);
        return -1;
    }
    const ReqsRoom m = reqs_room(r->n_req, r->max_tok, h);
    const int kc = dsv4_tree_chunks(d_qk, d_v);
    char *p = (char *)d_plan;
    PlanJob a{.by_h = IoDiv((uint32_t)h)};
    a.head = (Dsv4ReqsHead *)p;
    a.items = (Dsv4ReqsItem *)(p + pp.items);
    a.req = (Dsv4ReqsReq *)(p + pp.req);
    a.len = r->len;
    a.first = r->first;
    a.n_req = r->n_req;
    a.max_tok = r->max_tok;
    a.h = h;
    a.window = window;
    a.prefix = r->n_prefix;
    a.room = r->max_pages * r->page_rows;
    a.br = dsv4_tree_block_rows(fmt, kv_fmt, kc);
    a.br_split = tree_split(fmt, kv_fmt, kc);
    a.per_cu = tree_per_cu(fmt, kc);
    a.dvp = (d_v + 15) / 16 * 16;
    /* A lone workgroup's tile: bf16 1.66 us (576 columns) and 0.78 (128), f32 q over bf16
     * 1.94, f32 over f32 4.8, bf16 q over f32 2.8; over FP8 1.8 and, with the card full, 3.3.
     * From 16 rows to 64 it grows by 2 percent (bf16) to 25 (several products). */
    const int planes = tree_planes(fmt, kv_fmt), products = fmt == DSV4_WF32 ? planes == 1 ? 3 : 6 : planes;
    a.tile_us = 0.5f + 32.0f * kc * (0.002f * planes + 0.00025f * products +
                                     (kv_fmt == DSV4_WFP8 ? 0.001f : 0.0f));
    a.inv_h = 1.0f / (float)h;
    a.by_slots = 1.0f / (256.0f * (float)a.per_cu);
    a.wave_more = products > 1 ? 0.05f : 0.02f;
    a.max_items = reqs_items(m, r->n_req, a.br);
    a.max_parts = (int)m.parts;
    a.sig = reqs_sig(r, fmt, h, d_qk, d_v, kv_fmt, window);
    const size_t lds = 8 * ((size_t)r->n_req + 1) * sizeof(int);
    if (lds > 64 * 1024 - 1024) {
        static bool asked[64];
        int dev = 0;
        HIP_OK(hipGetDevice(&dev), "hipGetDevice");
        if (dev < 0 || dev >= 64 || !asked[dev]) {
            (void)dsv4_lds_optin((const void *)k_reqs_plan, 8 * 4097 * sizeof(int), "reqs plan");
            if (dev >= 0 && dev < 64) asked[dev] = true;
        }
    }
    hipLaunchKernelGGL(k_reqs_plan, dim3(1), dim3(RP_THREADS), lds, (hipStream_t)stream, a);
    HIP_OK(hipGetLastError(), "reqs plan launch");
    return 0;
}

extern "C" int dsv4_gpu_reqs_attn_d(void *d_o, const void *d_q, int fmt, int h, int d_qk, int d_v,
                                    const void *d_kv, const float *d_kv_scales, int kv_fmt,
                                    int kv_stride, int kv_rows, const dsv4_gpu_reqs *r,
                                    const void *d_plan, size_t plan_bytes, int window,
                                    const float *d_sink, float scale, void *d_scratch,
                                    size_t scratch_bytes, void *stream)
{
    const char *bad = reqs_bad(r, fmt, h, d_qk, d_v, kv_fmt, window);
    if (!bad && (kv_stride < d_qk || kv_rows <= 0)) bad = "a bad cache shape";
    if (!bad && r->max_tok && r->n_req &&
        (!d_o || !d_q || !d_kv || !r->pages || (kv_fmt == DSV4_GPU_KV_FP8 && !d_kv_scales)))
        bad = "a missing buffer";
    if (bad) {
        DSV4_ERR("reqs_attn: %s", bad);
        return -1;
    }
    if (r->max_tok == 0 || r->n_req == 0) return 0;
    const PlanParts pp = plan_parts(r->n_req, r->max_tok, h);
    const size_t need = dsv4_gpu_reqs_attn_scratch_bytes(fmt, h, d_qk, d_v, kv_fmt, r->n_req,
                                                         r->max_tok);
    if (!d_plan || ((uintptr_t)d_plan & 15) || plan_bytes < pp.bytes || !d_scratch ||
        ((uintptr_t)d_scratch & 15) || scratch_bytes < need) {
        DSV4_ERR("reqs_attn: a plan of %zu bytes at %p and %zu bytes of workspace at %p; the call "
                 "needs %zu and %zu, 16-byte aligned", plan_bytes, d_plan, scratch_bytes,
                 d_scratch, pp.bytes, need);
        return -1;
    }
    const ReqsRoom m = reqs_room(r->n_req, r->max_tok, h);
    const IoDiv pd((uint32_t)r->page_rows);
    const int es = fmt == DSV4_WBF16 ? 2 : 4, kc = dsv4_tree_chunks(d_qk, d_v);
    const char *p = (const char *)d_plan;
    Dsv4ReqsJob a{};
    a.o = d_o;
    a.q = d_q;
    a.h = h;
    a.dqk = d_qk;
    a.dv = d_v;
    a.kv = d_kv;
    a.ks = d_kv_scales;
    a.stride = kv_stride;
    a.rows = kv_rows;
    a.pages = r->pages;
    a.n_pages = r->max_pages;
    a.page = r->page_rows;
    a.page_m = pd.m;
    a.page_s = pd.s;
    a.window = window;
    a.sink = d_sink;
    a.scale = scale;
    a.dvp = (d_v + 15) / 16 * 16;
    a.pm = (float *)d_scratch;
    a.pl = a.pm + m.parts;
    a.part = a.pl + m.parts;
    a.vec = d_qk % 8 == 0 && kv_stride % 8 == 0 && ((uintptr_t)d_kv & 15) == 0;
    a.qvec = d_qk % 8 == 0 && ((uintptr_t)d_q & 15) == 0;
    a.ovec = d_v % 4 == 0 && (uintptr_t)d_o % (4 * es) == 0;
    a.head = (const Dsv4ReqsHead *)p;
    a.items = (const Dsv4ReqsItem *)(p + pp.items);
    a.req = (const Dsv4ReqsReq *)(p + pp.req);
    a.n_req = r->n_req;
    a.sig = reqs_sig(r, fmt, h, d_qk, d_v, kv_fmt, window);
    hipStream_t st = (hipStream_t)stream;
    /* a workgroup for every item that there may be: blocks of 16 rows by tiles */
    const long long tiles = (long long)r->max_pages * r->page_rows / TR_TILE + 2;
    long long groups = (2 * (m.rows / 16) + r->n_req + 1) * tiles;
    const int items = reqs_items(m, r->n_req, dsv4_tree_block_rows(fmt, kv_fmt, kc));
    if (groups > items) groups = items;
    const int rc = kv_fmt == DSV4_GPU_KV_F32 ? dsv4_reqs_f32_launch(a, fmt, kc, (unsigned)groups, st)
                 : kv_fmt == DSV4_GPU_KV_BF16
                     ? dsv4_reqs_bf16_launch(a, fmt, kc, (unsigned)groups, st)
                     : dsv4_reqs_fp8_launch(a, fmt, kc, (unsigned)groups, st);
    if (rc != 0) return rc;
    const JoinJob j{a.head, a.req, a.part, a.pm, a.pl, d_sink, r->n_req, h, d_v, a.dvp, a.ovec, m.rows,
                    IoDiv((uint32_t)h), a.sig};
    if (fmt == DSV4_WF32) join_launch(j, (float *)d_o, st);
    else join_launch(j, (uint16_t *)d_o, st);
    HIP_OK(hipGetLastError(), "reqs join launch");
    return 0;
}
