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

namespace {

#include "dsv4_rows_io.h"

constexpr int RP_THREADS = 1024;
constexpr int RP_SPLITS = 255;                    /* most of a request's, or of the prefix */
constexpr int RP_EXTRA = 1024;                    /* items for splits        */
constexpr int RP_ROWS = 65536, RP_PREFIX_ROWS = 262144;  /* rows of sums      */

/* What a batch's plan and workspace have room for. */
struct ReqsRoom {
    long long rows, items, blocks, parts;
};
ReqsRoom reqs_room(int n_req, int max_tok, int h)
{
    ReqsRoom m;
    m.rows = (long long)max_tok * h;
    /* blocks of 64 rows, the fewest that a workgroup takes at most, or of 16 */
    const long long few = m.rows / 16 + n_req, many = m.rows / 64 + n_req + RP_EXTRA;
    m.blocks = few < many ? few : many;
    m.items = 2 * (m.rows / 64) + n_req + 1 + RP_EXTRA;
    m.parts = RP_ROWS + (2 * m.rows < RP_PREFIX_ROWS ? 2 * m.rows : RP_PREFIX_ROWS);
    return m;
}

struct PlanJob {
    Dsv4ReqsHead *head;
    Dsv4ReqsBlock *blocks;
    Dsv4ReqsItem *items;
    int2 *req;
    const int *len, *first;
    int n_req, max_tok, h, window, prefix, room;  /* room: positions of a table */
    int br, br_split, per_cu, dvp;                /* most rows, waves a block of 16 */
    int max_items, max_blocks, max_parts;
    uint32_t sig;
};

/* A request's step: tokens, the position of the first, tiles behind the prefix's. */
struct PlanReq {
    int n, pos, tile0, tile1;
};
__device__ __forceinline__ PlanReq plan_req(const PlanJob &a, int b, int prefix_tiles)
{
    PlanReq r;
    r.n = a.first[b + 1] - a.first[b];
    const int len = a.len[b];
    r.pos = len - r.n;
    const int lo = a.window ? max(0, r.pos - a.window + 1) : 0;
    r.tile0 = max(prefix_tiles, lo / TR_TILE);
    r.tile1 = max(r.tile0, (len + TR_TILE - 1) / TR_TILE);
    return r;
}
__device__ __forceinline__ int plan_splits(int tiles, int each)
{
    return min((tiles + each - 1) / each, RP_SPLITS);
}

template <class V, class F>
__device__ __forceinline__ V wave_all(V v, F f)
{
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = f(v, __shfl_xor(v, o, 64));
    return v;
}

/* One workgroup. A plan is: with the prefix apart or not, the rows of a block and
 * the tiles of an item. 64 of them are priced as dsv4_tree.hip prices its own (in
 * halves of the time of a tile on a lone wave), the workgroups as rounds of the card
 * or as a stream of items that ends with the longest, whichever is less. */
__global__ void __launch_bounds__(RP_THREADS) k_reqs_plan(PlanJob a)
{
    extern __shared__ int lds[];
    __shared__ unsigned long long best, owner, work[8];
    __shared__ int bad, active, hi_min, lo_max, lo_min, longest[8];
    __shared__ int part_w[RP_THREADS / 64][3];
    __shared__ int rows_each, tiles_each, tiles_from;
    const int tid = threadIdx.x, lane = tid & 63;
    if (tid == 0) {
        best = ~0ull;
        owner = 0;
        bad = active = lo_max = 0;
        hi_min = lo_min = INT32_MAX;
    }
    if (tid < 8) {
        work[tid] = 0;
        longest[tid] = 0;
    }
    __syncthreads();
    const int tok0 = a.n_req ? a.first[0] : 0, tok1 = a.n_req ? a.first[a.n_req] : 0;
    {
        int b_bad = tok0 < 0 || tok1 > a.max_tok, n_act = 0, hmin = INT32_MAX, lmax = 0, lmin = INT32_MAX;
        unsigned long long own = 0;
        for (int b = tid; b < a.n_req; b += RP_THREADS) {
            const int f0 = a.first[b], f1 = a.first[b + 1], len = a.len[b], n = f1 - f0;
            if (f0 < 0 || f1 < f0 || f1 > a.max_tok || (n && (len < n || len > a.room))) {
                b_bad = 1;
                continue;
            }
            a.req[b] = int2{f0, len - n};
            if (!n) continue;
            n_act++;
            hmin = min(hmin, len - n + 1);
            lmax = max(lmax, a.window ? max(0, len - a.window) : 0);
            lmin = min(lmin, a.window ? max(0, len - n - a.window + 1) : 0);
            const unsigned long long o = (unsigned long long)len << 32 | (uint32_t)b;
            own = o > own ? o : own;
        }
        auto hi = [](auto x, auto y) { return x > y ? x : y; };
        auto lo = [](auto x, auto y) { return x < y ? x : y; };
        auto plus = [](int x, int y) { return x + y; };
        b_bad = wave_all(b_bad, hi);
        n_act = wave_all(n_act, plus);
        hmin = wave_all(hmin, lo);
        lmax = wave_all(lmax, hi);
        lmin = wave_all(lmin, lo);
        own = wave_all(own, hi);
        if (lane == 0) {
            if (b_bad) bad = 1;
            atomicAdd(&active, n_act);
            atomicMin(&hi_min, hmin);
            atomicMax(&lo_max, lmax);
            atomicMin(&lo_min, lmin);
            atomicMax(&owner, own);
        }
    }
    __syncthreads();
    const int R0 = tok0 * a.h, R = (tok1 - tok0) * a.h;
    if (bad || active == 0) {
        if (tid == 0) *a.head = Dsv4ReqsHead{bad ? ~a.sig : a.sig, 0, 0, 0, 0, 0, 0, 0};
        return;
    }
    /* whole tiles of the prefix, as far as the longest request has it */
    const int max_len = (int)(owner >> 32);
    const int pt1 = min(a.prefix, max_len) / TR_TILE, pt0 = min(pt1, lo_min / TR_TILE);
    const bool may = active > 1 && pt1 > pt0;

    /* group g (two waves): the prefix apart (g & 1), blocks of 16 << (g >> 1) rows */
    const int g = tid >> 7, gt = tid & 127, r = 16 << (g >> 1);
    const bool apart = g & 1, on = r <= a.br && (!apart || may);
    const int from = apart ? pt1 : 0, ptiles = apart ? pt1 - pt0 : 0;
    const int pblocks = apart ? (R + r - 1) / r : 0;
    if (on) {
        unsigned long long w = 0;
        int l = ptiles;
        for (int b = gt; b < a.n_req; b += 128) {
            const PlanReq q = plan_req(a, b, from);
            if (!q.n) continue;
            w += (unsigned long long)((q.n * a.h + r - 1) / r) * (q.tile1 - q.tile0);
            l = max(l, q.tile1 - q.tile0);
        }
        w = wave_all(w, [](auto x, auto y) { return x + y; });
        l = wave_all(l, [](int x, int y) { return max(x, y); });
        if (lane == 0) {
            atomicAdd(&work[g], w);
            atomicMax(&longest[g], l);
        }
    }
    __syncthreads();
    {
        /* tiles of an item, so that they are about so many workgroups' worth of the card */
        const int c = gt >> 4, cl = gt & 15;
        const unsigned long long w = work[g] + (unsigned long long)pblocks * ptiles;
        constexpr int SHARE[7] = {128, 256, 384, 512, 768, 1024, 1536};
        unsigned long long l = 1ull << 30;
        if (c < 7) l = (w + SHARE[c] - 1) / SHARE[c];
        const int each = (int)max(1ull, min(l, 1ull << 30));
        unsigned long long items = 0, blocks = 0, parts = 0;
        if (on) {
            for (int b = cl; b < a.n_req; b += 16) {
                const PlanReq q = plan_req(a, b, from);
                if (!q.n) continue;
                const int rows = q.n * a.h, nb = (rows + r - 1) / r;
                int ns = plan_splits(q.tile1 - q.tile0, each);
                if (!apart && ns < 1) ns = 1;
                items += (unsigned long long)nb * ns;
                blocks += nb;
                if (apart || ns > 1) parts += (unsigned long long)ns * rows;
            }
        }
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) {
            items += __shfl_xor(items, o, 64);
            blocks += __shfl_xor(blocks, o, 64);
            parts += __shfl_xor(parts, o, 64);
        }
        const int ps = plan_splits(ptiles, each);
        items += (unsigned long long)pblocks * ps;
        parts += (unsigned long long)ps * R * apart;
        if (on && cl == 0 && items <= (unsigned long long)a.max_items &&
            blocks <= (unsigned long long)a.max_blocks && parts <= (unsigned long long)a.max_parts) {
            const int waves = r / 16 * a.br_split;
            const float tile = waves > 4 ? 3.0f : 2.0f, start = 8.0f + 2.0f * waves;
            const float slots = 256.0f * a.per_cu, n = (float)items;
            const float one = (float)min(each, longest[g]) * tile + start;
            const float rounds = ceilf(n / slots) * one;
            const float flow = ((float)w * tile + n * start) / slots + one;
            const float cost = fminf(rounds, flow) + (parts ? 5.0f : 0.0f) +
                               (float)parts * (float)a.dvp * (1.0f / (1 << 20));
            /* a price over 0 orders as its bits do */
            atomicMin(&best, (unsigned long long)__float_as_uint(cost) << 32 | (uint32_t)(g << 3 | c));
        }
        __syncthreads();
        if ((int)(best & 63) == (g << 3 | c) && cl == 0) {
            rows_each = r;
            tiles_each = each;
            tiles_from = from;
        }
        __syncthreads();
    }
    const int br = rows_each, each = tiles_each, start = tiles_from;
    const int ps = start ? plan_splits(pt1 - pt0, each) : 0;
    const int pb = start ? (R + br - 1) / br : 0, pitems = ps * pb;

    /* where each request's items, blocks and sums begin */
    int *s_item = lds, *s_block = lds + a.n_req + 1, *s_part = s_block + a.n_req + 1;
    const int per = (a.n_req + RP_THREADS - 1) / RP_THREADS;
    const int b0 = min(a.n_req, tid * per), b1 = min(a.n_req, b0 + per);
    auto cut = [&](int b, int *n) {               /* items, blocks, rows of sums */
        const PlanReq q = plan_req(a, b, start);
        n[0] = n[1] = n[2] = 0;
        if (!q.n) return;
        const int rows = q.n * a.h;
        int ns = plan_splits(q.tile1 - q.tile0, each);
        if (!start && ns < 1) ns = 1;
        n[1] = (rows + br - 1) / br;
        n[0] = n[1] * ns;
        n[2] = start || ns > 1 ? ns * rows : 0;
    };
    int sum[3] = {0, 0, 0};
    for (int b = b0; b < b1; b++) {
        int n[3];
        cut(b, n);
        for (int k = 0; k < 3; k++) sum[k] += n[k];
    }
    int x[3] = {sum[0], sum[1], sum[2]};
#pragma unroll
    for (int o = 1; o < 64; o *= 2)
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const int v = __shfl_up(x[k], o, 64);
            if (lane >= o) x[k] += v;
        }
    if (lane == 63)
        for (int k = 0; k < 3; k++) part_w[tid >> 6][k] = x[k];
    __syncthreads();
    for (int k = 0; k < 3; k++) {
        x[k] -= sum[k];
        for (int w = 0; w < tid >> 6; w++) x[k] += part_w[w][k];
    }
    x[2] += ps * R;
    for (int b = b0; b < b1; b++) {
        int n[3];
        cut(b, n);
        s_item[b] = x[0];
        s_block[b] = x[1];
        s_part[b] = x[2];
        for (int k = 0; k < 3; k++) x[k] += n[k];
    }
    if (b0 < b1 && b1 == a.n_req) {
        s_item[b1] = x[0];
        s_block[b1] = x[1];
    }
    __syncthreads();
    const int items = s_item[a.n_req], blocks = s_block[a.n_req];
    if (tid == 0)
        *a.head = Dsv4ReqsHead{a.sig, pitems + items, pitems, blocks, ps, R0, R, 0};
    auto owner_of = [&](const int *base, int i) { /* the request with number i */
        int lo = 0, hi = a.n_req;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (base[mid] <= i) lo = mid;
            else hi = mid;
        }
        return lo;
    };
    /* (a request without items or blocks has the next one's numbers: the search ends
     * at the last of them, which has some) */
    for (int i = tid; i < blocks; i += RP_THREADS) {
        const int b = owner_of(s_block, i), blk = i - s_block[b];
        const PlanReq q = plan_req(a, b, start);
        const int rows = q.n * a.h;
        int ns = plan_splits(q.tile1 - q.tile0, each);
        if (!start && ns < 1) ns = 1;
        const bool direct = !start && ns == 1;
        a.blocks[i] = Dsv4ReqsBlock{a.first[b] * a.h + blk * br, min(br, rows - blk * br),
                                    direct ? -1 : s_part[b] + blk * br, rows, ns, {0, 0, 0}};
    }
    const bool all_see = hi_min >= pt1 * TR_TILE && lo_max == 0;
    for (int i = tid; i < pitems; i += RP_THREADS) {
        const int s = i / pb, blk = i - s * pb;
        Dsv4ReqsItem it{};
        it.row0 = R0 + blk * br;
        it.rows = min(br, R - blk * br);
        it.req = (int)(uint32_t)owner;
        it.tile0 = pt0 + (int)((long long)(pt1 - pt0) * s / ps);
        it.tile1 = pt0 + (int)((long long)(pt1 - pt0) * (s + 1) / ps);
        it.end = pt1 * TR_TILE;
        it.lo = all_see ? 0 : lo_max;
        it.hi = all_see ? INT32_MAX : hi_min;
        it.kind = all_see ? 0 : 2;
        it.part = s * R + blk * br;
        a.items[i] = it;
    }
    for (int i = tid; i < items; i += RP_THREADS) {
        const int b = owner_of(s_item, i), k = i - s_item[b];
        const PlanReq q = plan_req(a, b, start);
        const int rows = q.n * a.h, nb = (rows + br - 1) / br, s = k / nb, blk = k - s * nb;
        const int ns = (s_item[b + 1] - s_item[b]) / nb;
        Dsv4ReqsItem it{};
        it.rows = min(br, rows - blk * br);
        it.row0 = a.first[b] * a.h + blk * br;
        it.req = b;
        /* a block's first and last tokens bound what its rows see */
        const int p0 = q.pos + blk * br / a.h, p1 = q.pos + (blk * br + it.rows - 1) / a.h;
        const int t0 = max(q.tile0, a.window ? max(0, p0 - a.window + 1) / TR_TILE : 0);
        const int t1 = max(t0, p1 / TR_TILE + 1);
        it.tile0 = t0 + (int)((long long)(t1 - t0) * s / ns);
        it.tile1 = t0 + (int)((long long)(t1 - t0) * (s + 1) / ns);
        it.end = p1 + 1;
        it.lo = a.window ? max(0, p1 - a.window + 1) : 0;
        it.hi = p0 + 1;
        it.kind = 1;
        it.pos0 = p0;
        it.part = !start && ns == 1 ? -1 : s_part[b] + s * rows + blk * br;
        a.items[pitems + i] = it;
    }
}

constexpr int RJ_THREADS = 256, RJ_WAVES = RJ_THREADS / 64;

struct JoinJob {
    const Dsv4ReqsHead *head;
    const Dsv4ReqsBlock *blocks;
    const float *part, *pm, *pl, *sink;
    int h, dv, dvp, ovec;
    long long rows;                               /* of the whole buffer     */
    uint32_t sig;
};

/* Rows of a block whose sums lie in several places: the prefix's splits and then
 * the request's. Every wave has the weights, and adds every fourth place. */
template <class T>
__global__ void __launch_bounds__(RJ_THREADS) k_reqs_join(JoinJob a, T *o)
{
    __shared__ f32x4 sum[RJ_WAVES][TR_DV / 4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Dsv4ReqsHead hd = *a.head;
    if (hd.sig != a.sig) {                        /* not this call's plan    */
        const float nan = __uint_as_float(0x7FC00000u);
        const long long n = a.rows * a.dv, step = (long long)gridDim.x * gridDim.y * RJ_THREADS;
        for (long long i = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * RJ_THREADS + tid;
             i < n; i += step)
            io_store<T, 1>(o + i, &nan);
        return;
    }
    if ((int)blockIdx.x >= hd.blocks) return;
    const Dsv4ReqsBlock b = a.blocks[blockIdx.x];
    if (b.part < 0) return;
    const int ps = hd.prefix_splits, n = ps + b.splits;
    for (int i = blockIdx.y; i < b.rows; i += gridDim.y) {
        const int r = b.row0 + i;
        auto place = [&](int s) {
            return s < ps ? (size_t)s * hd.rows + (r - hd.row0)
                          : (size_t)b.part + (size_t)(s - ps) * b.stride + i;
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
        m = wave_max(m);
#pragma unroll
        for (int k = 0; k < NK; k++) {
            if (64 * k >= n) break;
            ms[k] = tree_join_weight(ms[k], ls[k], m);
            l += ms[k] * ls[k];
        }
        l = wave_sum(l);
        if (a.sink && l != 0.0f)
            l += __builtin_amdgcn_exp2f(a.sink[r % a.h] * 1.44269504088896340736f - m);
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        f32x4 v[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int k = 0; k < NK; k++) {
            if (64 * k >= n) break;
            for (int s = 64 * k + w; s < min(n, 64 * k + 64); s += RJ_WAVES) {
                const float e = __shfl(ms[k], s & 63, 64);
                const float *p = a.part + place(s) * a.dvp + 4 * lane;
#pragma unroll
                for (int c = 0; c < 2; c++)
                    if (256 * c + 4 * lane < a.dvp) v[c] += e * ldf4(p + 256 * c);
            }
        }
        sum[w][lane] = v[0];
        sum[w][64 + lane] = v[1];
        __syncthreads();
        if (tid < TR_DV / 4 && 4 * tid < a.dv) {
            f32x4 t = sum[0][tid];
#pragma unroll
            for (int k = 1; k < RJ_WAVES; k++) t += sum[k][tid];
            t = t * inv;
            const float y[4] = {t.x, t.y, t.z, t.w};
            T *d = o + (size_t)r * a.dv + 4 * tid;
            if (a.ovec) {
                io_store<T, 4>(d, y);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (4 * tid + e < a.dv) io_store<T, 1>(d + e, y + e);
            }
        }
        __syncthreads();
    }
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

/* A plan's arguments in 32 bits, not 0 or all ones' complement of another's by chance
 * only: it says that a plan is this call's, and is no protection. */
uint32_t reqs_sig(const dsv4_gpu_reqs *r, int fmt, int h, int d_qk, int d_v, int kv_fmt,
                  int window)
{
    const int v[] = {r->n_req, r->max_pages, r->page_rows, r->max_tok, r->n_prefix, fmt, h,
                     dsv4_tree_chunks(d_qk, d_v), (d_v + 15) / 16, kv_fmt, window};
    uint64_t x = 0x9E3779B97F4A7C15ull;
    for (const int k : v) {
        x = (x ^ (uint32_t)k) * 0xD6E8FEB86659FD93ull;
        x ^= x >> 32;
    }
    return (uint32_t)x;
}

struct PlanParts {
    size_t blocks, items, req, bytes;
};
PlanParts plan_parts(int n_req, int max_tok, int h)
{
    const ReqsRoom m = reqs_room(n_req, max_tok, h);
    PlanParts p;
    p.blocks = 64;
    p.items = p.blocks + (size_t)m.blocks * sizeof(Dsv4ReqsBlock);
    p.req = p.items + (size_t)m.items * sizeof(Dsv4ReqsItem);
    p.bytes = (p.req + (size_t)n_req * sizeof(int2) + 15) / 16 * 16;
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
    PlanJob a{};
    a.head = (Dsv4ReqsHead *)p;
    a.blocks = (Dsv4ReqsBlock *)(p + pp.blocks);
    a.items = (Dsv4ReqsItem *)(p + pp.items);
    a.req = (int2 *)(p + pp.req);
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
    a.max_items = (int)m.items;
    a.max_blocks = (int)m.blocks;
    a.max_parts = (int)m.parts;
    a.sig = reqs_sig(r, fmt, h, d_qk, d_v, kv_fmt, window);
    hipLaunchKernelGGL(k_reqs_plan, dim3(1), dim3(RP_THREADS),
                       3 * ((size_t)r->n_req + 1) * sizeof(int), (hipStream_t)stream, a);
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
    a.req = (const int2 *)(p + pp.req);
    a.n_req = r->n_req;
    a.sig = reqs_sig(r, fmt, h, d_qk, d_v, kv_fmt, window);
    hipStream_t st = (hipStream_t)stream;
    /* a workgroup for every item that there may be: blocks of 16 rows by tiles */
    const long long tiles = (long long)r->max_pages * r->page_rows / TR_TILE + 2;
    long long groups = (2 * (m.rows / 16) + r->n_req + 1) * tiles;
    if (groups > m.items) groups = m.items;
    const int rc = kv_fmt == DSV4_GPU_KV_F32 ? dsv4_reqs_f32_launch(a, fmt, kc, (unsigned)groups, st)
                 : kv_fmt == DSV4_GPU_KV_BF16
                     ? dsv4_reqs_bf16_launch(a, fmt, kc, (unsigned)groups, st)
                     : dsv4_reqs_fp8_launch(a, fmt, kc, (unsigned)groups, st);
    if (rc != 0) return rc;
    const JoinJob j{a.head, (const Dsv4ReqsBlock *)(p + pp.blocks), a.part, a.pm, a.pl, d_sink, h,
                    d_v, a.dvp, a.ovec, m.rows, a.sig};
    const long long y = 4096 / m.blocks;
    const dim3 grid((unsigned)m.blocks, (unsigned)(y < 8 ? 8 : y > 64 ? 64 : y));
    if (fmt == DSV4_WF32)
        hipLaunchKernelGGL(k_reqs_join<float>, grid, dim3(RJ_THREADS), 0, st, j, (float *)d_o);
    else
        hipLaunchKernelGGL(k_reqs_join<uint16_t>, grid, dim3(RJ_THREADS), 0, st, j,
                           (uint16_t *)d_o);
    HIP_OK(hipGetLastError(), "reqs join launch");
    return 0;
}
