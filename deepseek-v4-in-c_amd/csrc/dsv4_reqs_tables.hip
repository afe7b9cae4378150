/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_reqs_tables.hip - page tables and row maps of a batch's step, from the
 * requests' lengths, on gfx950.
 *
 * With L positions in use and n new tokens request i needs ceil((L + n) / P) -
 * ceil(L / P) pages of P rows. Inclusive sums over the requests of the needs, then
 * of the tokens of those whose needs are met, say who is served; the exclusive
 * ones are the place of its first new page behind the ring's first and of its
 * first token in the batch. A token finds its request by a binary search of the
 * first tokens, and a page that is new in the ring directly, so no token waits for
 * a table entry that another writes.
 *
 * Bound: latency, a chain of one load, two scans of the workgroup and the search
 * (12 n_tok bytes are written). Each workgroup makes the sums of all requests for
 * itself in LDS rather than wait for a launch that does. 64 requests of a token 7.8
 * us; 1000 requests with about 40000 tokens 11.7, and 6 for a launch of the state's own.
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

namespace {

#include "dsv4_rows_io.h"

constexpr int RT_REQS = 4096;
constexpr int RT_MAX = 0x7FFFFFFF;
constexpr int RT_TOKENS = 4;                      /* a thread's, neighbours  */

struct TablesJob {
    const int *len_in, *add;
    int *len, *pages, *first;
    int n_req, max_pages, max_tok, shared;        /* shared: whole pages     */
    int *ring;
    int cap;
    const int *free_in;
    int *free_out, *rows, *pos, *req;
    IoDiv page;
};

/* Sums of counts that may not fit stop at 2^31 - 1, more than any limit they are
 * compared with; so they stay associative. */
__device__ __forceinline__ int rt_add(int a, int b)
{
    const uint32_t s = (uint32_t)a + (uint32_t)b;
    return s > (uint32_t)RT_MAX ? RT_MAX : (int)s;
}

/* The sum of lanes 0 to this one's, by moves within the vector unit. */
template <int CTRL, int ROWS>
__device__ __forceinline__ int rt_moved(int v)
{
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int rt_wave_scan(int v)
{
    v = rt_add(v, rt_moved<0x111, 0xF>(v));       /* row_shr:1, 2, 4, 8      */
    v = rt_add(v, rt_moved<0x112, 0xF>(v));
    v = rt_add(v, rt_moved<0x114, 0xF>(v));
    v = rt_add(v, rt_moved<0x118, 0xF>(v));
    v = rt_add(v, rt_moved<DPP_ROW_BCAST15, 0xA>(v));
    return rt_add(v, rt_moved<DPP_ROW_BCAST31, 0xC>(v));
}
/* The largest of all lanes' v, none of them negative, in lane 63. */
__device__ __forceinline__ int rt_wave_top(int v)
{
    v = max(v, rt_moved<DPP_QUAD_XOR1, 0xF>(v));
    v = max(v, rt_moved<DPP_QUAD_XOR2, 0xF>(v));
    v = max(v, rt_moved<DPP_ROW_HMIRROR, 0xF>(v));
    v = max(v, rt_moved<DPP_ROW_MIRROR, 0xF>(v));
    v = max(v, rt_moved<DPP_ROW_BCAST15, 0xA>(v));
    return max(v, rt_moved<DPP_ROW_BCAST31, 0xC>(v));
}

/* Exclusive sums of a and b over the workgroup's threads. */
template <int W>
__device__ __forceinline__ void rt_scan(int &a, int &b, int (*part)[2])
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int x = rt_wave_scan(a), y = rt_wave_scan(b);
    __syncthreads();                              /* part was read           */
    if (lane == 63) {
        part[w][0] = x;
        part[w][1] = y;
    }
    const int u = __shfl_up(x, 1, 64), v = __shfl_up(y, 1, 64);
    a = lane ? u : 0;
    b = lane ? v : 0;
    __syncthreads();
    for (int k = 0; k < w; k++) {
        a = rt_add(a, part[k][0]);
        b = rt_add(b, part[k][1]);
    }
}

/* The largest of a and of b over the workgroup. */
template <int W>
__device__ __forceinline__ void rt_top(int &a, int &b, int (*part)[2])
{
    a = rt_wave_top(a);
    b = rt_wave_top(b);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) {
        part[threadIdx.x >> 6][0] = a;
        part[threadIdx.x >> 6][1] = b;
    }
    __syncthreads();
    for (int k = 0; k < W; k++) {
        a = max(a, part[k][0]);
        b = max(b, part[k][1]);
    }
}

/* tokens: this launch writes the maps, the new entries and the ended requests'
 * pages; state: the first workgroup writes the lengths, first tokens and the ring's
 * place (after every read of the old ones, where it may write over them). */
template <int THREADS>
__global__ void __launch_bounds__(THREADS) k_reqs_tables(TablesJob a, bool tokens, bool state)
{
    constexpr int W = THREADS / 64;
    extern __shared__ int lds[];
    __shared__ int part[W][2];
    int *first = lds, *have = lds + a.n_req + 1, *place = have + a.n_req;
    const int tid = threadIdx.x, n = a.n_req, per = (n + THREADS - 1) / THREADS;
    const int i0 = min(n, tid * per), i1 = min(n, i0 + per);
    const int cap = a.cap, room = a.max_pages * (int)a.page.d;
    int head = a.free_in[0], count = a.free_in[1];
    head = (uint32_t)head < (uint32_t)cap ? head : 0;
    count = max(0, min(count, cap));
    auto up = [&](int p) { return (int)a.page.div((uint32_t)p + a.page.d - 1); };
    /* positions in use that the table holds, of a request that ends */
    auto own = [&](int L) { return max(0, up(max(0, min(L, room))) - a.shared); };

    int need = 0, back = 0;
    for (int i = i0; i < i1; i++) {
        const int L = a.len_in[i], add = a.add[i];
        have[i] = L;
        const bool fits = add > 0 && L >= 0 && L <= room && add <= room - L;
        if (fits) need = rt_add(need, up(L + add) - up(L));
        if (add < 0) back = rt_add(back, own(L));
    }
    int need0 = need, back0 = back;
    rt_scan<W>(need0, back0, part);
    /* those with their pages: their tokens; place: of a request's first page */
    int sum = need0, tok = 0, bk = back0;
    for (int i = i0; i < i1; i++) {
        const int L = have[i], add = a.add[i];
        const bool fits = add > 0 && L >= 0 && L <= room && add <= room - L;
        const int k = fits ? up(L + add) - up(L) : 0;
        place[i] = add < 0 ? bk : sum;
        sum = rt_add(sum, k);
        const bool paged = fits && (k == 0 || sum <= count);
        first[i] = paged ? add : 0;
        if (paged) tok = rt_add(tok, add);
        if (add < 0) bk = rt_add(bk, own(L));
    }
    int tok0 = tok, none = 0;
    rt_scan<W>(tok0, none, part);
    int total = 0, taken = 0;                     /* tokens and pages served */
    sum = tok0;
    for (int i = i0; i < i1; i++) {
        const int add = first[i], at = sum;
        sum = rt_add(sum, add);
        const bool served = add > 0 && sum <= a.max_tok;
        if (served) {
            const int L = have[i], k = up(L + add) - up(L);
            total = sum;
            if (k) taken = place[i] + k;
        }
        first[i] = served ? at : -1 - at;         /* negative: without tokens */
    }
    rt_top<W>(total, taken, part);
    /* a request without tokens starts where the next one with some does */
    for (int i = i0; i < i1; i++) {
        const int at = first[i];
        first[i] = at >= 0 ? at : min(-1 - at, total);
    }
    int none2 = back, all_back = rt_add(back0, back);
    rt_top<W>(all_back, none2, part);             /* inclusive sums ascend   */
    all_back = min(all_back, cap - count);
    if (tid == 0) first[n] = total;
    __syncthreads();

    if (tokens) {
        const int step = gridDim.x * THREADS * RT_TOKENS;
        for (int t0 = (blockIdx.x * THREADS + tid) * RT_TOKENS; t0 < a.max_tok; t0 += step) {
            int lo = 0, hi = n;                   /* first[lo] <= t0 < first[hi] */
            if (t0 < total)
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (first[mid] <= t0) lo = mid;
                    else hi = mid;
                }
#pragma unroll
            for (int u = 0; u < RT_TOKENS; u++) {
                const int t = t0 + u;
                if (t >= a.max_tok) break;
                int row = -1, pos = -1, req = -1;
                if (t < total) {
                    while (first[lo + 1] <= t) lo++;
                    req = lo;
                    const int L = have[req], fresh = up(L);
                    pos = L + t - first[req];
                    const int e = (int)a.page.div((uint32_t)pos), off = pos - e * (int)a.page.d;
                    int *entry = a.pages + (size_t)req * a.max_pages + e;
                    int page;
                    if (e >= fresh) {
                        /* place and the entry's number are below count <= cap */
                        int at = head + place[req] + (e - fresh);
                        at -= at >= cap ? cap : 0;
                        page = a.ring[at];
                        if (off == 0) *entry = page;
                    } else {
                        page = *entry;
                    }
                    const long long r = (long long)page * a.page.d + off;
                    row = page >= 0 && r < RT_MAX ? (int)r : -1;
                }
                if (a.rows) a.rows[t] = row;
                if (a.pos) a.pos[t] = pos;
                if (a.req) a.req[t] = req;
            }
        }
        /* a wave for an ended request's pages */
        for (int i = blockIdx.x * W + (tid >> 6); i < n; i += gridDim.x * W) {
            if (a.add[i] >= 0) continue;
            const int k = own(have[i]);
            for (int j = tid & 63; j < k; j += 64) {
                const int b = rt_add(place[i], j);
                if (b >= all_back) break;
                int at = head + count;
                at -= at >= cap ? cap : 0;
                at += b;
                at -= at >= cap ? cap : 0;
                a.ring[at] = a.pages[(size_t)i * a.max_pages + a.shared + j];
            }
        }
    }
    if (state && blockIdx.x == 0) {
        for (int i = tid; i <= n; i += THREADS) a.first[i] = first[i];
        for (int i = tid; i < n; i += THREADS)
            a.len[i] = a.add[i] < 0 ? 0 : have[i] + first[i + 1] - first[i];
        if (tid == 0) {
            int at = head + taken;
            at -= at >= cap ? cap : 0;
            a.free_out[0] = at;
            a.free_out[1] = count - taken + all_back;
        }
    }
}

} // namespace

const char *dsv4_reqs_bad(const dsv4_gpu_reqs *r)
{
    if (!r) return "no batch";
    if (r->n_req < 0 || r->n_req > RT_REQS) return "0 to 4096 requests are taken";
    if (r->page_rows <= 0 || r->max_pages <= 0 ||
        (long long)r->max_pages * r->page_rows > 1ll << 30)
        return "tables of 1 to 2^30 positions are taken";
    if (r->max_tok < 0 || r->max_tok > 1 << 20) return "0 to 2^20 tokens are taken";
    if (r->n_prefix < 0) return "a negative prefix";
    return nullptr;
}

extern "C" int dsv4_gpu_reqs_tables_d(const dsv4_gpu_reqs *r, const int *d_len, const int *d_new,
                                      int *d_ring, int ring_cap, const int *d_free,
                                      int *d_free_out, int *d_rows, int *d_pos, int *d_req,
                                      void *stream)
{
    const char *bad = dsv4_reqs_bad(r);
    if (!bad && (ring_cap <= 0 || ring_cap > 1 << 30)) bad = "a ring of 1 to 2^30 pages is taken";
    if (!bad && (!r->first || !d_free || !d_free_out || !d_ring ||
                 (r->n_req && (!r->len || !r->pages || !d_len || !d_new))))
        bad = "a missing buffer";
    if (bad) {
        DSV4_ERR("reqs_tables: %s", bad);
        return -1;
    }
    TablesJob a{d_len, d_new, r->len, r->pages, r->first, r->n_req, r->max_pages, r->max_tok,
                r->n_prefix / r->page_rows, d_ring, ring_cap, d_free, d_free_out, d_rows, d_pos,
                d_req, IoDiv((uint32_t)r->page_rows)};
    hipStream_t st = (hipStream_t)stream;
    const size_t lds = (3 * (size_t)r->n_req + 1) * sizeof(int);
    auto launch = [&](int groups, bool tokens, bool state) {
        if (r->n_req <= 256)
            hipLaunchKernelGGL(k_reqs_tables<256>, dim3(groups), dim3(256), lds, st, a, tokens,
                               state);
        else
            hipLaunchKernelGGL(k_reqs_tables<1024>, dim3(groups), dim3(1024), lds, st, a, tokens,
                               state);
        return hipGetLastError();
    };
    /* One launch, where it is one workgroup's or the state is not written over the old one
     * that others read; else the state after them (1000 requests with about 40000 tokens
     * 17 us, in one launch 11). */
    const int threads = r->n_req <= 256 ? 256 : 1024, each = threads * RT_TOKENS;
    const int groups = (r->max_tok + each - 1) / each;
    auto meet = [](const int *w, size_t nw, const int *v, size_t nv) {
        const uintptr_t a0 = (uintptr_t)w, b0 = (uintptr_t)v;
        return a0 < b0 + nv * sizeof(int) && b0 < a0 + nw * sizeof(int);
    };
    const size_t n = (size_t)r->n_req;
    const struct {
        const int *p;
        size_t n;
    } writes[3] = {{r->len, n}, {r->first, n + 1}, {d_free_out, 2}},
      reads[3] = {{d_len, n}, {d_new, n}, {d_free, 2}};
    bool over = false;
    for (const auto &w : writes)
        for (const auto &v : reads) over |= meet(w.p, w.n, v.p, v.n);
    if (groups <= 1 || !over) {
        HIP_OK(launch(groups < 1 ? 1 : groups < 256 ? groups : 256, true, true), "reqs tables launch");
        return 0;
    }
    HIP_OK(launch(groups < 256 ? groups : 256, true, false), "reqs tables launch");
    HIP_OK(launch(1, false, true), "reqs tables state launch");
    return 0;
}
