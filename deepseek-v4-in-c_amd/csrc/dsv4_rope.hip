/* SPDX-License-Identifier: Apache-2.0 */
/* dsv4_rope.hip - rotary positions for the heads of many tokens on gfx950.
 *
 * A pair (a, b) of the rotated part becomes (a c - b s, a s + b c), c and s
 * the table's entries for the pair at the token's position (the reference's
 * dsv4_rope.c:105-119 in its neighbour layout; the half layout pairs i with i
 * + dim/2). The two products and the sum are rounded one by one, as the
 * attention block's are, so both rotate to the same bits.
 *
 * Bound: the element stream, read and written once; the tables are dim/2
 * pairs per token against heads * head_dim elements and come from L2. A thread
 * owns one 16-byte piece (neighbours) or two pieces dim/2 apart (halves) of a
 * head, so a pair's elements meet in one thread and d_out may be d_x. Where a
 * head has elements outside the rotated part and d_out is not d_x, further
 * threads copy them. 4099 tokens of 64 heads of 128, bf16: 26.5 us (halves) and
 * 27.6 us (pairs) from HBM, 5.1 TB/s, over a large copy's rate; a head or a part
 * that is not whole pieces goes element by element (60 rotated elements of the
 * 128: 100 us, 64 of them 29). Four heads a thread, to read the tables' entries
 * once for them, were slower nearly everywhere (31.1 us against 26.7 for these
 * tokens, 4.2 against 2.7 for one).
 */
#include "dsv4_dev.h"
#include "dsv4_internal.h"

namespace {

#include "dsv4_rows_io.h"

constexpr int RO_THREADS = 256;

struct RopeJob {
    const void *x;
    void *out;
    long long xs, os;
    const int *pos;
    const float *cos, *sin;
    int items, hd, max_pos, half, off, inverse;
    int nrot;                    /* a head's rotated units; copied ones follow */
    IoDiv units, heads;
};

/* V: elements per piece (16 bytes at any address, or 1 where a head or its
 * rotated part is not whole pieces). */
template <class T, int V, bool HALVES>
__global__ void __launch_bounds__(RO_THREADS) k_rope(RopeJob a)
{
    constexpr int W = HALVES ? V : (V > 1 ? V / 2 : 1);      /* pairs per unit */
    const uint32_t i = blockIdx.x * RO_THREADS + threadIdx.x;
    if (i >= (uint32_t)a.items) return;
    const uint32_t q = a.units.div(i);
    const int u = (int)(i - q * a.units.d);
    const int t = (int)a.heads.div(q), h = (int)(q - (uint32_t)t * a.heads.d);
    const T *x = (const T *)a.x + t * a.xs + (long long)h * a.hd;
    T *o = (T *)a.out + t * a.os + (long long)h * a.hd;
    if (u >= a.nrot) {                                       /* copied as it is */
        int c = (u - a.nrot) * V;
        if (c >= a.off) c += 2 * a.half;
        float v[V];
        io_load<T, V>(x + c, v);
        io_store<T, V>(o + c, v);
        return;
    }
    const int p = a.pos[t];
    const int c0 = a.off + (HALVES ? u * W : 2 * u * W);
    float v[2 * W], cs[W], sn[W];
    if constexpr (HALVES) {
        io_load<T, W>(x + c0, v);
        io_load<T, W>(x + c0 + a.half, v + W);
    } else {
        io_load<T, 2 * W>(x + c0, v);
    }
    if (p >= 0 && p < a.max_pos) {
        const size_t r = (size_t)p * a.half + u * W;
        io_load<float, W>(a.cos + r, cs);
        io_load<float, W>(a.sin + r, sn);
    } else {
#pragma unroll
        for (int k = 0; k < W; k++) cs[k] = sn[k] = __uint_as_float(0x7FC00000u);
    }
#pragma unroll
    for (int k = 0; k < W; k++) {
        if (a.inverse) sn[k] = -sn[k];
        float &e0 = HALVES ? v[k] : v[2 * k];
        float &e1 = HALVES ? v[W + k] : v[2 * k + 1];
        const float x0 = e0, x1 = e1;
        e0 = x0 * cs[k] - x1 * sn[k];
        e1 = x0 * sn[k] + x1 * cs[k];
    }
    if constexpr (HALVES) {
        io_store<T, W>(o + c0, v);
        io_store<T, W>(o + c0 + a.half, v + W);
    } else {
        io_store<T, 2 * W>(o + c0, v);
    }
}

template <class T, int V>
void rope_launch(const RopeJob &a, int layout, hipStream_t st)
{
    const dim3 grid((a.items + RO_THREADS - 1) / RO_THREADS);
    if (layout == DSV4_GPU_ROPE_HALVES)
        hipLaunchKernelGGL((k_rope<T, V, true>), grid, dim3(RO_THREADS), 0, st, a);
    else
        hipLaunchKernelGGL((k_rope<T, V, false>), grid, dim3(RO_THREADS), 0, st, a);
}

} // namespace

const char *dsv4_rope_bad(const dsv4_gpu_rope *r, int head_dim)
{
    if (!r || !r->cos || !r->sin) return "no table";
    if (r->max_pos <= 0) return "an empty table";
    if (r->dim <= 0 || (r->dim & 1)) return "an odd or empty rotated part";
    if (r->offset < 0 || r->offset > head_dim || r->dim > head_dim - r->offset)
        return "a rotated part outside the head";
    if (r->layout != DSV4_GPU_ROPE_PAIRS && r->layout != DSV4_GPU_ROPE_HALVES)
        return "an unknown layout";
    return nullptr;
}

extern "C" int dsv4_gpu_rope_n_d(void *d_out, long long out_stride, const void *d_x,
                                 long long x_stride, int fmt, const int *d_pos, int nt, int heads,
                                 int head_dim, const dsv4_gpu_rope *rope, int inverse,
                                 void *stream)
{
    const long long width = (long long)heads * head_dim;
    if (nt < 0 || nt > 1 << 30 || heads <= 0 || head_dim <= 0 || x_stride < width ||
        out_stride < width || width > INT32_MAX / 2 ||
        (fmt != DSV4_WF32 && fmt != DSV4_WBF16)) {
        DSV4_ERR("rope: bad arguments (nt %d, heads %d, head_dim %d, fmt %d, strides %lld, %lld)",
                 nt, heads, head_dim, fmt, x_stride, out_stride);
        return -1;
    }
    if (const char *bad = dsv4_rope_bad(rope, head_dim)) {
        DSV4_ERR("rope: %s", bad);
        return -1;
    }
    const bool here = d_out == d_x;
    if (nt == 0) return 0;
    if (!d_out || !d_x || !d_pos || (here && x_stride != out_stride)) {
        DSV4_ERR("rope: %s", here && d_x ? "in place with two strides" : "a missing buffer");
        return -1;
    }
    const int half = rope->dim / 2, es = fmt == DSV4_WBF16 ? 2 : 4;
    const bool halves = rope->layout == DSV4_GPU_ROPE_HALVES;
    int V = 16 / es;
    if (head_dim % V || rope->offset % V || (halves ? half : rope->dim) % V) V = 1;
    const int nrot = halves ? half / V : V > 1 ? rope->dim / V : half;
    const int units = nrot + (here ? 0 : (head_dim - rope->dim) / V);
    /* a launch's items stay below 2^30 */
    const long long per = (long long)units * heads;
    const int most = (int)((1ll << 30) / per);
    for (int t0 = 0; t0 < nt; t0 += most) {
        const int n = nt - t0 < most ? nt - t0 : most;
        RopeJob a{(const char *)d_x + (size_t)t0 * x_stride * es,
                  (char *)d_out + (size_t)t0 * out_stride * es, x_stride, out_stride,
                  d_pos + t0, rope->cos, rope->sin, (int)(n * per), head_dim,
                  rope->max_pos, half, rope->offset, inverse != 0, nrot,
                  IoDiv((uint32_t)units), IoDiv((uint32_t)heads)};
        hipStream_t st = (hipStream_t)stream;
        if (es == 4) {
            if (V > 1) rope_launch<float, 4>(a, rope->layout, st);
            else rope_launch<float, 1>(a, rope->layout, st);
        } else {
            if (V > 1) rope_launch<uint16_t, 8>(a, rope->layout, st);
            else rope_launch<uint16_t, 1>(a, rope->layout, st);
        }
        HIP_OK(hipGetLastError(), "rope launch");
    }
    return 0;
}
