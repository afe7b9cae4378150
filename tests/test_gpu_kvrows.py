"""Cache rows written from device rows (dsv4_gpu_kv_append_d) and read back
(dsv4_gpu_kv_read_d) against their definition in 64 bits. Without a rotation
the stored values are exact: scaling is by a power of two and each element is
rounded once, to nearest even."""
import ctypes

import numpy as np
import pytest

import common
import draft_common as dc

pytestmark = pytest.mark.gpu


def _append(dsv4, cache, ks, fmt, stride, rows, x, bf, xs, n, dim, at=None, row0=0, rp=None,
            pos=None):
    return dsv4.lib().dsv4_gpu_kv_append_d(
        cache.data_ptr(), dc.ptr(ks), fmt, stride, rows, x.data_ptr(), int(bf), xs, n, dim,
        dc.ptr(at), row0, None if rp is None else ctypes.byref(rp), dc.ptr(pos), dc.stream())


def _read(dsv4, out, bf, os_, cache, ks, fmt, stride, rows, n, dim, at=None, row0=0):
    return dsv4.lib().dsv4_gpu_kv_read_d(out.data_ptr(), int(bf), os_, cache.data_ptr(),
                                         dc.ptr(ks), fmt, stride, rows, dc.ptr(at), row0, n, dim,
                                         dc.stream())


def _rows(rng, n, d):
    """Rows of very different sizes, with the values where rounding turns."""
    x = (rng.standard_normal((n, d)) * np.exp2(rng.integers(-40, 40, (n, 1)))).astype(np.float32)
    if n > 6:
        x[0] = 0
        x[1, :] = 1e-42                                   # subnormal throughout
        x[2, :] = 0
        x[2, 0] = 448.0 * 2.0 ** 5                        # scale exactly 2^5
        x[3, :] = 0
        x[3, 0] = np.nextafter(np.float32(448.0), np.float32(500.0))   # just over: 2^1
        x[4, 0] = 3.0e38
        x[5, :d // 2] = (np.arange(d // 2) % 448 + 0.5) * 2.0 ** -9    # ties
        x[5, d // 2:] = 0
        x[5, -1] = 448.0
    return x


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("n,d", [(1, 576), (13, 33), (9, 512), (300, 72), (7, 1024), (5, 2051)])
def test_append_and_read_are_exact(gpu, dsv4, fmt, bf, n, d):
    import torch
    rng = np.random.default_rng(n * 7 + d)
    x = _rows(rng, n, d)
    x = dc.bf16(x) if bf else x
    rows, stride = n + 5, d + (3 if d % 2 else 16)
    old = rng.standard_normal((rows, stride)).astype(np.float32)
    old_v, old_s = dc.stored(old, fmt)
    cache, ks = dc.cache_of(old_v, fmt, scales=old_s)
    at = rng.permutation(rows)[:n].astype(np.int32)
    dat, dx = dc.dev(at), dc.to_fmt(x, bf)
    assert _append(dsv4, cache, ks, fmt, stride, rows, dx, bf, d, n, d, dat) == 0
    want_v, want_s = dc.stored(x, fmt)
    codes = cache.view(torch.float8_e4m3fn).float() if fmt == 2 else cache.float()
    codes = codes.cpu().numpy().astype(np.float64)
    full = old_v / old_s[:, None] if fmt == 2 else old_v.copy()
    full[at, :d] = want_v / want_s[:, None] if fmt == 2 else want_v
    assert np.array_equal(codes, full)                    # the rest of the cache too
    if fmt == 2:
        s = old_s.copy()
        s[at] = want_s
        assert np.array_equal(ks.cpu().numpy(), s.astype(np.float32))
    # back, in either type, out of order and with rows that are not there
    ask = np.concatenate([at[::-1], [-1, rows, 2 ** 31 - 1, -2 ** 31]]).astype(np.int32)
    dask = dc.dev(ask)
    for obf in (False, True):
        os_ = d + (8 if d % 8 == 0 else 1)
        out = torch.full((len(ask), os_), 9.0, device="cuda:0",
                         dtype=torch.bfloat16 if obf else torch.float32)
        assert _read(dsv4, out, obf, os_, cache, ks, fmt, stride, rows, len(ask), d, dask) == 0
        got = dc.host(out)
        want = np.concatenate([want_v[::-1], np.zeros((4, d))]).astype(np.float32)
        want = dc.bf16(want) if obf else want
        assert np.array_equal(got[:, :d], want) and (got[:, d:] == 9).all()


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("d,dim,off", [(576, 64, 512), (512, 64, 448), (90, 30, 7), (1000, 200, 400)])
def test_append_rotates(gpu, dsv4, fmt, halves, d, dim, off):
    """Rotated first: off by the f32 arithmetic's bound and half a step of the
    format (e4m3: 2^-4 of the element, or 2^-10 of the scale below 2^-6)."""
    rng = np.random.default_rng(d + dim)
    n, rows = 21, 40
    x = rng.standard_normal((n, d)).astype(np.float32)
    cos, sin = dc.tables(33, dim)
    pos = rng.integers(0, 33, n).astype(np.int32)
    dcos, dsin, dpos, dx = dc.dev(cos), dc.dev(sin), dc.dev(pos), dc.dev(x)
    rp = dc.rope_struct(dsv4, dcos, dsin, dim, off, halves)
    v, s = dc.stored(np.ones((rows, d)), fmt)
    cache, ks = dc.cache_of(v, fmt, scales=s)
    assert _append(dsv4, cache, ks, fmt, d, rows, dx, False, d, n, d, None, 11, rp, dpos) == 0
    got = dc.cache_values(cache, fmt, ks)
    want, slack = dc.rotate(x[:, None, :], cos, sin, pos, off, dim, halves)
    want, slack = want[:, 0], slack[:, 0]
    if fmt == 1:
        slack = slack + dc.U16 * (np.abs(want) + slack)
    if fmt == 2:
        step = dc.row_scales(want)[:, None]
        slack = slack + np.maximum(2.0 ** -4 * (np.abs(want) + slack), 2.0 ** -10 * step)
    assert (np.abs(got[11:11 + n] - want) <= slack).all()
    assert np.array_equal(got[:11], v[:11]) and np.array_equal(got[11 + n:], v[11 + n:])


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_infinities_and_nan(gpu, dsv4, fmt):
    """FP8 stores them as NaN under the finite elements' scale; the other
    formats keep them. A position outside the table gives NaN."""
    import torch
    x = np.ones((4, 64), np.float32)
    x[0, 3], x[1, 5], x[2, 7] = np.inf, -np.inf, np.nan
    x[3, :] = np.nan
    v, s = dc.stored(np.zeros((4, 64)), fmt)
    cache, ks = dc.cache_of(v, fmt, scales=s)
    assert _append(dsv4, cache, ks, fmt, 64, 4, dc.dev(x), False, 64, 4, 64) == 0
    got = dc.cache_values(cache, fmt, ks)
    want = x.astype(np.float64)
    if fmt == 2:
        want[~np.isfinite(want)] = np.nan
        assert np.array_equal(ks.cpu().numpy(), np.float32([2.0 ** -8] * 3 + [1]))
    assert np.array_equal(got, want, equal_nan=True)
    cos, sin = dc.dev(np.ones((2, 8), np.float32)), dc.dev(np.zeros((2, 8), np.float32))
    rp = dc.rope_struct(dsv4, cos, sin, 16, 0, False)
    pos = dc.dev(np.array([0, 2, -1, 1], np.int32))
    ones = torch.ones(4, 64, device="cuda:0")
    assert _append(dsv4, cache, ks, fmt, 64, 4, ones, False, 64, 4, 64, rp=rp, pos=pos) == 0
    got = dc.cache_values(cache, fmt, ks)
    bad = np.zeros((4, 64), bool)
    bad[1:3, :16] = True
    assert np.array_equal(np.isnan(got), bad) and (got[~bad] == 1).all()


@pytest.mark.parametrize("n", [2, 6, 700])
def test_rows_named_twice_and_rows_outside(gpu, dsv4, n):
    """The last token that names a row has it, whole; rows outside the cache
    are not written."""
    rng = np.random.default_rng(n)
    d, rows = 128, 5
    x = rng.standard_normal((n, d)).astype(np.float32)
    at = rng.integers(-2, rows + 2, n).astype(np.int32)
    at[-1] = at[0]
    v, s = dc.stored(np.full((rows, d), 3.0), 2)
    cache, ks = dc.cache_of(v, 2, scales=s)
    assert _append(dsv4, cache, ks, 2, d, rows, dc.dev(x), False, d, n, d, dc.dev(at)) == 0
    want = v.copy()
    xv, _ = dc.stored(x, 2)
    for t in range(n):
        if 0 <= at[t] < rows:
            want[at[t]] = xv[t]
    assert np.array_equal(dc.cache_values(cache, 2, ks), want)


@pytest.mark.parametrize("n,d", [(4096, 8), (4097, 8), (9001, 7), (20000, 32), (70001, 4)])
@pytest.mark.parametrize("rows", [1, 300, 1 << 20])
def test_long_lists(gpu, dsv4, n, d, rows):
    """Lists that are looked up in a table: one row for all, a few rows, and
    rows far apart, named once or more."""
    rng = np.random.default_rng(n + rows)
    x = rng.integers(-8, 9, (n, d)).astype(np.float32)
    at = rng.integers(-2, rows + 2, n).astype(np.int32)
    if rows > n:
        at[:n // 2] = np.arange(n // 2) * (rows // n)
        at[n // 2:n // 2 + 100] = at[:100]
    at[-1] = at[0]
    cache, _ = dc.cache_of(np.full((rows, d), 99.0, np.float32), 0)
    assert _append(dsv4, cache, None, 0, d, rows, dc.dev(x), False, d, n, d, dc.dev(at)) == 0
    want = np.full((rows, d), 99.0, np.float32)
    fine = (at >= 0) & (at < rows)
    last = np.full(rows, -1)
    np.maximum.at(last, at[fine], np.nonzero(fine)[0])
    want[last >= 0] = x[last[last >= 0]]
    assert np.array_equal(dc.cache_values(cache, 0, None), want)


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_rows_moved_keep_their_values(gpu, dsv4, fmt):
    """What a verified path does with its rows: read back, written elsewhere.
    A row whose largest code rounded down to 224 takes half the scale and the
    same values."""
    import torch
    rng = np.random.default_rng(8)
    n, d = 200, 96
    x = rng.standard_normal((n, d)).astype(np.float32)
    x[0] *= 0.01
    x[0, 0] = 226.0                                       # 448 s with s = 1 -> code 224
    v, s = dc.stored(np.zeros((2 * n, d)), fmt)
    cache, ks = dc.cache_of(v, fmt, scales=s)
    assert _append(dsv4, cache, ks, fmt, d, 2 * n, dc.dev(x), False, d, n, d) == 0
    mid = torch.empty(n, d, device="cuda:0")
    assert _read(dsv4, mid, False, d, cache, ks, fmt, d, 2 * n, n, d) == 0
    assert _append(dsv4, cache, ks, fmt, d, 2 * n, mid, False, d, n, d, row0=n) == 0
    got = dc.cache_values(cache, fmt, ks)
    assert np.array_equal(got[n:], got[:n])


def test_a_store_of_the_library(gpu, dsv4):
    """The handle's device arrays, written here and used by the indexer."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((50, 128)).astype(np.float32)
    kv = dsv4.KV(64, 128, dsv4.KV_FP8)
    L = dsv4.lib()
    data, scales = L.dsv4_gpu_kv_data(kv.h), L.dsv4_gpu_kv_scales(kv.h)
    dx = dc.dev(x)
    assert L.dsv4_gpu_kv_append_d(data, scales, 2, 128, 64, dx.data_ptr(), 0, 128, 50, 128, None,
                                  0, None, None, dc.stream()) == 0
    import torch
    torch.cuda.synchronize()
    import oracle
    q = rng.standard_normal((16, 128)).astype(np.float32)
    w = rng.standard_normal(16).astype(np.float32)
    v, _ = dc.stored(x, 2)
    got = dsv4.indexer_score(q, w, kv, 50)
    assert common.bits_equal(got, oracle.indexer_score(q, v.astype(np.float32), w))
    kv.free()


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_offsets_past_32_bits(gpu, dsv4, fmt):
    """A cache whose last row starts past 2^32 elements."""
    import torch
    d, stride = 64, 1 << 20
    rows = 4100 if fmt else 4098
    cache = torch.zeros(rows * stride, device="cuda:0",
                        dtype=[torch.float32, torch.bfloat16, torch.uint8][fmt])
    ks = torch.ones(rows, device="cuda:0") if fmt == 2 else None
    x = np.random.default_rng(1).standard_normal((3, d)).astype(np.float32)
    at = dc.dev(np.array([rows - 1, 0, rows - 2], np.int32))
    assert _append(dsv4, cache, ks, fmt, stride, rows, dc.dev(x), False, d, 3, d, at) == 0
    out = torch.empty(3, d, device="cuda:0")
    assert _read(dsv4, out, False, d, cache, ks, fmt, stride, rows, 3, d, at) == 0
    assert np.array_equal(dc.host(out), dc.stored(x, fmt)[0].astype(np.float32))
    del cache
    torch.cuda.empty_cache()
