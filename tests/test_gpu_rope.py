"""Rotary positions for many tokens (dsv4_gpu_rope_n_d) against the formula in
64 bits. f32: two products and a sum, each rounded. bf16: that, and one more
rounding of half a bf16 step."""
import ctypes

import numpy as np
import pytest

import common
import draft_common as dc

pytestmark = pytest.mark.gpu


def _call(dsv4, x, out, pos, heads, hd, xs, os_, bf, rp, inverse, nt):
    L = dsv4.lib()
    return L.dsv4_gpu_rope_n_d(out.data_ptr(), os_, x.data_ptr(), xs, int(bf), pos.data_ptr(),
                               nt, heads, hd, ctypes.byref(rp), int(inverse), dc.stream())


# (nt, heads, hd, dim, off): whole pieces, odd ones, one token and many, parts at either end,
# enough work for four heads per thread (with a number of heads that four does not divide)
SHAPES = [(1, 64, 512, 64, 448), (1, 1, 2, 2, 0), (3, 5, 72, 24, 40), (7, 3, 33, 10, 3),
          (64, 2, 576, 64, 512), (300, 130, 128, 128, 0), (2000, 7, 192, 64, 128)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("bf", [False, True])
def test_rope(gpu, dsv4, shape, halves, bf):
    import torch
    nt, heads, hd, dim, off = shape
    rng = np.random.default_rng(nt * 31 + hd)
    x = rng.standard_normal((nt, heads, hd)).astype(np.float32)
    if bf:
        x = dc.bf16(x)
    cos, sin = dc.tables(97, dim)
    pos = rng.integers(0, 97, nt).astype(np.int32)
    dcos, dsin, dpos = dc.dev(cos), dc.dev(sin), dc.dev(pos)
    rp = dc.rope_struct(dsv4, dcos, dsin, dim, off, halves)
    for inverse in (False, True):
        want, slack = dc.rotate(x, cos, sin, pos, off, dim, halves, inverse)
        if bf:
            slack = slack + dc.U16 * (np.abs(want) + slack)
            rot = np.zeros(hd, bool)
            rot[off:off + dim] = True
            slack[:, :, ~rot] = 0
        dx = dc.to_fmt(x, bf)
        out = torch.full_like(dx, 9.0)
        assert _call(dsv4, dx, out, dpos, heads, hd, heads * hd, heads * hd, bf, rp, inverse,
                     nt) == 0
        got = dc.host(out).astype(np.float64)
        assert (np.abs(got - want) <= slack).all()
        # in place: the same bits
        assert _call(dsv4, dx, dx, dpos, heads, hd, heads * hd, heads * hd, bf, rp, inverse,
                     nt) == 0
        assert common.bits_equal(dc.host(dx), dc.host(out))


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("pad", [1, 16])
def test_strides_addresses_and_far_positions(gpu, dsv4, bf, pad):
    """Padded tokens, a base that is not a whole piece, positions outside the
    table, and nothing written outside the heads."""
    import torch
    nt, heads, hd, dim, off = 5, 3, 64, 32, 16
    rng = np.random.default_rng(5)
    width, xs, os_ = heads * hd, heads * hd + pad, heads * hd + 2 * pad
    raw = rng.standard_normal(1 + nt * xs).astype(np.float32)
    raw = dc.bf16(raw) if bf else raw
    dx = dc.to_fmt(raw, bf)[1:] if pad == 1 else dc.to_fmt(raw[1:], bf)
    x = np.lib.stride_tricks.as_strided(raw[1:], (nt, width), (4 * xs, 4)).reshape(nt, heads, hd)
    out = torch.full((nt * os_ + 8,), 9.0, device="cuda:0", dtype=dx.dtype)
    cos, sin = dc.tables(10, dim)
    pos = np.array([0, 9, 10, -1, 2 ** 31 - 1], np.int32)
    dcos, dsin, dpos = dc.dev(cos), dc.dev(sin), dc.dev(pos)
    rp = dc.rope_struct(dsv4, dcos, dsin, dim, off, True)
    assert _call(dsv4, dx, out, dpos, heads, hd, xs, os_, bf, rp, False, nt) == 0
    want, slack = dc.rotate(x, cos, sin, pos, off, dim, True)
    if bf:
        slack = slack + dc.U16 * (np.abs(want) + slack)
    flat = dc.host(out)
    rows = flat[:nt * os_].reshape(nt, os_)
    got = rows[:, :width].reshape(nt, heads, hd).astype(np.float64)
    assert np.isnan(got[2:, :, off:off + dim]).all()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(got - want)[fine] <= slack[fine]).all()
    assert (rows[:, width:] == 9).all() and (flat[nt * os_:] == 9).all()


def test_matches_the_attention_blocks_rotation(gpu, dsv4):
    """The neighbour layout has the bits of the separately rounded products and
    sum that the attention block rotates with."""
    import torch
    rng = np.random.default_rng(3)
    x = rng.standard_normal((9, 4, 64)).astype(np.float32)
    cos, sin = dc.tables(50, 64)
    pos = rng.integers(0, 50, 9).astype(np.int32)
    dcos, dsin, dpos, dx = dc.dev(cos), dc.dev(sin), dc.dev(pos), dc.dev(x)
    out = torch.empty_like(dx)
    rp = dc.rope_struct(dsv4, dcos, dsin, 64, 0, False)
    assert _call(dsv4, dx, out, dpos, 4, 64, 256, 256, False, rp, False, 9) == 0
    c, s = cos[pos][:, None, :], sin[pos][:, None, :]
    want = np.empty_like(x)
    want[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    want[..., 1::2] = x[..., 0::2] * s + x[..., 1::2] * c
    assert common.bits_equal(dc.host(out), want)
