"""Attention of drafted tokens at the ends of what it takes: the longest
windows, the largest values, few rows that carry all the weight."""
import numpy as np
import pytest

import common
import draft_common as dc
import test_gpu_tree as tt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, True)])
def test_the_longest_window_is_no_window(gpu, dsv4, fmt, bf):
    """A window of 2^31 - 1 splits the cache as none does and has its bits."""
    nt, h, dqk, dv, ctx = 3, 16, 128, 96, 9000
    _, dq, _, _, cache, ks, rows, _ = tt.problem(3, nt, h, dqk, ctx, fmt, bf)
    out = []
    for window in (0, 2 ** 31 - 1, ctx + nt):
        rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx, window=window, scale=0.1)
        assert rc == 0
        out.append(dc.host(o))
    assert common.bits_equal(out[1], out[0]) and common.bits_equal(out[2], out[0])


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, False), (0, True), (1, True),
                                    (2, True)])
@pytest.mark.parametrize("ctx", [40, 2000, 30000])
def test_the_largest_values(gpu, dsv4, fmt, bf, ctx):
    """Rows of one sign whose largest element times their number is 1e36, with a
    maximum that creeps up (head 0 sees its scores in ascending order) and, for the
    longer contexts, in several splits: the sums stay in range. The bounds are
    those of the other tests, relative."""
    nt, h, d = 2, 4, 64
    rng = np.random.default_rng(ctx + fmt)
    n = ctx + nt
    top = 1e36 / n
    q = (rng.standard_normal((nt, h, d)) * 1e-30).astype(np.float32)
    q = dc.bf16(q) if bf else q
    x = rng.uniform(0.5, 0.99, (n, d))
    x = x[np.argsort(x @ q[0, 0].astype(np.float64))] * top
    v, s = dc.stored(x.astype(np.float32), fmt)
    assert v.max() * n <= 1e36
    cache, ks = dc.cache_of(v, fmt, scales=s)
    scale = np.float32(8.0 / np.abs(q.astype(np.float64) @ v.T).max())
    # twice over: spread scores and equal ones
    for sc in (scale, np.float32(scale * 1e-6)):
        rc, o = dc.tree(dsv4, dc.to_fmt(q, bf), bf, cache, ks, fmt, n, d, d, ctx, scale=sc)
        assert rc == 0
        want, size = dc.attention(q, v, dc.visible(None, nt, ctx, 0), None, sc, d)
        tt.check(dc.host(o) / top, want / top, size / top, bf)


@pytest.mark.parametrize("fmt,bf", [(0, True), (1, True), (2, True), (2, False)])
def test_the_mean_of_equal_rows_is_the_row(gpu, dsv4, fmt, bf):
    """Rows that differ in their scores alone: whatever the weights and their
    rounding, o is the row's values, which bf16 holds, as the weights are divided by
    their own sum. The first tile's weights are 1; the later ones' would be 2^7 (1 +
    0.0038), just under the middle of two bf16 numbers, over a maximum that has not
    moved. f32 sums of 200 rows are off by 200 2^-24 at most, far under half a step
    of bf16; with f32 q that is the bound."""
    nt, h, dqk, dv, ctx = 64, 520, 64, 56, 136
    n = ctx + nt
    rng = np.random.default_rng(fmt)
    rows = np.zeros((n, dqk))
    rows[:, :dv] = 2.0 ** rng.integers(-1, 2, dv) * (1 + rng.integers(0, 8, dv) / 8)
    rows[32:, dv], rows[32:, dv + 1] = 7.0, 0.75
    q = np.zeros((nt, h, dqk), np.float32)
    q[:, :, dv], q[:, :, dv + 1] = 1.0, dc.bf16(0.00555 / 0.75)
    assert 0.0050 < 0.75 * q[0, 0, dv + 1] < np.log2(1 + 2.0 ** -8) - 1e-5
    scales = np.exp2(rng.integers(-2, 3, n)) if fmt == 2 else None
    cache, ks = dc.cache_of(rows, fmt, scales=scales)
    words = dc.dev(np.full(nt, 2 ** 64 - 1, np.uint64))
    rc, o = dc.tree(dsv4, dc.to_fmt(q, bf), bf, cache, ks, fmt, n, dqk, dv, ctx, words,
                    scale=np.float32(np.log(2.0)))
    assert rc == 0
    want = np.broadcast_to(rows[0, :dv], (nt, h, dv))
    if bf:
        assert np.array_equal(dc.host(o), want)
    else:
        assert np.abs(dc.host(o) / want - 1).max() <= n * dc.U32


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, True), (2, False)])
@pytest.mark.parametrize("nt", [2, 7, 63, 64])
def test_words_of_any_kind_under_a_window(gpu, dsv4, fmt, bf, nt):
    """Tokens that see later ones, not themselves or bits past the last token: a
    token further on than the one that sees it is not back behind its window."""
    h, d, ctx = 3, 40, 50
    rng, dq, q, v, cache, ks, rows, _ = tt.problem(nt, nt, h, d, ctx, fmt, bf)
    w = [int(x) for x in rng.integers(0, 2 ** 64, nt, dtype=np.uint64)]
    for window in (0, 1, 3, 20, 64):
        rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, d, d, ctx,
                        dc.dev(np.array(w, np.uint64)), window, scale=0.2)
        assert rc == 0
        see = dc.visible(w, nt, ctx, window)
        want, size = dc.attention(q, v, see, None, 0.2, d)
        tt.check(dc.host(o), want, size, bf)
        assert (dc.host(o)[~see.any(1)] == 0).all()
