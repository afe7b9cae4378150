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
