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
