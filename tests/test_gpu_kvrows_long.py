"""Cache rows written by calls of so many that they take several launches."""
import numpy as np
import pytest

import draft_common as dc
import test_gpu_kvrows as tk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [0, 2])
@pytest.mark.parametrize("n", [(1 << 17) + 1, 3 * (1 << 17) - 5, 600000])
def test_a_lists_later_launches(gpu, dsv4, fmt, n):
    """Rows named once, twice within a launch and by tokens of different ones:
    the last token has the row, whole and with its scale."""
    rng = np.random.default_rng(n + fmt)
    d, rows = 5, 1 << 18
    x = rng.integers(-8, 9, (n, d)).astype(np.float32) * np.exp2(
        rng.integers(-3, 4, (n, 1))).astype(np.float32)
    at = rng.integers(-2, rows + 2, n).astype(np.int32)
    at[[0, 1 << 17, n - 1]] = 77
    at[n - 2], at[5] = 78, 78
    v, s = dc.stored(np.full((rows, d), 96.0), fmt)
    cache, ks = dc.cache_of(v, fmt, scales=s)
    assert tk._append(dsv4, cache, ks, fmt, d, rows, dc.dev(x), False, d, n, d, dc.dev(at)) == 0
    xv, xs = dc.stored(x, fmt)
    fine = (at >= 0) & (at < rows)
    last = np.full(rows, -1)
    np.maximum.at(last, at[fine], np.nonzero(fine)[0])
    want = v.copy()
    want[last >= 0] = xv[last[last >= 0]]
    assert np.array_equal(dc.cache_values(cache, fmt, ks), want)
    if fmt == 2:
        s[last >= 0] = xs[last[last >= 0]]
        assert np.array_equal(ks.cpu().numpy(), s.astype(np.float32))


def test_more_rows_than_a_launch_has_threads_for(gpu, dsv4):
    """2^26 and a few rows of one element, behind row0."""
    import torch
    n, row0 = (1 << 26) + 5, 3
    x = torch.arange(n, device="cuda:0", dtype=torch.int32).remainder_(251).to(torch.bfloat16)
    cache = torch.full((n + 7, 1), 300.0, device="cuda:0", dtype=torch.bfloat16)
    assert tk._append(dsv4, cache, None, 1, 1, n + 7, x, True, 1, n, 1, row0=row0) == 0
    assert torch.equal(cache[row0:row0 + n, 0], x)
    assert bool((cache[:row0] == 300).all()) and bool((cache[row0 + n:] == 300).all())
    del cache, x
    torch.cuda.empty_cache()
