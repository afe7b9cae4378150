"""min_p of dsv4_gpu_sample_d at its ends: so low that it reaches tokens whose weight is
no part of any sum, and not a number."""
import numpy as np
import pytest

import reqs_common as rc
from test_gpu_sample import NAN, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [5, 700, 40000])
@pytest.mark.parametrize("bf", [False, True])
def test_floors_under_the_sums(gpu, dsv4, vocab, bf):
    """Tokens down to 2^-160 of the first's probability, under floors down to f32's least:
    those at or over the floor are kept."""
    rng = np.random.default_rng(vocab + bf)
    floor = np.array([1e-45, 1e-40, 1e-38, 1e-30, 1e-25, 1e-20, 2e-20, 1e-15, 1e-10], np.float32)
    n = len(floor)
    x = (-rng.random((n, vocab)) * 110).astype(np.float32)
    x[:, rng.integers(0, vocab)] = 1.0
    u = rng.random(n).astype(np.float32)
    few = np.full(n, 10)
    for kw in (dict(), dict(top_k=few), dict(top_k=np.full(n, 600)), dict(top_p=np.full(n, 0.999)),
               dict(temperature=np.linspace(0.7, 1.4, n))):
        check(dsv4, x, bf, u=u, min_p=floor, **kw)


@pytest.mark.parametrize("vocab", [700, 40000])
def test_a_floor_that_is_not_a_number(gpu, dsv4, vocab):
    """No such rule, as with top_p."""
    rng = np.random.default_rng(vocab)
    n = 6
    x = rng.standard_normal((n, vocab)).astype(np.float32) * np.float32(2)
    u = rng.random(n).astype(np.float32)
    for kw in (dict(), dict(top_k=np.full(n, 9)), dict(top_k=np.full(n, 600)),
               dict(top_p=np.full(n, 0.7)), dict(temperature=np.full(n, 0.8))):
        got = check(dsv4, x, u=u, min_p=np.full(n, NAN), **kw)
        want = rc.run_sample(dsv4, x, u=u, **kw)
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
