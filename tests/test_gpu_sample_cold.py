"""Sampling (dsv4_gpu_sample_d) at temperatures so low that f32 holds them, or what is
computed from them, with few bits, of logits about as small."""
import numpy as np
import pytest

from test_gpu_sample import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [700, 5003, 40000])
@pytest.mark.parametrize("scale", [1e-7, 1e-20, 1e-36, 1e-41])
def test_temperatures_under_the_least_normal(gpu, dsv4, vocab, scale):
    rng = np.random.default_rng(vocab)
    units = np.array([1, 2, 69, 70, 715, 725, 760, 100003, 3000001])
    t = np.concatenate([units * 2.0 ** -149, [1e-38, 3e-37, 1e-36, 1e-30]]).astype(np.float32)
    n = len(t)
    x = (rng.standard_normal((n, vocab)) * scale).astype(np.float32)
    x[:, ::3] -= np.float32(scale)
    u = rng.random(n).astype(np.float32)
    p = rng.uniform(0.3, 0.99, n)
    for kw in (dict(), dict(top_p=p), dict(top_k=np.full(n, 600)), dict(top_k=np.full(n, 7)),
               dict(min_p=np.full(n, 0.003)), dict(min_p=np.full(n, 0.2), top_p=p)):
        check(dsv4, x, temperature=t, u=u, **kw)
