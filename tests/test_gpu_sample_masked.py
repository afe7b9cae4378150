"""Sampling (dsv4_gpu_sample_d) of rows most of whose logits are -infinity or NaN, as
rules that allow a few ranges of ids leave them: fewer places of a row with a token
than top-k asks for, as many, one less and one more."""
import numpy as np
import pytest

import common
import draft_common as dc
import reqs_common as rc
import test_gpu_reqs_step as steps
from test_gpu_sample import INF, NAN, check

pytestmark = pytest.mark.gpu

CHUNK = 64                                       # neighbours that are looked at together


def ids(rng, vocab, kind, k):
    """The allowed ids of a row."""
    nc = -(-vocab // CHUNK)
    spread = lambda n: np.sort(rng.permutation(nc - 1)[:n])[:, None] * CHUNK
    if kind == "a chunk":
        return CHUNK * 3 + np.arange(CHUNK)
    if kind == "part of one":
        return 15 + np.arange(45)
    if kind == "three":
        return CHUNK * 7 - 40 + np.arange(200)
    if kind == "run":
        return 1000 + np.arange(600)
    if kind == "last":
        return np.arange((nc - 1) * CHUNK, vocab)
    if kind == "one token":
        return np.array([vocab // 2])
    if kind == "many of few":                    # more than are put in order
        return (spread(20) + np.arange(CHUNK)).ravel()
    n = min(nc - 1, max(1, k + {"k - 1": -1, "k": 0, "k + 1": 1}[kind]))
    return (spread(n) + rng.permutation(CHUNK)[:5]).ravel()


KINDS = ["a chunk", "part of one", "three", "run", "last", "one token", "many of few", "k - 1", "k",
         "k + 1"]
TOP = [2, 20, 50, 512]


@pytest.mark.parametrize("vocab", [4096, 8190, 32003, 129280])
@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("out", [-INF, NAN])
def test_few_places_with_tokens(gpu, dsv4, vocab, bf, out):
    rng = np.random.default_rng(vocab + bf)
    k = np.repeat(TOP, len(KINDS))
    n = len(k)
    x = np.full((n, vocab), out, np.float32)
    for r in range(n):
        at = ids(rng, vocab, KINDS[r % len(KINDS)], k[r])
        x[r, at] = rng.standard_normal(len(at)).astype(np.float32) * np.float32(2)
    t, p = rng.uniform(0.3, 2.0, n), rng.uniform(0.2, 0.99, n)
    m = 10.0 ** rng.uniform(-4, -0.5, n)
    for kw in (dict(), dict(temperature=t), dict(top_p=p), dict(min_p=m),
               dict(temperature=t, top_p=p, min_p=m)):
        check(dsv4, x, bf, top_k=k, u=rng.random(n).astype(np.float32), **kw)
    # and the rules without a top-k
    for kw in (dict(), dict(top_p=p), dict(min_p=m), dict(temperature=t, top_p=p, min_p=m)):
        check(dsv4, x, bf, u=rng.random(n).astype(np.float32), **kw)


@pytest.mark.parametrize("bf", [False, True])
def test_infinities_among_few(gpu, dsv4, bf):
    """One chunk of tokens, some of them +infinity or the lowest finite value."""
    rng = np.random.default_rng(3 + bf)
    n, vocab = 12, 129280
    low = np.float32(-3.3895314e38) if bf else np.float32(-3.4028235e38)
    x = np.full((n, vocab), -INF, np.float32)
    x[:, 640:704] = rng.standard_normal((n, 64)).astype(np.float32)
    x[::3, 650] = low
    x[1::3, [641, 690]] = INF
    check(dsv4, x, bf, top_k=np.tile([1, 2, 30, 64, 65, 512], 2), u=rng.random(n).astype(np.float32))
    check(dsv4, x, bf, top_k=np.full(n, 20), top_p=np.full(n, 0.6), u=rng.random(n).astype(np.float32))


@pytest.mark.parametrize("case", steps.CASES[:3])
def test_steps_with_runs_of_allowed_ids(gpu, dsv4, case):
    """Whole steps of a batch whose rules on the logits allow some tens of neighbouring
    ids, each request with a top-k."""
    import torch
    s = steps.Serve(dsv4, *case[:2], 41, *case[2:])
    allow = np.zeros((s.n, s.allow.shape[1] * 32), np.uint8)
    for b in range(s.n):
        at = int(s.rng.integers(0, steps.VOCAB - 80))
        allow[b, at:at + int(s.rng.integers(20, 80))] = 1
    s.allow = np.packbits(allow, axis=1, bitorder="little").view(np.uint32)
    s.rule["top_k"] = s.rng.integers(2, 17, s.n).astype(np.int32)
    s.dallow.copy_(dc.dev(s.allow))
    s.drule["top_k"].copy_(dc.dev(s.rule["top_k"]))
    for k in range(4):
        s.begin()
        new = s.next(k)
        s.inputs(new)
        s.queue(dc.stream())
        torch.cuda.synchronize()
        s.check(new)
