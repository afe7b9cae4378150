"""Sampling (dsv4_gpu_sample_d) against the same limits in 64 bits: picks and
counts have to be equal, and probabilities within f32's rounding."""
import numpy as np
import pytest

import common
import draft_common as dc
import reqs_common as rc

pytestmark = pytest.mark.gpu

INF, NAN = np.inf, np.nan


def logits(rng, n, vocab, kind="likely"):
    x = rng.standard_normal((n, vocab)).astype(np.float32) * np.float32(2)
    if kind == "likely":
        at = rng.integers(0, vocab, (n, min(48, vocab)))
        for r in range(n):
            x[r, at[r]] += (4 + 4 * np.abs(rng.standard_normal(at.shape[1]))).astype(np.float32)
    return x


def check(dsv4, x, bf=False, **kw):
    """One call against the oracle, row by row."""
    n = len(x)
    x = dc.bf16(x) if bf else np.asarray(x, np.float32)
    got = rc.run_sample(dsv4, x, bf, **kw)
    rule = [np.full(n, d) if kw.get(k) is None else np.asarray(kw[k], np.float32)
            for k, d in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0),
                         ("u", 0.0))]
    for r in range(n):
        want = rc.sample(x[r], *[v[r] for v in rule[:1]], int(rule[1][r]),
                         *[v[r] for v in rule[2:]])
        assert got[2][r] == want[2], (r, got[2][r], want)
        assert got[0][r] == want[0], (r, got[0][r], want)
        # one rounding to f32, and weights to 2^-40 of the largest in the sum
        assert abs(got[1][r] - want[1]) <= want[1] * (2.0 ** -24 + 2.0 ** -39), (r, got[1][r], want)
    return got


def rules(rng, n):
    """A mix of rules, some of them off."""
    pick = lambda v, off, p: np.where(rng.random(n) < p, v, off)
    return dict(temperature=pick(rng.uniform(0.3, 2.0, n), 1.0, 0.8) * (rng.random(n) > 0.08),
                top_k=pick(np.exp(rng.uniform(0, 7, n)).astype(int), 0, 0.5),
                top_p=pick(rng.uniform(0.05, 0.999, n), 1.0, 0.6),
                min_p=pick(10.0 ** rng.uniform(-4, 0, n), 0.0, 0.4),
                u=rng.random(n).astype(np.float32))


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 127, 1000, 4095, 8191, 8192, 8193, 32003,
                                   129280, 200001])
@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("kind", ["likely", "flat"])
def test_rules(gpu, dsv4, vocab, bf, kind):
    rng = np.random.default_rng(vocab * 4 + 2 * bf + (kind == "flat"))
    n = 24 if vocab < 100000 else 12
    check(dsv4, logits(rng, n, vocab, kind), bf, **rules(rng, n))


@pytest.mark.parametrize("n", [1, 2, 17, 64, 130, 300])
def test_rows(gpu, dsv4, n):
    rng = np.random.default_rng(n)
    check(dsv4, logits(rng, n, 5003), **rules(rng, n))


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("stride,shift", [(1003, 0), (1003, 1), (1010, 3), (1000, 5)])
def test_strides_and_addresses(gpu, dsv4, bf, stride, shift):
    rng = np.random.default_rng(stride + shift)
    check(dsv4, logits(rng, 9, 1000), bf, stride=stride, shift=shift, **rules(rng, 9))


@pytest.mark.parametrize("one", ["temperature", "top_k", "top_p", "min_p"])
def test_rules_left_out(gpu, dsv4, one):
    """Each rule alone, the others' arrays missing; and outputs left out."""
    rng = np.random.default_rng(3)
    x, r = logits(rng, 40, 20000), rules(rng, 40)
    a = check(dsv4, x, u=r["u"], **{one: r[one]})
    b = rc.run_sample(dsv4, x, u=r["u"], prob=False, kept=False, **{one: r[one]})
    assert np.array_equal(a[0], b[0]) and (b[1] == -7).all() and (b[2] == -7).all()


@pytest.mark.parametrize("vocab", [1, 5, 64, 1500, 8192, 30000])
def test_equal_logits(gpu, dsv4, vocab):
    """All equal: weights are equal whole numbers, so every border lies exactly
    between two tokens, and the lowest ids come first."""
    us = np.array([0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24], np.float32)
    for value in (0.0, -0.0, 3.25, -1e30, 1e30, INF):
        x = np.full((len(us), vocab), value, np.float32)
        if value == 0.0:
            x[:, ::2] = -0.0
        n = len(us)
        check(dsv4, x, u=us)
        check(dsv4, x, u=us, temperature=np.full(n, 0.7))
        check(dsv4, x, u=us, top_k=np.array([1, 2, 3, vocab, vocab + 1]))
        check(dsv4, x, u=us, top_p=np.array([0, 0.25, 0.5, 0.75, 0.9999]))
        check(dsv4, x, u=us, min_p=np.array([1, 0.5, 1e-6, 2, 0]))


@pytest.mark.parametrize("vocab", [700, 40000, 129280, 262145])
@pytest.mark.parametrize("few", [1, 2, 1023, 1024, 1025, 2048, 2049, 30000])
def test_min_p_alone(gpu, dsv4, vocab, few):
    """Of a row, `few` tokens at or above min_p and the others a step below it, in a
    heap, spread and one in each chunk; top-k long, off and at the number."""
    few = min(few, vocab)
    rng = np.random.default_rng(vocab + few)
    low = np.float32(-4.5)                       # e^-4.5 = 0.0111, under 0.012 and over 0.011
    x = np.full((6, vocab), low, np.float32)
    for r in range(6):
        at = (rng.permutation(vocab)[:few], np.arange(vocab - few, vocab),
              (np.arange(few) * 64 + np.arange(few) * 64 // vocab) % vocab)[r % 3]
        x[r, at] = rng.uniform(-4.42, -1, len(at)).astype(np.float32)
        x[r, at[0]] = 0
    x[5, rng.integers(0, vocab)] = INF
    k = np.array([0, vocab, few, max(1, few - 1), 600, 0])
    for min_p in (0.012, 0.011, 1.0):
        check(dsv4, x, min_p=np.full(6, min_p), top_k=k, u=rng.random(6).astype(np.float32))
        check(dsv4, x * 1e30, temperature=np.full(6, 1e30), min_p=np.full(6, min_p), top_k=k,
              u=rng.random(6).astype(np.float32))
    check(dsv4, x, True, min_p=np.full(6, 0.0078125), top_p=np.where(k == 600, 0.5, 1.0),
          u=rng.random(6).astype(np.float32))


@pytest.mark.parametrize("vocab", [60000, 129280])
@pytest.mark.parametrize("bf", [False, True])
def test_flat_rows(gpu, dsv4, vocab, bf):
    """Rows whose limits' and pick's tokens stand among hundreds to thousands that weigh
    about the same, which are too many together or alone."""
    rng = np.random.default_rng(vocab + bf)
    x = rng.standard_normal((32, vocab)).astype(np.float32) * np.float32(2)
    t = np.exp(rng.uniform(np.log(0.5), np.log(6), 32))
    k = np.where(np.arange(32) % 4 == 3, rng.integers(2000, vocab, 32), 0)
    p = np.where(np.arange(32) % 4 == 2, 1.0, rng.uniform(0.5, 0.99, 32))
    m = np.where(np.arange(32) % 8 == 1, 10.0 ** rng.uniform(-4, -1, 32), 0.0)
    check(dsv4, x, bf, temperature=t, top_k=k, top_p=p, min_p=m, u=rng.random(32).astype(np.float32))


@pytest.mark.parametrize("vocab", [20000, 129280, 262145, 300000])
def test_likely_tokens_that_stand_together(gpu, dsv4, vocab):
    """Sorted logits, and a block of equal ones: many tokens of few chunks as large as
    the k-th largest chunk."""
    rng = np.random.default_rng(vocab)
    n = 9
    x = -np.sort(-logits(rng, n, vocab, "flat"), axis=1)
    x[3:6] = x[3:6, ::-1]
    x[6:, 1000:4000] = 20.0
    k = np.array([1, 40, 512, 2, 200, 513, 50, 3, 400])
    r = rules(rng, n)
    for keys in (("u",), ("u", "top_p"), ("u", "min_p", "temperature"), tuple(r)):
        kw = {name: r[name] for name in keys}
        kw["top_k"] = k
        check(dsv4, x, **kw)
    check(dsv4, x, True, u=r["u"], top_k=k)


def test_far_ahead(gpu, dsv4):
    """One token far ahead of the rest, the k-th among the tokens of no weight."""
    rng = np.random.default_rng(31)
    n, vocab = 8, 129280
    x = logits(rng, n, vocab, "flat")
    x[:, 77] = 60
    check(dsv4, x, u=rng.random(n), temperature=np.full(n, 0.5), top_k=np.full(n, 50),
          top_p=np.array([0.5, 0.9, 1, 1, 0.99, 0.999, 1, 0.3]))
    check(dsv4, x, u=rng.random(n), top_k=np.full(n, 5000), top_p=np.full(n, 0.9))


def test_two_values(gpu, dsv4):
    """Long runs of equal logits on both sides of a border."""
    rng = np.random.default_rng(8)
    n, vocab = 30, 40000
    x = np.where(rng.random((n, vocab)) < 0.3, np.float32(1.0), np.float32(0.5))
    check(dsv4, x, **rules(rng, n))
    check(dsv4, x, True, **rules(rng, n))


def test_logits_that_are_not_numbers(gpu, dsv4):
    """NaN and -infinity are out; +infinity takes all; rows of nothing give -1."""
    rng = np.random.default_rng(4)
    n, vocab = 16, 9001
    for bf in (False, True):
        x = logits(rng, n, vocab)
        x[rng.random(x.shape) < 0.3] = NAN
        x[rng.random(x.shape) < 0.3] = -INF
        x[0] = NAN
        x[1] = -INF
        x[2, :8500] = -INF                       # slices of nothing
        x[3, 600:] = NAN
        x[4, [17, 8999, 300]] = INF
        x[5, 8192:] = INF
        x[6] = -INF
        x[6, 9000] = -3.0e38
        for t in (None, np.full(n, 0.0), np.full(n, 0.8)):
            check(dsv4, x, bf, u=rng.random(n), temperature=t)
            check(dsv4, x, bf, u=rng.random(n), temperature=t, top_k=rng.integers(1, 400, n),
                  top_p=rng.uniform(0.1, 0.99, n))


def test_values_of_rules_at_their_ends(gpu, dsv4):
    rng = np.random.default_rng(6)
    ts = np.array([1e-45, 1e-30, 1e-3, 0.01, 5.0, 20.0, 1e4, 1e38, INF, -1.0, -INF, NAN], np.float32)
    x = logits(rng, len(ts), 30011)
    us = rng.random(len(ts))
    check(dsv4, x, temperature=ts, u=us)
    check(dsv4, x, temperature=ts, u=us, top_p=np.full(len(ts), 0.9))
    check(dsv4, x, temperature=ts, u=us, top_k=np.full(len(ts), 30000))
    check(dsv4, x * np.float32(1e37), temperature=ts, u=us)
    us = np.array([0, 1e-45, 1e-38, 1e-10, 1 - 2.0 ** -24, 1, 2, INF, -1, -INF, NAN, 0.5], np.float32)
    x = logits(rng, len(us), 700)
    check(dsv4, x, u=us, top_k=np.full(len(us), 9))
    n = 10
    x = logits(rng, n, 3001)
    us = rng.random(n)
    check(dsv4, x, u=us, top_k=np.array([-1, 0, 1, 2, 3000, 3001, 3002, 2 ** 31 - 1, -2 ** 31, 50]))
    check(dsv4, x, u=us, top_p=np.array([-1, 0, 1e-45, 1e-9, 1 - 2.0 ** -24, 1, 2, INF, NAN, 0.5]))
    check(dsv4, x, u=us, min_p=np.array([-1, 0, 1e-45, 1e-30, 1 - 2.0 ** -24, 1, 2, INF, 0.3, 0.5]))


def test_picks_follow_the_probabilities(gpu, dsv4):
    """One row under many numbers: each token's share of evenly spread u is its
    probability to a step of the spread."""
    rng = np.random.default_rng(7)
    n = 4096
    row = logits(rng, 1, 500)[0]
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    pick = rc.run_sample(dsv4, np.tile(row, (n, 1)), u=u, temperature=np.full(n, 1.5))[0]
    p = np.exp(row.astype(np.float64) / 1.5)
    p /= p.sum()
    assert np.abs(np.bincount(pick, minlength=500) / n - p).max() <= 1.01 / n


def test_the_same_bits_on_a_busy_card_and_in_a_graph(gpu, dsv4):
    """Captured on a side stream and replayed with other calls between, its rules
    changed on the device: every replay as the eager call."""
    import ctypes

    import torch
    rng = np.random.default_rng(12)
    n, vocab = 12, 129280
    L = dsv4.lib()
    r = rules(rng, n)
    x = dc.dev(logits(rng, n, vocab))
    d = {k: dc.dev(np.asarray(v, np.int32 if k == "top_k" else np.float32)) for k, v in r.items()}
    s = dsv4.Sampling(**{k: v.data_ptr() for k, v in d.items()})
    space = torch.full((L.dsv4_gpu_sample_scratch_bytes(n, vocab),), 255, device="cuda:0",
                       dtype=torch.uint8)
    out = [torch.zeros(n, device="cuda:0", dtype=t) for t in
           (torch.int32, torch.float32, torch.int32)]

    def queue(st):
        assert L.dsv4_gpu_sample_d(*[o.data_ptr() for o in out], x.data_ptr(), 0, n, vocab, vocab,
                                   ctypes.byref(s), space.data_ptr(), space.numel(), st) == 0

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        queue(torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        r = rules(rng, n)
        for name, v in r.items():
            d[name].copy_(dc.dev(np.asarray(v, np.int32 if name == "top_k" else np.float32)))
        for o in out:
            o.zero_()
        torch.cuda.synchronize()
        g.replay()
        other = logits(rng, 3, 50000)
        rc.run_sample(dsv4, other, u=rng.random(3))
        torch.cuda.synchronize()
        got = [o.cpu().numpy() for o in out]
        want = rc.run_sample(dsv4, dc.host(x), **r)
        for a, b in zip(got, want):
            assert common.bits_equal(a, b)
