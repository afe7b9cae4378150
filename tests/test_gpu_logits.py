"""A request's rules on its logits (dsv4_gpu_logits_adjust_d) against the
same steps in f32, bit for bit, and the head's scan over the allowed tokens."""
import ctypes

import numpy as np
import pytest

import common
import draft_common as dc

pytestmark = pytest.mark.gpu


def run(dsv4, x, ids=(), drafts=None, words=None, rep=1.0, freq=0.0, pres=0.0, bias=None,
        allow=None, stride=None, shift=0, in_place=False, picks=True, out=True):
    import torch
    L = dsv4.lib()
    nt, vocab = x.shape
    stride = stride or vocab
    buf = torch.full((shift + nt * stride + 8,), 5.0, device="cuda:0")
    buf[shift:shift + nt * stride].view(nt, stride)[:, :vocab] = dc.dev(x)
    dst = buf if in_place else torch.full_like(buf, 9.0)
    pick = torch.full((nt + 1,), -7, device="cuda:0", dtype=torch.int32)
    keep = [None if a is None else dc.dev(np.asarray(a, t)) for a, t in (
        (ids if len(ids) else None, np.int32), (drafts, np.int32),
        (None if words is None else np.array(words, np.uint64), None), (bias, np.float32))]
    dallow, astride = None, 0
    if allow is not None:
        w = -(-vocab // 32)
        bits = np.zeros((allow.shape[0], w * 32), np.uint8)
        bits[:, :vocab] = allow
        bits[:, vocab:] = 1                            # what follows the vocabulary is not read
        packed = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
        astride = w + 1 if allow.shape[0] > 1 else 0
        if astride:
            packed = np.concatenate([packed, np.zeros((allow.shape[0], 1), np.uint32)], 1)
        dallow = dc.dev(packed)
    r = dsv4.LogitRules(hist=dc.ptr(keep[0]), n_hist=len(ids), draft=dc.ptr(keep[1]),
                        mask=dc.ptr(keep[2]), repetition=rep, frequency=freq, presence=pres,
                        bias=dc.ptr(keep[3]), allow=dc.ptr(dallow), allow_stride=astride)
    n = L.dsv4_gpu_logits_scratch_bytes(nt, vocab)
    space = torch.full((n + 16,), 255, device="cuda:0", dtype=torch.uint8)
    at = 4 * shift
    rc = L.dsv4_gpu_logits_adjust_d(dst.data_ptr() + at if out else None,
                                    pick.data_ptr() if picks else None, buf.data_ptr() + at, nt,
                                    vocab, stride, ctypes.byref(r), space.data_ptr(), n,
                                    dc.stream())
    assert rc == 0
    assert (space[n:] == 255).all()
    flat = dc.host(dst)
    rows = flat[shift:shift + nt * stride].reshape(nt, stride)
    edge = 5.0 if in_place else 9.0
    assert (rows[:, vocab:] == edge).all() and (flat[:shift] == edge).all()
    p = pick.cpu().numpy()
    assert p[nt] == -7
    return rows[:, :vocab], p[:nt]


def check(got, want):
    assert np.array_equal(np.isnan(got[0]), np.isnan(want[0]))
    fine = ~np.isnan(want[0])
    assert common.bits_equal(got[0][fine], want[0][fine])
    assert np.array_equal(got[1], want[1])


@pytest.mark.parametrize("nt,vocab", [(1, 1), (1, 129280), (3, 1000), (4, 4097), (64, 8195),
                                      (17, 129283), (64, 32000)])
@pytest.mark.parametrize("hist", [0, 1, 1003, 20000])
def test_rules(gpu, dsv4, nt, vocab, hist):
    rng = np.random.default_rng(nt * vocab + hist)
    x = (rng.standard_normal((nt, vocab)) * 3).astype(np.float32)
    # some ids outside the vocabulary, some many times
    ids = rng.integers(-3, max(2, vocab // 3), hist).astype(np.int32)
    if hist > 10:
        ids[:5] = [vocab, 2 ** 31 - 1, -2 ** 31, vocab - 1, vocab - 1]
    drafts = rng.integers(-1, vocab + 1, nt).astype(np.int32)
    drafts[-1] = drafts[0]
    words = dc.words(rng, nt)
    bias = rng.standard_normal(vocab).astype(np.float32)
    allow = rng.random((nt, vocab)) < 0.5
    check(run(dsv4, x, ids, drafts, words, 1.3, 0.25, 0.5, bias, allow),
          dc.logit_rules(x, ids, drafts, words, 1.3, 0.25, 0.5, bias, allow))
    # parts of it: a chain of drafts, one shared set, each rule by itself
    check(run(dsv4, x, ids, drafts, None, 0.8, 0, 0, None, allow[:1], in_place=True),
          dc.logit_rules(x, ids, drafts, None, 0.8, 0, 0, None, allow[:1]))
    check(run(dsv4, x, ids, None, None, 1, 0.1, -0.2), dc.logit_rules(
        x, ids, None, None, 1, 0.1, -0.2, None, None))
    check(run(dsv4, x, (), None, None, 1, 0, 0, bias), dc.logit_rules(
        x, (), None, None, 1, 0, 0, bias, None))


@pytest.mark.parametrize("stride,shift", [(1003, 0), (1004, 0), (1008, 3), (1000, 4)])
def test_strides_and_addresses(gpu, dsv4, stride, shift):
    rng = np.random.default_rng(stride)
    x = rng.standard_normal((5, 1000)).astype(np.float32)
    ids = rng.integers(0, 1000, 300)
    allow = rng.random((5, 1000)) < 0.3
    want = dc.logit_rules(x, ids, None, None, 1.2, 0.1, 0.1, None, allow)
    for in_place in (False, True):
        check(run(dsv4, x, ids, rep=1.2, freq=0.1, pres=0.1, allow=allow, stride=stride,
                  shift=shift, in_place=in_place), want)


@pytest.mark.parametrize("nt", [3, 9])
def test_picks(gpu, dsv4, nt):
    """Nothing allowed; NaN first, in the middle and everywhere; ties; both
    zeros; infinities; all minus infinity. Picks alone, and rows alone."""
    rng = np.random.default_rng(0)
    vocab = 5000
    for k in range(10):
        x = rng.integers(-3, 3, (nt, vocab)).astype(np.float32)
        allow = rng.random((nt, vocab)) < 0.4
        if k == 0:
            allow[:] = False
        if k == 1:
            allow[0] = False
            allow[0, vocab - 1] = True
        if k == 2:
            x[:] = np.nan
        if k == 3:
            x[0, np.nonzero(allow[0])[0][0]] = np.nan
        if k == 4:
            x[:, 1000:] = np.nan
        if k == 5:
            x[:] = np.where(rng.random(x.shape) < 0.5, np.float32(0.0), np.float32(-0.0))
        if k == 6:
            x[:] = -np.inf
        if k == 7:
            x[:, 77], x[:, 4000] = np.inf, np.inf
            allow[:, 4000] = True
        if k == 8:
            x[:, 0] = np.nan
            allow[:, 0] = False
        if k == 9:
            x = rng.standard_normal((nt, vocab)).astype(np.float32)
        want = dc.logit_rules(x, (), None, None, 1, 0, 0, None, allow)
        check(run(dsv4, x, allow=allow), want)
        assert np.array_equal(run(dsv4, x, allow=allow, out=False)[1], want[1])
        got = run(dsv4, x, allow=allow, picks=False)
        assert common.bits_equal(np.nan_to_num(got[0]), np.nan_to_num(want[0]))


def test_without_rules_the_pick_is_the_heads(gpu, dsv4):
    """No rule at all: the rows unchanged and dsv4_gpu_argmax_d's picks."""
    import torch
    rng = np.random.default_rng(4)
    x = rng.standard_normal((6, 20001)).astype(np.float32)
    x[1, 0] = np.nan
    x[2, 5] = np.nan
    got, picks = run(dsv4, x)
    assert common.bits_equal(np.nan_to_num(got), np.nan_to_num(x))
    for t in range(6):
        tok = torch.zeros(1, device="cuda:0", dtype=torch.int32)
        row = dc.dev(x[t])
        assert gpu.dsv4_gpu_argmax_d(tok.data_ptr(), row.data_ptr(), 20001, dc.stream()) == 0
        assert tok.item() == picks[t]


@pytest.mark.parametrize("nt,vocab", [(1, 5), (1, 40001), (5, 8192), (64, 3001)])
@pytest.mark.parametrize("hist", [24576, 24577, 100003])
def test_long_histories(gpu, dsv4, nt, vocab, hist):
    """Histories that a launch of their own counts, and the same without a
    workspace, where only rows are asked for."""
    import torch
    rng = np.random.default_rng(nt * vocab + hist)
    x = (rng.standard_normal((nt, vocab)) * 3).astype(np.float32)
    ids = rng.integers(-3, vocab + 3, hist).astype(np.int32)
    drafts = rng.integers(-1, vocab + 1, nt).astype(np.int32)
    words = dc.words(rng, nt)
    want = dc.logit_rules(x, ids, drafts, words, 1.3, 0.25, 0.5, None, None)
    check(run(dsv4, x, ids, drafts, words, 1.3, 0.25, 0.5), want)
    keep = [dc.dev(a) for a in (x, ids, drafts, np.array(words, np.uint64))]
    out = torch.empty(nt, vocab, device="cuda:0")
    r = dsv4.LogitRules(hist=dc.ptr(keep[1]), n_hist=hist, draft=dc.ptr(keep[2]),
                        mask=dc.ptr(keep[3]), repetition=1.3, frequency=0.25, presence=0.5,
                        bias=None, allow=None, allow_stride=0)
    assert gpu.dsv4_gpu_logits_adjust_d(out.data_ptr(), None, dc.ptr(keep[0]), nt, vocab, vocab,
                                        ctypes.byref(r), None, 0, dc.stream()) == 0
    assert common.bits_equal(dc.host(out), want[0])
