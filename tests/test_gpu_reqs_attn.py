"""Attention of a batch of requests over their pages (dsv4_gpu_reqs_plan_d,
dsv4_gpu_reqs_attn_d) against softmax attention in 64 bits, request by request.

f32 q: within 1e-5 of the output vector. bf16 q: each weight and each output
rounded to bf16 once, half a step of 2^-8: |error| <= 2^-8 (|o| + sum |weight
value|), and the f32 arithmetic's 1e-5 beside it."""
import numpy as np
import pytest

import common
import draft_common as dc
import reqs_common as rc

pytestmark = pytest.mark.gpu


def check(got, want, size, bf):
    assert np.isfinite(got).all()
    if bf:
        bound = dc.U16 * (np.abs(want) + size) * 1.01 + 1e-5 * size
        assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())
    else:
        err = common.vec_rel_err(got, want)
        assert err < 1e-5, err


# (lens, tokens, h, dqk, dv, page): one token of one position up to pieces of prompts, every
# width class and odd ones, requests without tokens, lengths that end anywhere in a page
SHAPES = [
    ([1], [1], 1, 1, 1, 1),
    ([1, 1, 2], [1, 1, 2], 3, 8, 8, 16),
    ([31, 32, 33], [1, 1, 1], 64, 576, 512, 16),
    ([700, 1, 64, 65, 0, 300], [1, 1, 0, 3, 0, 8], 5, 72, 40, 7),
    ([5000, 20], [1, 1], 16, 512, 512, 64),
    ([128] * 40, [1] * 40, 4, 128, 128, 32),
    ([300, 40, 900], [150, 40, 1], 7, 255, 200, 5),
    ([97, 211], [97, 70], 33, 192, 128, 64),
    ([260, 10], [130, 10], 12, 570, 511, 100),
    ([2050], [33], 40, 512, 512, 16),
    ([100, 64], [3, 2], 300, 33, 17, 1),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("bf", [False, True])
def test_shapes(gpu, dsv4, shape, fmt, bf):
    lens, news, h, dqk, dv, page = SHAPES[shape]
    b = rc.Batch(shape, lens, news, h, dqk, fmt, bf, page, scale=1.5, room=shape % 3)
    sink = b.rng.standard_normal(h).astype(np.float32) if shape % 2 else None
    scale = 1 / np.sqrt(dqk)
    got = b.call(dsv4, dv, 0, None if sink is None else dc.dev(sink), scale)
    check(got, *b.want(dv, 0, sink, scale), bf)


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, True), (2, False), (1, True)])
@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 100, 517])
@pytest.mark.parametrize("window", [0, 1, 40, 128, 5000])
def test_prefixes_and_windows(gpu, dsv4, fmt, bf, prefix, window):
    """A prefix that ends inside a tile or a page; requests that end inside it, or have
    no tokens; windows that start in it and behind it."""
    own = [1, 30, 64, 5, 200, 17, 90]
    lens = [prefix + n for n in own] + [max(prefix // 2, 4), max(prefix - 1, 3)]
    news = [1, 2, 0, 5, 1, 17, 3, 2, 1]
    b = rc.Batch(prefix * 7 + window, lens, news, 6, 96, fmt, bf, 16, prefix)
    got = b.call(dsv4, 64, window, scale=0.2)
    check(got, *b.want(64, window, None, 0.2), bf)


@pytest.mark.parametrize("fmt,bf", [(1, True), (2, False), (0, True)])
@pytest.mark.parametrize("dqk,dv", [(128, 128), (576, 512)])
@pytest.mark.parametrize("n_req,h,prefix,longest", [
    (2, 64, 4096, 60), (40, 64, 1000, 3), (300, 3, 333, 40), (9, 128, 0, 3000), (130, 16, 64, 700)])
def test_batches(gpu, dsv4, fmt, bf, dqk, dv, n_req, h, prefix, longest):
    """Batches that split what they share, what they do not, both and neither."""
    rng = np.random.default_rng(n_req)
    lens = prefix + np.exp(rng.uniform(0, np.log(longest), n_req)).astype(int)
    b = rc.Batch(n_req, lens, np.ones(n_req, int), h, dqk, fmt, bf, 16, prefix, 1.2)
    sink = rng.standard_normal(h).astype(np.float32)
    got = b.call(dsv4, dv, 0, dc.dev(sink), 0.06)
    check(got, *b.want(dv, 0, sink, 0.06), bf)


@pytest.mark.parametrize("fmt,bf", [(1, True), (0, False)])
@pytest.mark.parametrize("n_req,h,prefix,length,room", [
    (3, 64, 0, 300, 9000), (300, 64, 96, 110, 0), (300, 64, 96, 110, 3000), (2, 1, 0, 2000, 100000)])
def test_room_for_many_more_tokens(gpu, dsv4, fmt, bf, n_req, h, prefix, length, room):
    """Few tokens where the step's buffers hold many, and many rows that are joined."""
    b = rc.Batch(room + n_req, [length] * n_req, [1] * n_req, h, 40, fmt, bf, prefix=prefix, room=room)
    check(b.call(dsv4, 24), *b.want(24), bf)


def test_idle_requests_that_are_long(gpu, dsv4):
    """Requests without tokens in this step have no part in it, whatever their length."""
    b = rc.Batch(3, [70, 9000, 40, 130, 20000], [1, 0, 3, 1, 0], 16, 128, 1, True, prefix=64)
    check(b.call(dsv4, 128), *b.want(128), True)


def test_the_most_requests(gpu, dsv4):
    rng = np.random.default_rng(2)
    lens = rng.integers(0, 50, 4096)
    news = np.minimum(rng.integers(0, 3, 4096), lens)
    b = rc.Batch(1, lens, news, 2, 64, 1, False, 8)
    check(b.call(dsv4, 64, scale=0.2), *b.want(64, scale=0.2), False)


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, False), (1, True), (2, True)])
@pytest.mark.parametrize("prefix", [0, 64])
def test_rows_that_nobody_may_see(gpu, dsv4, fmt, bf, prefix):
    """NaN and infinities in all rows that are no position of a request, and in one
    position of one request: they reach the tokens that see that one, and no other."""
    lens, news = [prefix + n for n in (70, 33, 40, 5)], [4, 1, 6, 2]
    b = rc.Batch(prefix + fmt, lens, news, 4, 128, fmt, bf, 16, prefix)
    used = np.zeros(b.rows, bool)
    for i, n in enumerate(lens):
        used[[b.row(i, p) for p in range(n)]] = True
    bad = ~used
    poisoned = b.row(2, lens[2] - 3)             # seen by the last three tokens of request 2
    bad[poisoned] = True
    at = dc.dev(np.nonzero(bad)[0])
    if fmt == 2:
        b.cache[at, 3] = 0x7F
        b.ks[at] = float("nan")
    else:
        b.cache[at, 1], b.cache[at, 2] = float("inf"), -float("inf")
        b.cache[at, 3] = float("nan")
    got = b.call(dsv4, 128, 0, None, 0.1)
    x = b.x.copy()
    x[bad] = 0
    want, size = b.want(128, 0, None, 0.1, x=x)
    hit = np.zeros(b.tokens, bool)
    hit[b.first[3] - 3:b.first[3]] = True
    check(got[~hit], want[~hit], size[~hit], bf)
    assert np.isnan(got[hit]).any(axis=(1, 2)).all()


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, True), (2, False)])
@pytest.mark.parametrize("prefix", [0, 96])
def test_pages_that_are_not_there(gpu, dsv4, fmt, bf, prefix):
    """Negative pages and pages behind the cache are masked; with all of them gone a
    token gets zeros, a sink or not."""
    lens, news = [prefix + n for n in (200, 150, 64, 20)], [3, 1, 5, 2]
    b = rc.Batch(5, lens, news, 6, 200, fmt, bf, 16, prefix)
    own = prefix // 16
    b.table[0, own + 1], b.table[0, own + 3], b.table[1, own] = -1, 2 ** 31 - 1, b.rows // 16
    b.table[3, own:] = -7
    if prefix:
        b.table[:, 2] = -1
    else:
        b.table[2, :] = 2 ** 27
    b.dev["pages"] = dc.dev(b.table)
    sink = b.rng.standard_normal(6).astype(np.float32)
    for sk in (None, sink):
        got = b.call(dsv4, 150, 0, None if sk is None else dc.dev(sk), 0.1)
        check(got, *b.want(150, 0, sk, 0.1), bf)
    if not prefix:
        assert (got[b.first[2]:] == 0).all()


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (1, True), (2, False), (2, True)])
@pytest.mark.parametrize("dqk,stride", [(64, 72), (63, 67), (576, 577), (7, 9)])
def test_strides(gpu, dsv4, fmt, bf, dqk, stride):
    b = rc.Batch(dqk, [100, 37, 300], [2, 9, 1], 5, dqk, fmt, bf, 16, stride=stride)
    dv = min(dqk, 512)
    check(b.call(dsv4, dv, scale=0.1), *b.want(dv, scale=0.1), bf)


def test_tokens_that_start_behind_the_first_row(gpu, dsv4):
    """first[0] > 0: the rows before it stay as they are."""
    b = rc.Batch(3, [40, 50, 7], [2, 3, 1], 4, 128, 1, False, 16, room=4)
    b.q = np.concatenate([b.q[:4], b.q[:6]])
    b.dq = dc.dev(b.q)
    b.dev["first"] += 4
    b.buffers(dsv4, 128)
    assert b.make_plan(dsv4, 128) == 0 and b.attend(dsv4, 128, scale=0.1) == 0
    got = dc.host(b.o)
    assert (got[:4] == 99).all() and (got[10:] == 99).all()
    b.q = b.q[4:]
    check(got[4:10], *b.want(128, scale=0.1), False)


def test_plans_that_do_not_fit(gpu, dsv4):
    """Lengths and first tokens that cannot be, and plans of other sizes: NaN in all
    rows, and nothing out of range; no tokens at all: nothing."""
    b = rc.Batch(4, [40, 50, 7], [2, 3, 1], 4, 128, 2, True, 16, room=2)
    good = {k: v.clone() for k, v in b.dev.items()}
    room = b.table.shape[1] * 16

    def go(sizes=None, **kw):
        b.dev = {k: v.clone() for k, v in good.items()}
        for k, v in kw.items():
            b.dev[k] = dc.dev(np.asarray(v, np.int32))
        b.buffers(dsv4, 128)
        assert b.make_plan(dsv4, 128) == 0
        assert b.attend(dsv4, 128, **(sizes or {})) == 0
        return dc.host(b.o)

    assert np.isfinite(go()).all()
    for kw in (dict(len=[40, 2, 7]), dict(len=[40, 50, -1]), dict(len=[room + 1, 50, 7]),
               dict(len=[40, 2 ** 31 - 1, 7]), dict(first=[-1, 2, 5, 6]), dict(first=[0, 2, 5, 9]),
               dict(first=[0, 5, 2, 6]), dict(first=[0, 2 ** 31 - 1, 5, 6]),
               dict(sizes=dict(prefix=32)), dict(sizes=dict(window=7)), dict(sizes=dict(page=8))):
        got = go(**kw)
        assert np.isnan(got[:b.max_tok]).all() and (got[b.max_tok:] == 99).all(), kw
    # (a request without tokens may have any length)
    got = go(first=[0, 0, 3, 4], len=[-5, 50, 7])
    assert np.isfinite(got[:4]).all() and (got[4:] == 99).all()
    assert (go(first=[3, 3, 3, 3]) == 99).all()


def test_rows_past_32_bits(gpu, dsv4):
    """Pages whose rows lie past 2^32 bytes of the cache."""
    import torch
    b = rc.Batch(6, [300, 90], [2, 5], 16, 576, 1, True, 64)
    k = 4300000 // 64                            # pages before: 4.95e9 bytes
    big = torch.zeros((k * 64 + b.rows, 576), device="cuda:0", dtype=torch.bfloat16)
    big[k * 64:] = b.cache
    want = b.want(512, scale=0.05)
    b.cache, b.rows = big, big.shape[0]
    b.dev["pages"] = torch.where(b.dev["pages"] >= 0, b.dev["pages"] + k, -1)
    check(b.call(dsv4, 512, scale=0.05), *want, True)


def test_captured_with_lengths_that_change(gpu, dsv4):
    """A plan and two layers' attention in a graph, replayed with other lengths, pages and
    queries and eager calls between; the same bits as the eager calls."""
    import torch
    b = rc.Batch(8, [700, 330, 64, 1000], [1, 4, 2, 1], 16, 128, 1, False, 16, 320)
    other = rc.Batch(9, [100, 90], [3, 2], 8, 128, 2, True, 16)
    b.buffers(dsv4, 128)
    o2 = torch.zeros_like(b.o)

    def queue(st):
        assert b.make_plan(dsv4, 128, st=st) == 0
        assert b.attend(dsv4, 128, scale=0.1, st=st) == 0
        first, b.o = b.o, o2
        assert b.attend(dsv4, 128, scale=0.2, st=st) == 0
        b.o = first

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        queue(torch.cuda.current_stream().cuda_stream)
    for lens, news in (([700, 330, 64, 1000], [1, 4, 2, 1]), ([701, 340, 40, 1], [1, 2, 4, 1]),
                       ([321, 322, 323, 324], [2, 2, 2, 2]), ([900, 5, 6, 7], [5, 1, 1, 1]),
                       ([0, 0, 0, 600], [0, 0, 0, 8])):
        b.lens, b.news = lens, news
        b.first = np.concatenate([[0], np.cumsum(news)])
        b.dev["len"].copy_(dc.dev(np.array(lens, np.int32)))
        b.dev["first"].copy_(dc.dev(b.first.astype(np.int32)))
        b.dev["pages"].copy_(dc.dev(b.rng.integers(0, b.rows // 16, b.table.shape).astype(np.int32)))
        b.dev["pages"][:, :20] = b.dev["pages"][0, :20]
        b.dq.copy_(dc.dev(b.rng.standard_normal(b.q.shape).astype(np.float32)))
        b.o.fill_(99), o2.fill_(99)
        torch.cuda.synchronize()
        g.replay()
        other.call(dsv4, 128, scale=0.1)
        torch.cuda.synchronize()
        got = dc.host(b.o), dc.host(o2)
        b.table, b.q = b.dev["pages"].cpu().numpy(), dc.host(b.dq)
        want, size = b.want(128, scale=0.1)
        n = int(b.first[-1])
        check(got[0][:n], want, size, False)
        b.o.fill_(99), o2.fill_(99)
        queue(dc.stream())
        torch.cuda.synchronize()
        assert common.bits_equal(got[0], dc.host(b.o)) and common.bits_equal(got[1], dc.host(o2))


def test_two_streams_at_once(gpu, dsv4):
    import torch
    jobs = [rc.Batch(1, [3000, 700, 2500], [1, 2, 1], 64, 576, 1, True, 64, 600),
            rc.Batch(2, [500] * 20, [1] * 20, 16, 512, 2, False, 16)]
    dvs, alone = (512, 512), []
    for b, dv in zip(jobs, dvs):
        alone.append(b.call(dsv4, dv, scale=0.05))
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(5):
        for b, dv, st in zip(jobs, dvs, streams):
            assert b.make_plan(dsv4, dv, st=st.cuda_stream) == 0
            assert b.attend(dsv4, dv, scale=0.05, st=st.cuda_stream) == 0
    torch.cuda.synchronize()
    for b, want in zip(jobs, alone):
        assert common.bits_equal(dc.host(b.o)[:b.tokens], want)
