"""Attention of a tree of drafted tokens over a cache (dsv4_gpu_tree_attn_d)
against softmax attention in 64 bits.

f32 q: within 1e-5 of the output vector (the contract of the sparse
attention). bf16 q: each weight and each output rounded to bf16 once, half a
step of 2^-8: |error| <= 2^-8 (|o| + sum |weight value|), and the f32
arithmetic's 1e-5 beside it."""
import numpy as np
import pytest

import common
import draft_common as dc

pytestmark = pytest.mark.gpu


def check(got, want, size, bf):
    assert np.isfinite(got).all()
    if bf:
        bound = dc.U16 * (np.abs(want) + size) * 1.01 + 1e-5 * size
        assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())
    else:
        err = common.vec_rel_err(got, want)
        assert err < 1e-5, err


def problem(seed, nt, h, dqk, ctx, fmt, bf, scale=1.0, page=0):
    """q, the sequence's rows as the cache holds them, the device cache with
    its pages shuffled, and the pages."""
    rng = np.random.default_rng(seed)
    q = (rng.standard_normal((nt, h, dqk)) * scale).astype(np.float32)
    q = dc.bf16(q) if bf else q
    n = ctx + nt
    pages = None
    rows = n
    if page:
        k = -(-n // page)
        pages = rng.permutation(k + 2)[:k].astype(np.int32)
        rows = (k + 2) * page
    v, s = dc.stored(rng.standard_normal((rows, dqk)), fmt)
    cache, ks = dc.cache_of(v, fmt, scales=s)
    at = np.arange(n)
    if page:
        at = pages[at // page].astype(np.int64) * page + at % page
    return rng, dc.to_fmt(q, bf), q, v[at], cache, ks, rows, None if pages is None else dc.dev(pages)


# (nt, h, dqk, dv, ctx): one token to 64, every width class and odd ones, contexts from none
# to several splits, tiles that end anywhere
SHAPES = [(1, 1, 1, 1, 0), (1, 64, 576, 512, 1), (1, 16, 512, 512, 31), (2, 3, 40, 24, 95),
          (1, 128, 576, 512, 4097), (5, 7, 33, 17, 130), (13, 5, 72, 40, 777),
          (64, 2, 128, 128, 64), (64, 16, 576, 512, 1000), (17, 40, 192, 128, 2050),
          (9, 11, 255, 200, 333), (33, 8, 570, 511, 150), (64, 64, 512, 512, 260)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("bf", [False, True])
def test_tree(gpu, dsv4, shape, fmt, bf):
    nt, h, dqk, dv, ctx = shape
    rng, dq, q, v, cache, ks, rows, _ = problem(nt + ctx, nt, h, dqk, ctx, fmt, bf, 1.5)
    w = dc.words(rng, nt)
    sink = rng.standard_normal(h).astype(np.float32)
    dw, dsink = dc.dev(np.array(w, np.uint64)), dc.dev(sink)
    scale = 1.0 / np.sqrt(dqk)
    rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx, dw, sink=dsink, scale=scale)
    assert rc == 0
    want, size = dc.attention(q, v, dc.visible(w, nt, ctx, 0), sink, scale, dv)
    check(dc.host(o), want, size, bf)


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, True), (2, False), (1, True)])
@pytest.mark.parametrize("page", [0, 1, 5, 16, 64])
@pytest.mark.parametrize("window", [0, 1, 7, 128, 5000])
def test_pages_windows_and_chains(gpu, dsv4, fmt, bf, page, window):
    """Pages that end inside a tile; windows down to the token itself; no
    words: every token sees those before it."""
    nt, h, dqk, dv, ctx = 11, 6, 96, 64, 517
    _, dq, q, v, cache, ks, rows, pages = problem(page + window, nt, h, dqk, ctx, fmt, bf, 1.0,
                                                  page)
    rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx, None, window, pages, page,
                    scale=0.2)
    assert rc == 0
    want, size = dc.attention(q, v, dc.visible(None, nt, ctx, window), None, 0.2, dv)
    check(dc.host(o), want, size, bf)


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, False), (1, True), (2, True)])
@pytest.mark.parametrize("dqk,dv", [(128, 128), (576, 512)])
def test_tokens_that_see_nothing_and_rows_nobody_may_see(gpu, dsv4, fmt, bf, dqk, dv):
    """An empty word with a window past the context, or no context: zeros, a
    sink or not. NaN and infinities in rows that a token does not see reach
    nothing of it; those that see one get NaN."""
    nt, h = 6, 4
    for ctx, window in ((0, 0), (40, 1)):
        rng, dq, q, v, cache, ks, rows, _ = problem(ctx, nt, h, dqk, ctx, fmt, bf)
        w = [0, 0b10, 0b100, 0b1010, 0b11110, 0]
        # row 4 of the drafts is poisoned; only token 4 sees it
        row = ctx + 4
        if fmt == 2:
            cache[row, 3] = 0x7F
            ks[row] = float("nan")
        else:
            cache[row, 1], cache[row, 2], cache[row, 3] = float("inf"), -float("inf"), float("nan")
        sink = dc.dev(rng.standard_normal(h).astype(np.float32))
        for sk in (None, sink):
            rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx,
                            dc.dev(np.array(w, np.uint64)), window, scale=0.3, sink=sk)
            assert rc == 0
            got = dc.host(o)
            see = dc.visible(w, nt, ctx, window)
            assert not see[0].any() and not see[5].any() and not see[:4, row].any()
            clean = v.copy()
            clean[row] = 0
            assert see[4, row]
            want, size = dc.attention(q, clean, see, None if sk is None else sk.cpu().numpy(),
                                      0.3, dv)
            assert (got[[0, 5]] == 0).all()
            check(got[:4], want[:4], size[:4], bf)
            assert np.isnan(got[4]).any(axis=1).all()


@pytest.mark.parametrize("fmt", [0, 1, 2])
def test_rows_and_pages_outside_the_cache(gpu, dsv4, fmt):
    """Positions whose page is missing, negative or past the cache are masked."""
    nt, h, dqk, dv, ctx, page = 3, 5, 64, 48, 100, 8
    rng, dq, q, v, cache, ks, rows, pages = problem(4, nt, h, dqk, ctx, fmt, False, 1.0, page)
    see = dc.visible(None, nt, ctx, 0)
    pages[2], pages[5], pages[7] = -1, rows // page, 2 ** 31 - 1
    for k in (2, 5, 7, 12):
        see[:, k * page:(k + 1) * page] = False
    rc, o = dc.tree(dsv4, dq, False, cache, ks, fmt, rows, dqk, dv, ctx, None, 0, pages, page,
                    n_pages=12, scale=0.2)
    assert rc == 0
    see[:, 12 * page:] = False
    want, size = dc.attention(q, v, see, None, 0.2, dv)
    check(dc.host(o), want, size, False)
    # a cache shorter than the sequence
    rng, dq, q, v, cache, ks, rows, _ = problem(5, nt, h, dqk, ctx, fmt, False)
    rc, o = dc.tree(dsv4, dq, False, cache, ks, fmt, 90, dqk, dv, ctx, scale=0.2)
    assert rc == 0
    see = dc.visible(None, nt, ctx, 0)
    see[:, 90:] = False
    want, size = dc.attention(q, v, see, None, 0.2, dv)
    check(dc.host(o), want, size, False)


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, False), (1, True)])
def test_scores_far_apart(gpu, dsv4, fmt, bf):
    """Scores of hundreds: the maximum moves late, weights vanish, and a sink
    far above or below. The scores' own rounding, 2^-22 of their size of 600
    at most, is that much of a weight: 1.5e-4."""
    nt, h, dqk, dv, ctx = 4, 16, 64, 64, 600
    rng, dq, q, v, cache, ks, rows, _ = problem(6, nt, h, dqk, ctx, fmt, bf, 8.0)
    for sk in (-200.0, 0.0, 300.0):
        sink = np.full(h, sk, np.float32)
        rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx, sink=dc.dev(sink),
                        scale=1.0)
        assert rc == 0
        want, size = dc.attention(q, v, dc.visible(None, nt, ctx, 0), sink, 1.0, dv)
        got = dc.host(o)
        rnd = dc.U16 * (np.abs(want) + size) if bf else 0
        assert (np.abs(got - want) <= rnd + 1.5e-4 * size + 1e-30).all()


@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("dqk,dv,stride,shift", [(64, 64, 72, 0), (64, 64, 65, 0),
                                                 (64, 32, 64, 1), (576, 512, 592, 0),
                                                 (512, 512, 513, 3)])
def test_strides_and_addresses(gpu, dsv4, fmt, dqk, dv, stride, shift):
    """Row pitches and bases that are not whole 16-byte pieces."""
    import torch
    rng = np.random.default_rng(stride)
    nt, h, ctx = 5, 3, 90
    v, s = dc.stored(rng.standard_normal((ctx + nt, dqk)), fmt)
    cache, ks = dc.cache_of(v, fmt, stride, s)
    flat = torch.zeros(cache.numel() + shift, device="cuda:0", dtype=cache.dtype)
    flat[shift:] = cache.flatten()
    q = rng.standard_normal((nt, h, dqk)).astype(np.float32)
    dq = torch.zeros(q.size + shift, device="cuda:0")
    dq[shift:] = dc.dev(q).flatten()
    dq = dq[shift:].view(nt, h, dqk)
    rc, o = dc.tree(dsv4, dq, False, flat[shift:], ks, fmt, ctx + nt, dqk, dv, ctx, scale=0.2,
                    stride=stride)
    assert rc == 0
    want, size = dc.attention(q, v, dc.visible(None, nt, ctx, 0), None, 0.2, dv)
    check(dc.host(o), want, size, False)


@pytest.mark.parametrize("fmt,bf", [(1, False), (2, True)])
def test_long_contexts_and_offsets_past_32_bits(gpu, dsv4, fmt, bf):
    """A cache whose rows start past 2^32 elements, most of it reached through
    pages that repeat a few."""
    import torch
    nt, h, dqk, dv, page = 2, 8, 512, 512, 64
    stride = 1 << 20
    rng = np.random.default_rng(12)
    rows = 64 * 65
    cache = torch.zeros(rows, stride, device="cuda:0", dtype=[None, torch.bfloat16, torch.uint8][fmt])
    ks = torch.ones(rows, device="cuda:0") if fmt == 2 else None
    v, s = dc.stored(rng.standard_normal((page * 2, dqk)), fmt)
    small, sks = dc.cache_of(v, fmt, scales=s)
    for k, at in enumerate((0, 64)):
        cache[at * page:(at + 1) * page, :dqk] = small[k * page:(k + 1) * page]
        if fmt == 2:
            ks[at * page:(at + 1) * page] = sks[k * page:(k + 1) * page]
    ctx = 20000
    n_pages = -(-(ctx + nt) // page)
    which = rng.integers(0, 2, n_pages)
    pages = dc.dev((which * 64).astype(np.int32))
    q = rng.standard_normal((nt, h, dqk)).astype(np.float32)
    q = dc.bf16(q) if bf else q
    rc, o = dc.tree(dsv4, dc.to_fmt(q, bf), bf, cache, ks, fmt, rows, dqk, dv, ctx, None, 0,
                    pages, page, scale=0.05, stride=stride)
    assert rc == 0
    at = np.arange(ctx + nt)
    full = v[which[at // page] * page + at % page]
    want, size = dc.attention(q, full, dc.visible(None, nt, ctx, 0), None, 0.05, dv)
    check(dc.host(o), want, size, bf)
    del cache
    torch.cuda.empty_cache()


def test_the_same_bits_again_and_the_workspace(gpu, dsv4):
    """A call repeats its bits whatever its workspace held; one byte less is
    refused."""
    import torch
    L = dsv4.lib()
    nt, h, dqk, dv, ctx = 3, 16, 576, 512, 9000
    _, dq, q, v, cache, ks, rows, _ = problem(1, nt, h, dqk, ctx, 1, False)
    need = L.dsv4_gpu_tree_attn_scratch_bytes(0, nt, h, dqk, dv, 1, ctx, 0)
    assert need >= L.dsv4_gpu_tree_attn_scratch_bytes(0, nt, h, dqk, dv, 1, ctx // 2, 0)
    outs = []
    for fill in (0, 255):
        space = torch.full((need + 64,), fill, device="cuda:0", dtype=torch.uint8)
        rc, o = dc.tree(dsv4, dq, False, cache, ks, 1, rows, dqk, dv, ctx, scale=0.04, space=space)
        assert rc == 0 and (space[need:] == fill).all()
        outs.append(dc.host(o))
    assert common.bits_equal(outs[0], outs[1])
    if need:
        space = torch.zeros(need - 1, device="cuda:0", dtype=torch.uint8)
        assert dc.tree(dsv4, dq, False, cache, ks, 1, rows, dqk, dv, ctx, scale=0.04,
                       space=space)[0] == -1


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, True)])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales_of_zero_and_below(gpu, dsv4, fmt, bf, scale):
    """A scale of 0 averages the visible rows; a negative one turns the order."""
    nt, h, dqk, dv, ctx = 5, 4, 64, 64, 70
    rng, dq, q, v, cache, ks, rows, _ = problem(9, nt, h, dqk, ctx, fmt, bf)
    w = dc.words(rng, nt)
    rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx,
                    dc.dev(np.array(w, np.uint64)), 20, scale=scale)
    assert rc == 0
    want, size = dc.attention(q, v, dc.visible(w, nt, ctx, 20), None, scale, dv)
    check(dc.host(o), want, size, bf)


# (nt, h, dqk, dv, ctx): workgroups of 16 rows of q and of all they can take, one split, a tile
# a split, over 64 splits, and joins of many rows, odd widths among them
PLANS = [(1, 16, 576, 512, 40), (1, 64, 576, 512, 1500), (2, 128, 576, 512, 6000),
         (1, 16, 512, 512, 16500), (1, 5, 96, 64, 20011), (64, 40, 100, 75, 700),
         (63, 33, 512, 509, 1100), (64, 128, 160, 128, 900), (64, 64, 576, 512, 2000)]


@pytest.mark.parametrize("shape", PLANS)
@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, False), (1, True), (2, True)])
def test_plans(gpu, dsv4, shape, fmt, bf):
    nt, h, dqk, dv, ctx = shape
    rng, dq, q, v, cache, ks, rows, pages = problem(nt * h + ctx, nt, h, dqk, ctx, fmt, bf, 1.0, 16)
    w = dc.words(rng, nt)
    sink = rng.standard_normal(h).astype(np.float32)
    scale = 1.0 / np.sqrt(dqk)
    rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx,
                    dc.dev(np.array(w, np.uint64)), 0, pages, 16, sink=dc.dev(sink), scale=scale)
    assert rc == 0
    # rows of q of a few heads, the first and the last among them
    few = sorted({0, h // 3, h - 1})
    want, size = dc.attention(q[:, few], v, dc.visible(w, nt, ctx, 0), sink[few], scale, dv)
    check(dc.host(o)[:, few], want, size, bf)


@pytest.mark.parametrize("bf", [False, True])
@pytest.mark.parametrize("fmt", [0, 1, 2])
@pytest.mark.parametrize("ctx", [1, 31, 32, 33, 63, 64, 96, 127])
def test_edges_of_tiles_and_windows(gpu, dsv4, fmt, bf, ctx):
    """Contexts that end at, before and after a tile's end, with windows of the
    same lengths: whole tiles inside the window, at its edge and none."""
    nt, h, dqk, dv = 40, 2, 64, 64
    rng, dq, q, v, cache, ks, rows, _ = problem(ctx, nt, h, dqk, ctx, fmt, bf)
    w = dc.words(rng, nt)
    dw = dc.dev(np.array(w, np.uint64))
    for window in (0, 1, 31, 32, 33, 64, ctx, ctx + nt):
        rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, dqk, dv, ctx, dw, window, scale=0.2)
        assert rc == 0
        want, size = dc.attention(q, v, dc.visible(w, nt, ctx, window), None, 0.2, dv)
        check(dc.host(o), want, size, bf)


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, False), (0, True), (1, True),
                                    (2, True)])
@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 8, 9, 15, 63, 65, 129, 257, 449, 513, 575])
def test_rows_of_any_width(gpu, dsv4, fmt, bf, d):
    """Rows of less than one piece of eight elements, and last pieces of any
    length in every width class."""
    nt, h, ctx = 4, 5, 45
    rng, dq, q, v, cache, ks, rows, _ = problem(d, nt, h, d, ctx, fmt, bf)
    dv = min(d, 512)
    rc, o = dc.tree(dsv4, dq, bf, cache, ks, fmt, rows, d, dv, ctx, scale=0.3)
    assert rc == 0
    want, size = dc.attention(q, v, dc.visible(None, nt, ctx, 0), None, 0.3, dv)
    check(dc.host(o), want, size, bf)
