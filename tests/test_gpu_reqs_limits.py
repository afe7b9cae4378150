"""Batches of requests at their ends: tables of 2^30 positions, and who has which pages
over a batch's life."""
import ctypes

import numpy as np
import pytest

import draft_common as dc
import reqs_common as rc
from test_gpu_reqs_attn import check
from test_gpu_reqs_tables import call, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, True), (2, False)])
@pytest.mark.parametrize("page", [1 << 20, (1 << 20) - 1])
def test_attention_at_the_last_positions(gpu, dsv4, fmt, bf, page):
    """Windows that end at a table's last position; each of its pages is the same."""
    import torch
    L, h, d, dv, window = dsv4.lib(), 4, 64, 48, 200
    pages, news = 1 << 10, [3, 1]
    lens = [pages * page, pages * page - page // 2]
    rng = np.random.default_rng(fmt)
    near = {n: (n - window - 8 + np.arange(window + 8)) % page for n in lens}
    at = np.unique(np.concatenate(list(near.values())))
    x, s = dc.stored(rng.standard_normal((len(at), d)), fmt)
    part, ps = dc.cache_of(x, fmt, scales=s)
    cache = torch.zeros((page, d), device="cuda:0", dtype=part.dtype)
    cache[dc.dev(at)] = part
    ks = None if ps is None else torch.ones(page, device="cuda:0")
    if ks is not None:
        ks[dc.dev(at)] = ps
    held = dict(zip(at.tolist(), x))
    tok = sum(news)
    q = rng.standard_normal((tok, h, d)).astype(np.float32)
    q = dc.bf16(q) if bf else q
    dq = dc.to_fmt(q, bf)
    g = {k: dc.dev(np.asarray(v, np.int32)) for k, v in dict(
        len=lens, first=[0, 3, 4], pages=np.zeros((2, pages))).items()}
    r = rc.reqs(dsv4, g["len"], g["pages"], g["first"], page, tok)
    space = lambda n: torch.zeros(n, device="cuda:0", dtype=torch.uint8)
    plan = space(L.dsv4_gpu_reqs_plan_bytes(2, tok, h))
    ws = space(L.dsv4_gpu_reqs_attn_scratch_bytes(int(bf), h, d, dv, fmt, 2, tok))
    o = torch.zeros((tok, h, dv), device="cuda:0", dtype=dq.dtype)
    assert L.dsv4_gpu_reqs_plan_d(plan.data_ptr(), plan.numel(), ctypes.byref(r), int(bf), h, d, dv,
                                  fmt, window, dc.stream()) == 0
    assert L.dsv4_gpu_reqs_attn_d(
        o.data_ptr(), dq.data_ptr(), int(bf), h, d, dv, cache.data_ptr(), dc.ptr(ks), fmt, d, page,
        ctypes.byref(r), plan.data_ptr(), plan.numel(), window, None, ctypes.c_float(0.2),
        ws.data_ptr(), ws.numel(), dc.stream()) == 0
    torch.cuda.synchronize()
    got, t0 = dc.host(o), 0
    for n, k in zip(lens, news):
        pos = np.arange(n - window - k, n)
        rows = np.array([held[p % page] for p in pos.tolist()])
        own = np.arange(n - k, n)[:, None]
        see = (pos[None] <= own) & (own - pos[None] < window)
        want, size = dc.attention(q[t0:t0 + k], rows, see, None, np.float32(0.2), dv)
        check(got[t0:t0 + k], want, size, bf)
        t0 += k


@pytest.mark.parametrize("page", [1 << 20, (1 << 20) - 1, 1 << 30])
def test_tables_at_the_last_positions(gpu, dsv4, page):
    width = (1 << 30) // page
    room = width * page
    have = np.array([room - 1, room - 5, room, room - page, 0, max(0, room - page - 3), room])
    new = np.array([1, 6, 1, page, room, 5, -1])
    table = np.arange(7 * width).reshape(7, width).astype(np.int32) % 500
    ring = np.arange(3000, dtype=np.int32)
    for max_tok in (20, 1 << 20):
        args = (have, new, table, ring, [2900, 2500], page, 0, max_tok)
        same(call(dsv4, *args), rc.schedule(*args))


def test_pages_come_back(gpu, dsv4):
    """Requests that begin behind the shared pages give all of theirs back, whatever the
    steps between; one that grows through them leaves as many pages as it filled for all."""
    rng = np.random.default_rng(2)
    page, shared, n = 4, 8, 9
    ring = np.arange(2, 102, dtype=np.int32)     # pages 0 and 1 are the shared ones
    table = np.full((n, 30), -1, np.int32)
    table[:, :2] = [0, 1]
    state = dict(len=np.full(n, shared), pages=table, ring=ring, free=[40, 100])
    step = lambda s, new, prefix: call(dsv4, s["len"], new, s["pages"], s["ring"], s["free"], page,
                                       prefix, 100)
    for _ in range(12):
        state = step(state, rng.choice([0, 1, 1, 2, 7], n), shared)
    used = (-(-state["len"] // page) - 2).sum()
    assert used > 0 and state["free"][1] == 100 - used
    state = step(state, np.full(n, -1), shared)
    assert state["free"][1] == 100 and sorted(state["ring"].tolist()) == list(range(2, 102))
    # 14 tokens from 0 are four pages, of which two are the prefix's
    state["len"] = np.zeros(n, np.int32)
    state = step(state, np.array([14] + [0] * (n - 1)), shared)
    assert state["free"][1] == 96
    mine = state["pages"][0, :4].tolist()
    state = step(state, np.array([-1] + [0] * (n - 1)), shared)
    assert state["free"][1] == 98
    at = (state["free"][0] + 96 + np.arange(2)) % 100
    assert state["ring"][at].tolist() == mine[2:]
    # and without a prefix all of them come back
    state["len"] = np.zeros(n, np.int32)
    state = step(state, np.array([14] + [0] * (n - 1)), 0)
    state = step(state, np.array([-1] + [0] * (n - 1)), 0)
    assert state["free"][1] == 98
