"""Page tables and row maps of a batch's step (dsv4_gpu_reqs_tables_d) against a
scheduler that goes request by request; all of them whole numbers."""
import ctypes

import numpy as np
import pytest

import draft_common as dc
import reqs_common as rc

pytestmark = pytest.mark.gpu


def call(dsv4, have, new, table, ring, free, page, shared, max_tok, in_place=False, maps=True):
    import torch
    n = len(have)
    d = {k: dc.dev(np.asarray(v, np.int32)) for k, v in dict(
        have=have, new=new, pages=table, ring=ring, free=free).items()}
    d["len"] = d["have"] if in_place else torch.full((max(n, 1),), 77, device="cuda:0",
                                                     dtype=torch.int32)
    d["out"] = d["free"] if in_place else torch.full((2,), 77, device="cuda:0", dtype=torch.int32)
    d["first"] = torch.full((n + 2,), 77, device="cuda:0", dtype=torch.int32)
    for k in ("rows", "pos", "req"):
        d[k] = torch.full((max_tok + 4,), 77, device="cuda:0", dtype=torch.int32)
    r = rc.reqs(dsv4, d["len"], d["pages"], d["first"], page, max_tok, shared)
    m = [d[k].data_ptr() if maps else None for k in ("rows", "pos", "req")]
    assert dsv4.lib().dsv4_gpu_reqs_tables_d(
        ctypes.byref(r), d["have"].data_ptr(), d["new"].data_ptr(), d["ring"].data_ptr(),
        len(ring), d["free"].data_ptr(), d["out"].data_ptr(), *m, dc.stream()) == 0
    torch.cuda.synchronize()
    g = {k: v.cpu().numpy() for k, v in d.items()}
    assert g["first"][n + 1] == 77
    for k in ("rows", "pos", "req"):
        assert (g[k][max_tok:] == 77).all() and (maps or (g[k] == 77).all())
        g[k] = g[k][:max_tok]
    return dict(first=g["first"][:n + 1], len=g["len"][:n], pages=g["pages"], ring=g["ring"],
                free=g["out"], rows=g["rows"], pos=g["pos"], req=g["req"])


def same(got, want, keys=None):
    for k in keys or want:
        assert np.array_equal(got[k], np.asarray(want[k]).reshape(got[k].shape)), k


@pytest.mark.parametrize("n_req,page,kind", [
    (1, 64, "one"), (2, 1, "drafts"), (63, 16, "one"), (64, 16, "drafts"), (65, 7, "prompts"),
    (256, 64, "prompts"), (257, 64, "one"), (300, 1, "prompts"), (1000, 33, "prompts"),
    (1025, 16, "drafts"), (4096, 16, "one"), (4096, 16, "prompts")])
@pytest.mark.parametrize("room", ["all", "pages", "tokens"])
def test_steps(gpu, dsv4, n_req, page, kind, room):
    """Requests that wait, end and start, pages or tokens that run out."""
    rng = np.random.default_rng(n_req * 131 + page)
    shared = int(rng.integers(0, 100))
    have = shared + rng.integers(0, 300, n_req)
    have[rng.random(n_req) < 0.1] = 0
    hi = {"one": 2, "drafts": 9, "prompts": 200}[kind]
    new = rng.integers(1, hi, n_req)
    if kind == "prompts":
        new = np.where(rng.random(n_req) < 0.8, 1, new)
    new[rng.random(n_req) < 0.1] = 0
    new[rng.random(n_req) < 0.1] = -1
    width = -(-(shared + 520) // page)
    total = int(new[new > 0].sum())
    need = int(sum(-(-(h + n) // page) - -(-h // page) for h, n in zip(have, new) if n > 0))
    table, ring, free = rc.pool(rng, have, page, shared, need // 2 if room == "pages" else need + 3,
                                width)
    max_tok = total * 2 // 3 if room == "tokens" else total + 5
    args = (have, new, table, ring, free, page, shared, max_tok)
    want = rc.schedule(*args)
    same(call(dsv4, *args), want)
    same(call(dsv4, *args, in_place=True), want)
    same(call(dsv4, *args, maps=False), want, ("first", "len", "pages", "ring", "free"))


def test_lengths_and_states_that_do_not_fit(gpu, dsv4):
    """Negative and too long lengths, huge counts, tables that are full to the last
    row, negative pages, a ring's place out of range, pages behind a full ring."""
    page = 8
    rng = np.random.default_rng(5)
    big = 2 ** 31 - 1
    have = np.array([32, 31, 24, 25, -1, -5, 33, big, 0, 16, big, -3])
    new = np.array([1, 1, 8, 8, 1, -1, -1, 1, big, 1, -1, 0])
    table = rng.permutation(200)[:12 * 4].reshape(12, 4).astype(np.int32)
    table[1, 3] = -2
    table[9, 2] = big                            # not taken: position 16 gets a new page
    ring = rng.permutation(200)[:50].astype(np.int32)
    for free in ([49, 10], [3, 48], [0, 0]):
        args = (have, new, table, ring, free, page, 0, 40)
        same(call(dsv4, *args), rc.schedule(*args))
    # a place that is not one counts as none, and more pages than a ring holds as all
    for free, means in (([-1, 5], [0, 5]), ([50, 5], [0, 5]), ([3, 99], [3, 50]),
                        ([3, -4], [3, 0])):
        got = call(dsv4, have, new, table, ring, free, page, 0, 40)
        same(got, rc.schedule(have, new, table, ring, means, page, 0, 40))
    # rows past the last that a row number can name
    table[:] = 2 ** 28 + np.arange(48).reshape(12, 4)
    args = (np.full(12, 3), np.full(12, 1), table, ring, [0, 50], page, 0, 12)
    want = rc.schedule(*args)
    assert (np.asarray(want["rows"]) == -1).all()
    same(call(dsv4, *args), want)
    # no requests, no tokens
    none = np.zeros(0, np.int32)
    got = call(dsv4, none, none, np.zeros((0, 4), np.int32), ring, [7, 9], page, 0, 3)
    assert got["first"].tolist() == [0] and got["free"].tolist() == [7, 9]
    assert got["rows"].tolist() == got["pos"].tolist() == got["req"].tolist() == [-1] * 3
    args = (have, new, table, ring, [0, 50], page, 0, 0)
    same(call(dsv4, *args), rc.schedule(*args))


def test_captured_steps_go_on_in_place(gpu, dsv4):
    """One captured call, replayed step after step on its own lengths, tables and
    ring, with eager calls of another batch between."""
    import torch
    rng = np.random.default_rng(9)
    n_req, page, max_tok = 70, 4, 90
    lens = rng.integers(0, 40, n_req)
    table, ring, free = rc.pool(rng, lens, page, 0, 300, 64)
    d = {k: dc.dev(np.asarray(v, np.int32)) for k, v in dict(
        len=lens, pages=table, ring=ring, free=free, new=np.ones(n_req)).items()}
    d["first"] = torch.zeros(n_req + 1, device="cuda:0", dtype=torch.int32)
    maps = [torch.zeros(max_tok, device="cuda:0", dtype=torch.int32) for _ in range(3)]
    r = rc.reqs(dsv4, d["len"], d["pages"], d["first"], page, max_tok)

    def queue(st):
        assert dsv4.lib().dsv4_gpu_reqs_tables_d(
            ctypes.byref(r), d["len"].data_ptr(), d["new"].data_ptr(), d["ring"].data_ptr(),
            len(ring), d["free"].data_ptr(), d["free"].data_ptr(), *[m.data_ptr() for m in maps],
            st) == 0

    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=side):
        queue(torch.cuda.current_stream().cuda_stream)
    have, other = lens, (rng.integers(0, 50, 300), np.ones(300, np.int32))
    for step in range(8):
        new = rng.choice([1, 1, 1, 2, 3, 0, -1], n_req).astype(np.int32)
        d["new"].copy_(dc.dev(new))
        torch.cuda.synchronize()
        want = rc.schedule(have, new, table, ring, free, page, 0, max_tok)
        g.replay()
        ot, oring, ofree = rc.pool(rng, other[0], page, 0, 300, 64)
        call(dsv4, *other, ot, oring, ofree, page, 0, 300)
        torch.cuda.synchronize()
        have, table, ring, free = want["len"], want["pages"], want["ring"], want["free"]
        for k in ("len", "pages", "ring", "free", "first"):
            assert np.array_equal(d[k].cpu().numpy().reshape(-1), np.asarray(want[k]).reshape(-1)), (step, k)
        for m, k in zip(maps, ("rows", "pos", "req")):
            assert np.array_equal(m.cpu().numpy(), want[k]), (step, k)
