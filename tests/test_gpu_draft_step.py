"""The operators on drafted tokens as a program uses them together: rotate,
append, attend, score, pick; then keep the accepted path and go on. And what
they promise beside their results: streams, captured graphs, repeated bits."""
import ctypes

import numpy as np
import pytest

import common
import draft_common as dc

pytestmark = pytest.mark.gpu

H, D, ROT, VOCAB, PAGE = 8, 128, 32, 3001, 16


class Step:
    """A sequence over a paged cache, and one step's buffers."""

    def __init__(self, dsv4, fmt, bf, seed, nt):
        import torch
        self.dsv4, self.fmt, self.bf, self.nt = dsv4, fmt, bf, nt
        self.L = dsv4.lib()
        rng = self.rng = np.random.default_rng(seed)
        self.n_pages = 40
        self.pages = rng.permutation(self.n_pages + 3)[:self.n_pages].astype(np.int32)
        self.rows = (self.n_pages + 3) * PAGE
        v, s = dc.stored(np.zeros((self.rows, D)), fmt)
        self.cache, self.ks = dc.cache_of(v, fmt, scales=s)
        self.cos, self.sin = dc.tables(700, ROT)
        self.dcos, self.dsin = dc.dev(self.cos), dc.dev(self.sin)
        self.dpages = dc.dev(self.pages)
        self.head = rng.standard_normal((VOCAB, H * D)).astype(np.float32) * 0.05
        self.dt = torch.bfloat16 if bf else torch.float32
        self.o = torch.zeros(nt, H, D, device="cuda:0", dtype=self.dt)
        self.logits = torch.zeros(nt, VOCAB, device="cuda:0")
        self.pick = torch.zeros(nt, device="cuda:0", dtype=torch.int32)
        self.dhead = dc.dev(self.head)
        self.hist = np.zeros(0, np.int32)

    def row_of(self, pos):
        return self.pages[pos // PAGE] * PAGE + pos % PAGE

    def append(self, x, pos, at, st):
        """Rotate and store rows x (host) at positions pos, cache rows at."""
        self.keep = [dc.dev(x), dc.dev(pos.astype(np.int32)), dc.dev(at.astype(np.int32))]
        rp = dc.rope_struct(self.dsv4, self.dcos, self.dsin, ROT, D - ROT, False)
        assert self.L.dsv4_gpu_kv_append_d(
            self.cache.data_ptr(), dc.ptr(self.ks), self.fmt, D, self.rows,
            self.keep[0].data_ptr(), 0, D, len(x), D, self.keep[2].data_ptr(), 0,
            ctypes.byref(rp), self.keep[1].data_ptr(), st) == 0

    def verify(self, q, kv, ctx, w, toks, st):
        """Queue one step on st; buffers stay in self."""
        import torch
        nt, L = self.nt, self.L
        depth = np.array([bin(w[t] & ~(1 << t)).count("1") for t in range(nt)])
        pos = ctx + depth                        # a draft's place, not its slot
        self.append(kv, pos, self.row_of(ctx + np.arange(nt)), st)
        self.dq = dc.to_fmt(q, self.bf)
        self.dpos, self.dw = dc.dev(pos.astype(np.int32)), dc.dev(np.array(w, np.uint64))
        self.dtoks, self.dhist = dc.dev(toks), dc.dev(self.hist)
        n = L.dsv4_gpu_tree_attn_scratch_bytes(int(self.bf), nt, H, D, D, self.fmt, ctx, 0)
        self.space = torch.zeros(max(n, 16), device="cuda:0", dtype=torch.uint8)
        self.lspace = torch.zeros(L.dsv4_gpu_logits_scratch_bytes(nt, VOCAB), device="cuda:0",
                                  dtype=torch.uint8)
        self.args = (ctx, nt)
        self.queue(st)
        return pos

    def queue(self, st):
        L, nt, ctx = self.L, self.nt, self.args[0]
        rp = dc.rope_struct(self.dsv4, self.dcos, self.dsin, ROT, D - ROT, False)
        dq = self.dq.clone()
        self.q_turned = dq
        assert L.dsv4_gpu_rope_n_d(dq.data_ptr(), H * D, dq.data_ptr(), H * D, int(self.bf),
                                   self.dpos.data_ptr(), nt, H, D, ctypes.byref(rp), 0, st) == 0
        assert L.dsv4_gpu_tree_attn_d(
            self.o.data_ptr(), dq.data_ptr(), int(self.bf), nt, H, D, D, self.cache.data_ptr(),
            dc.ptr(self.ks), self.fmt, D, self.rows, self.dpages.data_ptr(), self.n_pages, PAGE,
            ctx, self.dw.data_ptr(), 0, None, ctypes.c_float(0.1), self.space.data_ptr(),
            self.space.numel(), st) == 0
        self.raw = self.o.float().view(nt, H * D) @ self.dhead.t()
        r = self.dsv4.LogitRules(hist=self.dhist.data_ptr(), n_hist=len(self.hist),
                                 draft=self.dtoks.data_ptr(), mask=self.dw.data_ptr(),
                                 repetition=1.2, frequency=0.1, presence=0.1)
        assert L.dsv4_gpu_logits_adjust_d(
            self.logits.data_ptr(), self.pick.data_ptr(), self.raw.data_ptr(), nt, VOCAB, VOCAB,
            ctypes.byref(r), self.lspace.data_ptr(), self.lspace.numel(), st) == 0


@pytest.mark.parametrize("fmt,bf", [(0, False), (1, False), (2, False), (2, True)])
def test_steps_of_a_drafted_sequence(gpu, dsv4, fmt, bf):
    """Three steps: a prompt, drafts checked, the accepted path's rows moved to
    their places, drafts again. Attention against 64 bits over the rows as the
    device holds them, logits bit for bit from its scores."""
    import torch
    nt = 9
    s = Step(dsv4, fmt, bf, 21 + fmt, nt)
    rng, st = s.rng, dc.stream()
    ctx = 300
    s.append(rng.standard_normal((ctx, D)).astype(np.float32), np.arange(ctx),
             s.row_of(np.arange(ctx)), st)
    s.hist = rng.integers(0, VOCAB, ctx).astype(np.int32)
    for _ in range(3):
        w = dc.words(rng, nt)
        toks = rng.integers(0, VOCAB, nt).astype(np.int32)
        q = rng.standard_normal((nt, H, D)).astype(np.float32)
        kv = rng.standard_normal((nt, D)).astype(np.float32)
        pos = s.verify(q, kv, ctx, w, toks, st)
        torch.cuda.synchronize()
        held = dc.cache_values(s.cache, fmt, s.ks)[s.row_of(np.arange(ctx + nt))]
        turned, slack = dc.rotate(kv[:, None, :], s.cos, s.sin, pos, D - ROT, ROT, False)
        near = 2.0 ** -4 if fmt == 2 else dc.U16 if fmt == 1 else 0
        low = 2.0 ** -10 * dc.row_scales(turned[:, 0])[:, None] if fmt == 2 else 0
        assert (np.abs(held[ctx:] - turned[:, 0]) <= slack[:, 0] + np.maximum(
            near * (np.abs(turned[:, 0]) + slack[:, 0]), low)).all()
        qv = dc.host(s.q_turned)
        want, size = dc.attention(qv, held, dc.visible(w, nt, ctx, 0), None, np.float32(0.1), D)
        got = dc.host(s.o)
        if bf:
            assert (np.abs(got - want) <= 1.01 * dc.U16 * (np.abs(want) + size)
                    + 1e-5 * size).all()
        else:
            assert common.vec_rel_err(got, want) < 1e-5
        lw = dc.logit_rules(dc.host(s.raw), s.hist, toks, w, 1.2, 0.1, 0.1, None, None)
        assert common.bits_equal(dc.host(s.logits), lw[0])
        assert np.array_equal(s.pick.cpu().numpy(), lw[1])
        # the path of the last draft is accepted: its rows move up behind the context
        path = [t for t in range(nt) if w[nt - 1] >> t & 1]
        src = dc.dev(s.row_of(ctx + np.array(path)).astype(np.int32))
        dst = dc.dev(s.row_of(ctx + np.arange(len(path))).astype(np.int32))
        mid = torch.empty(len(path), D, device="cuda:0")
        assert s.L.dsv4_gpu_kv_read_d(mid.data_ptr(), 0, D, s.cache.data_ptr(), dc.ptr(s.ks),
                                      fmt, D, s.rows, src.data_ptr(), 0, len(path), D, st) == 0
        assert s.L.dsv4_gpu_kv_append_d(s.cache.data_ptr(), dc.ptr(s.ks), fmt, D, s.rows,
                                        mid.data_ptr(), 0, D, len(path), D, dst.data_ptr(), 0,
                                        None, None, st) == 0
        after = dc.cache_values(s.cache, fmt, s.ks)[s.row_of(ctx + np.arange(len(path)))]
        assert np.array_equal(after, held[ctx + np.array(path)])
        ctx += len(path)
        s.hist = np.concatenate([s.hist, toks[path]])


@pytest.mark.parametrize("fmt,bf", [(1, False), (2, True)])
def test_captured_and_replayed(gpu, dsv4, fmt, bf):
    """A step captured into a graph, replayed between eager steps of another
    sequence: every replay has the eager bits, also with new inputs."""
    import torch
    a, b = Step(dsv4, fmt, bf, 5, 7), Step(dsv4, fmt, bf, 6, 7)
    side = torch.cuda.Stream()
    for s in (a, b):
        s.hist = s.rng.integers(0, VOCAB, 50).astype(np.int32)
        s.append(s.rng.standard_normal((400, D)).astype(np.float32), np.arange(400),
                 s.row_of(np.arange(400)), dc.stream())

    def inputs(s):
        return (s.rng.standard_normal((7, H, D)).astype(np.float32),
                s.rng.standard_normal((7, D)).astype(np.float32))
    w = dc.words(a.rng, 7)
    toks = a.rng.integers(0, VOCAB, 7).astype(np.int32)
    q, kv = inputs(a)
    a.verify(q, kv, 400, w, toks, dc.stream())
    torch.cuda.synchronize()
    want = (dc.host(a.o), dc.host(a.logits), a.pick.cpu().numpy())
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.queue(side.cuda_stream)                # warm up torch's product on this stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a.queue(side.cuda_stream)
    for k in range(4):
        a.o.zero_(), a.logits.zero_(), a.pick.zero_()
        if k == 2:                               # new queries in the captured buffer
            q2, _ = inputs(a)
            a.dq.copy_(dc.to_fmt(q2, bf))
        g.replay()
        bq, bkv = inputs(b)
        b.verify(bq, bkv, 400, w, toks, dc.stream())
        torch.cuda.synchronize()
        got = (dc.host(a.o), dc.host(a.logits), a.pick.cpu().numpy())
        if k == 2:
            a.queue(dc.stream())
            torch.cuda.synchronize()
            want = (dc.host(a.o), dc.host(a.logits), a.pick.cpu().numpy())
        assert common.bits_equal(got[0], want[0]) and np.array_equal(got[2], want[2])
        assert common.vec_rel_err(got[1], want[1]) < 1e-5   # the library's product between


def test_two_streams_at_once(gpu, dsv4):
    """Calls queued on two streams, each with its own workspace, have the bits
    that each has alone."""
    import torch
    streams = [torch.cuda.Stream() for _ in range(2)]
    rng = np.random.default_rng(1)
    jobs = []
    for k, (nt, h, dqk, dv, ctx, fmt) in enumerate([(4, 16, 576, 512, 6000, 1),
                                                    (7, 8, 512, 512, 3000, 2)]):
        v, s = dc.stored(rng.standard_normal((ctx + nt, dqk)), fmt)
        cache, ks = dc.cache_of(v, fmt, scales=s)
        q = dc.dev(rng.standard_normal((nt, h, dqk)).astype(np.float32))
        n = dsv4.lib().dsv4_gpu_tree_attn_scratch_bytes(0, nt, h, dqk, dv, fmt, ctx, 0)
        space = torch.zeros(max(16, n), device="cuda:0", dtype=torch.uint8)
        x = dc.dev(rng.standard_normal((nt, 20000)).astype(np.float32))
        lspace = torch.zeros(dsv4.lib().dsv4_gpu_logits_scratch_bytes(nt, 20000),
                             device="cuda:0", dtype=torch.uint8)
        jobs.append((q, cache, ks, fmt, ctx + nt, dqk, dv, ctx, space, x, lspace))

    def go(j, st):
        q, cache, ks, fmt, rows, dqk, dv, ctx, space, x, lspace = j
        rc, o = dc.tree(dsv4, q, False, cache, ks, fmt, rows, dqk, dv, ctx, scale=0.05,
                        space=space, st=st)
        assert rc == 0
        pick = torch.zeros(x.shape[0], device="cuda:0", dtype=torch.int32)
        y = torch.empty_like(x)
        r = dsv4.LogitRules(repetition=1.0)
        assert dsv4.lib().dsv4_gpu_logits_adjust_d(
            y.data_ptr(), pick.data_ptr(), x.data_ptr(), x.shape[0], 20000, 20000,
            ctypes.byref(r), lspace.data_ptr(), lspace.numel(), st) == 0
        return o, pick

    alone = []
    for j in jobs:
        o, p = go(j, dc.stream())
        torch.cuda.synchronize()
        alone.append((dc.host(o), p.cpu().numpy()))
    got = []
    for _ in range(5):
        for j, st in zip(jobs, streams):
            with torch.cuda.stream(st):
                got.append(go(j, st.cuda_stream))
    torch.cuda.synchronize()
    for k, (o, p) in enumerate(got):
        assert common.bits_equal(dc.host(o), alone[k % 2][0])
        assert np.array_equal(p.cpu().numpy(), alone[k % 2][1])
