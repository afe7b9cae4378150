"""The operators on batches of requests as a serving program runs them: tables,
rotated rows into the pages, one plan, two layers' attention, logits under each
request's rules, sampling, the next lengths; requests that come, wait, go on with
drafts and end. Eagerly and as one captured graph whose lengths lie on the device."""
import ctypes

import numpy as np
import pytest

import common
import draft_common as dc
import reqs_common as rc

pytestmark = pytest.mark.gpu

H, D, DV, ROT, VOCAB, LAYERS = 4, 96, 80, 32, 2003, 2


class Serve:
    """Requests over one pool of pages, two layers' caches and one step's buffers."""

    def __init__(self, dsv4, fmt, bf, seed, n_req, page, shared, max_tok, window, spare=6):
        import torch
        self.dsv4, self.L, self.fmt, self.bf = dsv4, dsv4.lib(), fmt, bf
        self.n, self.page, self.shared, self.max_tok, self.window = n_req, page, shared, max_tok, window
        rng = self.rng = np.random.default_rng(seed)
        self.have = np.where(rng.random(n_req) < 0.3, shared, shared + rng.integers(0, 300, n_req))
        self.width = -(-(shared + 700) // page)
        self.table, self.ring, self.free = rc.pool(rng, self.have, page, shared, spare, self.width)
        self.rows = (int(self.table.max()) + spare + 1) * page
        i32 = lambda a: dc.dev(np.asarray(a, np.int32))
        self.d = dict(len=i32(self.have), pages=i32(self.table), ring=i32(self.ring),
                      free=i32(self.free), new=i32([0] * n_req), first=i32([0] * (n_req + 1)))
        self.maps = [i32([0] * max_tok) for _ in range(3)]
        self.r = rc.reqs(dsv4, self.d["len"], self.d["pages"], self.d["first"], page, max_tok,
                         shared)
        self.cos, self.sin = dc.tables(shared + 1200, ROT)
        self.dcos, self.dsin = dc.dev(self.cos), dc.dev(self.sin)
        self.dt = torch.bfloat16 if bf else torch.float32
        self.caches, self.sinks = [], []
        for _ in range(LAYERS):
            x = rng.standard_normal((self.rows, D))
            self.caches.append(dc.cache_of(*[dc.stored(x, fmt)[0], fmt], scales=dc.stored(x, fmt)[1]))
            self.sinks.append(dc.dev(rng.standard_normal(H).astype(np.float32)))
        zeros = lambda *s, t=torch.float32: torch.zeros(*s, device="cuda:0", dtype=t)
        self.q = [zeros(max_tok, H, D, t=self.dt) for _ in range(LAYERS)]
        self.turned = [zeros(max_tok, H, D, t=self.dt) for _ in range(LAYERS)]
        self.kv = [zeros(max_tok, D) for _ in range(LAYERS)]
        self.o = [zeros(max_tok, H, DV, t=self.dt) for _ in range(LAYERS)]
        self.head = dc.dev(rng.standard_normal((H * DV, VOCAB)).astype(np.float32))
        self.raw, self.logits = zeros(n_req, VOCAB), zeros(n_req, VOCAB)
        self.bias = dc.dev(rng.standard_normal(VOCAB).astype(np.float32))
        self.allow = rng.integers(0, 2 ** 32, (n_req, (VOCAB + 31) // 32), dtype=np.uint32)
        self.dallow = dc.dev(self.allow)
        self.rule = dict(temperature=rng.uniform(0.3, 2, n_req) * (rng.random(n_req) > 0.2),
                         top_k=np.where(rng.random(n_req) < 0.5, rng.integers(1, 200, n_req), 0),
                         top_p=np.where(rng.random(n_req) < 0.6, rng.uniform(0.1, 0.99, n_req), 1),
                         min_p=np.where(rng.random(n_req) < 0.3, 0.01, 0), u=np.zeros(n_req))
        self.rule = {k: v.astype(np.int32 if k == "top_k" else np.float32)
                     for k, v in self.rule.items()}
        self.drule = {k: dc.dev(v) for k, v in self.rule.items()}
        self.pick, self.kept = (zeros(n_req, t=torch.int32) for _ in range(2))
        self.prob = zeros(n_req)
        L, space = self.L, lambda n: zeros(max(16, n), t=torch.uint8)
        self.plan = space(L.dsv4_gpu_reqs_plan_bytes(n_req, max_tok, H))
        self.aspace = space(L.dsv4_gpu_reqs_attn_scratch_bytes(int(bf), H, D, DV, fmt, n_req, max_tok))
        self.lspace = space(L.dsv4_gpu_logits_scratch_bytes(n_req, VOCAB))
        self.sspace = space(L.dsv4_gpu_sample_scratch_bytes(n_req, VOCAB))

    def inputs(self, new):
        """New tokens' queries and rows, random numbers, and what each request adds."""
        for q, kv in zip(self.q, self.kv):
            q.copy_(dc.to_fmt(self.rng.standard_normal(q.shape), self.bf))
            kv.copy_(dc.dev(self.rng.standard_normal(kv.shape).astype(np.float32)))
        self.rule["u"] = self.rng.random(self.n).astype(np.float32)
        self.drule["u"].copy_(dc.dev(self.rule["u"]))
        self.d["new"].copy_(dc.dev(np.asarray(new, np.int32)))

    def queue(self, st):
        """One step."""
        L, d, n, bf = self.L, self.d, self.n, int(self.bf)
        rows, pos, req = [m.data_ptr() for m in self.maps]
        rp = dc.rope_struct(self.dsv4, self.dcos, self.dsin, ROT, D - ROT, False)
        r, plan = ctypes.byref(self.r), (self.plan.data_ptr(), self.plan.numel())
        assert L.dsv4_gpu_reqs_tables_d(r, d["len"].data_ptr(), d["new"].data_ptr(),
                                        d["ring"].data_ptr(), len(self.ring), d["free"].data_ptr(),
                                        d["free"].data_ptr(), rows, pos, req, st) == 0
        assert L.dsv4_gpu_reqs_plan_d(*plan, r, bf, H, D, DV, self.fmt, self.window, st) == 0
        for i, (cache, ks) in enumerate(self.caches):
            assert L.dsv4_gpu_kv_append_d(cache.data_ptr(), dc.ptr(ks), self.fmt, D, self.rows,
                                          self.kv[i].data_ptr(), 0, D, self.max_tok, D, rows, 0,
                                          ctypes.byref(rp), pos, st) == 0
            assert L.dsv4_gpu_rope_n_d(self.turned[i].data_ptr(), H * D, self.q[i].data_ptr(), H * D,
                                       bf, pos, self.max_tok, H, D, ctypes.byref(rp), 0, st) == 0
            assert L.dsv4_gpu_reqs_attn_d(
                self.o[i].data_ptr(), self.turned[i].data_ptr(), bf, H, D, DV, cache.data_ptr(),
                dc.ptr(ks), self.fmt, D, self.rows, r, *plan, self.window, self.sinks[i].data_ptr(),
                ctypes.c_float(0.1), self.aspace.data_ptr(), self.aspace.numel(), st) == 0
        last = (d["first"][1:] - 1).clamp(min=0).long()
        self.raw.copy_(self.o[-1].float().view(self.max_tok, H * DV)[last] @ self.head)
        lr = self.dsv4.LogitRules(bias=self.bias.data_ptr(), allow=self.dallow.data_ptr(),
                                  allow_stride=self.allow.shape[1], repetition=1.0)
        assert L.dsv4_gpu_logits_adjust_d(self.logits.data_ptr(), None, self.raw.data_ptr(), n,
                                          VOCAB, VOCAB, ctypes.byref(lr), self.lspace.data_ptr(),
                                          self.lspace.numel(), st) == 0
        rules = self.dsv4.Sampling(**{k: v.data_ptr() for k, v in self.drule.items()})
        assert L.dsv4_gpu_sample_d(self.pick.data_ptr(), self.prob.data_ptr(), self.kept.data_ptr(),
                                   self.logits.data_ptr(), 0, n, VOCAB, VOCAB, ctypes.byref(rules),
                                   self.sspace.data_ptr(), self.sspace.numel(), st) == 0

    def check(self, new):
        """The step's results against the definitions, and the state taken over."""
        want = rc.schedule(self.have, new, self.table, self.ring, self.free, self.page,
                           self.shared, self.max_tok)
        for k in ("len", "pages", "ring", "free", "first"):
            assert np.array_equal(self.d[k].cpu().numpy().reshape(-1), np.ravel(want[k])), k
        for m, k in zip(self.maps, ("rows", "pos", "req")):
            assert np.array_equal(m.cpu().numpy(), want[k]), k
        first, length, table = want["first"], want["len"], want["pages"]
        T = first[-1]
        at, pos = np.array(want["rows"][:T], int), np.array(want["pos"][:T], int)
        assert (at >= 0).all()
        for i, (cache, ks) in enumerate(self.caches):
            held = dc.cache_values(cache, self.fmt, ks)
            x = dc.host(self.kv[i])[:T, None, :]
            turned, slack = dc.rotate(x, self.cos, self.sin, pos, D - ROT, ROT, False)
            near = (0, dc.U16, 2.0 ** -4)[self.fmt]
            low = 2.0 ** -10 * dc.row_scales(turned[:, 0])[:, None] if self.fmt == 2 else 0
            assert (np.abs(held[at] - turned[:, 0]) <= slack[:, 0] + np.maximum(
                near * (np.abs(turned[:, 0]) + slack[:, 0]), low)).all()
            q, got = dc.host(self.turned[i]), dc.host(self.o[i])
            for b in range(self.n):
                f0, f1, n = first[b], first[b + 1], length[b]
                if f0 == f1:
                    continue
                p = np.arange(n)
                rows = held[table[b, p // self.page].astype(int) * self.page + p % self.page]
                own = np.arange(n - (f1 - f0), n)[:, None]
                see = (p[None] <= own) & ((own - p[None] < self.window) if self.window else True)
                o, size = dc.attention(q[f0:f1], rows, see, self.sinks[i].cpu().numpy(),
                                       np.float32(0.1), DV)
                if self.bf:
                    assert (np.abs(got[f0:f1] - o) <= 1.01 * dc.U16 * (np.abs(o) + size)
                            + 1e-5 * size).all(), b
                else:
                    assert common.vec_rel_err(got[f0:f1], o) < 1e-5, b
        bits = np.unpackbits(self.allow.view(np.uint8), axis=1, bitorder="little")[:, :VOCAB] > 0
        with np.errstate(invalid="ignore"):
            lw = dc.logit_rules(dc.host(self.raw), [], None, None, 1.0, 0, 0,
                                self.bias.cpu().numpy(), bits)
        x, pick = dc.host(self.logits), self.pick.cpu().numpy()
        kept, prob = self.kept.cpu().numpy(), dc.host(self.prob)
        for b in range(self.n):
            if first[b] == first[b + 1]:
                continue
            assert common.bits_equal(x[b], lw[0][b])
            s = rc.sample(x[b], *[self.rule[k][b] for k in ("temperature", "top_k", "top_p", "min_p",
                                                            "u")])
            assert (pick[b], kept[b]) == (s[0], s[2]) and bits[b, pick[b]]
            assert abs(prob[b] - s[1]) <= s[1] * (2.0 ** -24 + 2.0 ** -39)
        served = [int(length[b] - self.have[b]) for b in range(self.n)]
        self.have, self.table = np.array(length), table
        self.ring, self.free = want["ring"], want["free"]
        return served

    def next(self, steps):
        """What the requests ask for next: tokens, pieces of prompts, drafts, nothing, or
        their end; a request that ended begins again behind the shared positions."""
        new = self.rng.choice([1, 1, 1, 1, 3, 0, -1, 40], self.n).astype(np.int32)
        new[self.have + new > self.width * self.page] = -1
        return new

    def begin(self):
        """The host's part: ended requests are new ones that have the shared positions."""
        gone = self.have == 0
        if gone.any() and self.shared % self.page == 0:
            self.have = np.where(gone, self.shared, self.have)
            own = self.shared // self.page
            whole = self.table[~gone][0, :own] if (~gone).any() else self.table[0, :own]
            self.table[gone, :own] = whole
            self.d["len"].copy_(dc.dev(self.have.astype(np.int32)))
            self.d["pages"].copy_(dc.dev(self.table))


CASES = [  # fmt, bf16 q, requests, page, shared, tokens of a step, window
    (1, True, 12, 16, 128, 90, 0),
    (2, False, 7, 32, 0, 60, 0),
    (0, False, 20, 7, 70, 64, 50),
    (2, True, 30, 64, 512, 200, 0),
    (1, False, 1, 16, 0, 41, 0),
]


@pytest.mark.parametrize("case", CASES)
def test_steps_of_a_batch(gpu, dsv4, case):
    import torch
    s = Serve(dsv4, *case[:2], 31, *case[2:])
    total = 0
    for k in range(6):
        s.begin()
        new = s.next(k)
        s.inputs(new)
        s.queue(dc.stream())
        torch.cuda.synchronize()
        total += sum(v for v in s.check(new) if v > 0)
    assert total > 0


@pytest.mark.parametrize("case", CASES[:4])
def test_captured_and_replayed(gpu, dsv4, case):
    """One graph serves all steps of a batch, while an eager batch steps between."""
    import torch
    a = Serve(dsv4, *case[:2], 5, *case[2:])
    b = Serve(dsv4, *CASES[1][:2], 6, *CASES[1][2:])
    side = torch.cuda.Stream()
    new = a.next(0)
    a.inputs(new)
    state = {k: v.clone() for k, v in a.d.items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.queue(side.cuda_stream)                # warm up torch's product on this stream
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            a.queue(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for k, v in state.items():
        a.d[k].copy_(v)
    for k in range(5):
        if k:
            a.begin()
            new = a.next(k)
            a.inputs(new)
        torch.cuda.synchronize()
        g.replay()
        b.begin()
        other = b.next(k)
        b.inputs(other)
        b.queue(dc.stream())
        torch.cuda.synchronize()
        a.check(new)
        b.check(other)


def test_two_graphs_of_one_workspace(gpu, dsv4):
    """Two batches' steps captured over the same plan and scratch, replayed in turn."""
    import torch
    a = Serve(dsv4, 1, True, 8, 12, 16, 128, 90, 0)
    b = Serve(dsv4, 1, True, 9, 12, 16, 128, 90, 0)
    for k in ("plan", "aspace", "lspace", "sspace"):
        setattr(b, k, getattr(a, k))
    side, graphs = torch.cuda.Stream(), []
    news = [s.next(0) for s in (a, b)]
    for s, new in zip((a, b), news):
        s.inputs(new)
        state = {k: v.clone() for k, v in s.d.items()}
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.queue(side.cuda_stream)
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                s.queue(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for k, v in state.items():
            s.d[k].copy_(v)
        graphs.append(g)
    for k in range(4):
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, new in zip((a, b), news):
            s.check(new)
        for i, s in enumerate((a, b)):
            s.begin()
            news[i] = s.next(k)
            s.inputs(news[i])


def test_two_batches_on_two_streams(gpu, dsv4):
    import torch
    s = [Serve(dsv4, 2, True, 10, 30, 64, 512, 200, 0), Serve(dsv4, 0, False, 11, 20, 7, 70, 64, 50)]
    streams = [torch.cuda.Stream() for _ in s]
    for k in range(4):
        news = []
        for v in s:
            v.begin()
            news.append(v.next(k))
            v.inputs(news[-1])
        torch.cuda.synchronize()
        for v, st in zip(s, streams):
            with torch.cuda.stream(st):
                v.queue(st.cuda_stream)
        torch.cuda.synchronize()
        for v, new in zip(s, news):
            v.check(new)
