"""The operators on batches of requests (page tables and row maps, attention of
all requests, sampling) from their definitions, in Python's integers and numpy's
64 bits, and the device-side helpers their tests share."""
import ctypes

import numpy as np

import draft_common as dc


# ------------------------------------------------------------------ tables
def schedule(have, new, table, ring, free, page, shared, max_tok):
    """A step's tables, request by request. table [n_req][max_pages], ring [cap];
    returns a dict of what the call writes."""
    have, new = [int(v) for v in have], [int(v) for v in new]
    table, ring, cap = table.copy(), ring.copy(), len(ring)
    head, count = free
    room = table.shape[1] * page
    own = shared // page
    first, length, taken, back = [0], [], 0, []
    rows, pos, req = [], [], []
    asked = tokens = 0
    for i, (L, n) in enumerate(zip(have, new)):
        fits = n > 0 and 0 <= L <= room and n <= room - L
        need = -(-(L + n) // page) - -(-L // page) if fits else 0
        asked += need
        paged = fits and (need == 0 or asked <= count)
        tokens += n if paged else 0
        served = paged and tokens <= max_tok
        if served:
            for e in range(-(-L // page), -(-(L + n) // page)):
                table[i, e] = ring[(head + taken) % cap]
                taken += 1
            for p in range(L, L + n):
                r = int(table[i, p // page]) * page + p % page
                rows.append(r if table[i, p // page] >= 0 and r < 2 ** 31 - 1 else -1)
                pos.append(p)
                req.append(i)
        first.append(len(rows))
        length.append(0 if n < 0 else L + (n if served else 0))
        if n < 0:
            back += table[i, own:max(own, -(-max(0, min(L, room)) // page))].tolist()
    back = back[:cap - count]
    for j, p in enumerate(back):
        ring[(head + count + j) % cap] = p
    rest = [-1] * (max_tok - len(rows))
    return dict(first=first, len=length, pages=table, ring=ring,
                free=[(head + taken) % cap, count - taken + len(back)], rows=rows + rest,
                pos=pos + rest, req=req + rest)


def pool(rng, lens, page, shared, spare, width):
    """(table, ring, free) of requests with lens positions in use: random pages, the
    shared ones the same in every request, and `spare` free ones in a ring that may
    wrap."""
    own = shared // page
    need = own + sum(max(0, -(-n // page) - own) for n in lens) + spare
    order = rng.permutation(need).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    used = own
    for i, n in enumerate(lens):
        k = -(-n // page)
        table[i, :min(own, width)] = order[:min(own, width)]
        table[i, own:k] = order[used:used + max(0, k - own)]
        used += max(0, k - own)
    cap = need + 1
    ring = np.full(cap, -5, np.int32)
    head = int(rng.integers(0, cap))
    ring[(head + np.arange(need - used)) % cap] = order[used:]
    return table, ring, [head, need - used]


def reqs(dsv4, length, pages, first, page, max_tok, prefix=0):
    """The call's struct of device tensors."""
    return dsv4.Reqs(len=dc.ptr(length), pages=dc.ptr(pages), first=dc.ptr(first),
                     n_req=pages.shape[0], max_pages=pages.shape[1], page_rows=page,
                     max_tok=max_tok, n_prefix=prefix)


# ---------------------------------------------------------------- sampling
def sample(x, temperature, top_k, top_p, min_p, u):
    """(pick, prob, kept) of one row of logits (f32 values), in 64 bits."""
    x = np.asarray(x, np.float64)
    ids = np.nonzero(x > -np.inf)[0]
    if not len(ids):
        return -1, 0.0, 0
    order = ids[np.argsort(-x[ids], kind="stable")]
    v = x[order]
    if not temperature > 0:
        return int(order[0]), 1.0, 1
    if v[0] == np.inf:
        w = (v == np.inf).astype(np.float64)
    else:
        w = np.exp((v - v[0]) / np.float64(temperature))
    n = len(v) if top_k <= 0 else min(len(v), top_k)
    c = np.cumsum(w[:n])
    if top_p < 1:
        n = 1 + int((c[:-1] < max(0.0, float(top_p)) * c[-1]).sum())
    if min_p > 0:
        n = max(1, min(n, int((w >= min(1.0, float(min_p))).sum())))
    c = c[:n]
    u = 0.0 if np.isnan(u) or u < 0 else float(u)
    at = int((w[:n] > 0).sum()) - 1 if u >= 1 else int((c <= u * c[-1]).sum())
    return int(order[at]), w[at] / c[-1], n


def run_sample(dsv4, x, bf=False, u=None, temperature=None, top_k=None, top_p=None, min_p=None,
               stride=None, shift=0, prob=True, kept=True, space=None, st=None):
    """dsv4_gpu_sample_d of rows x (f32 values); (pick, prob, kept) on the host, with
    what lies around every buffer checked."""
    import torch
    L = dsv4.lib()
    n, vocab = x.shape
    stride = stride or vocab
    dt = torch.bfloat16 if bf else torch.float32
    buf = torch.full((shift + n * stride + 8,), 50.0, device="cuda:0", dtype=dt)
    buf[shift:shift + n * stride].view(n, stride)[:, :vocab] = dc.dev(np.asarray(x, np.float32)).to(dt)
    keep = [None if v is None else dc.dev(np.asarray(v, t)) for v, t in (
        (temperature, np.float32), (top_k, np.int32), (top_p, np.float32), (min_p, np.float32),
        (u, np.float32))]
    rules = dsv4.Sampling(*[dc.ptr(k) for k in keep])
    need = L.dsv4_gpu_sample_scratch_bytes(n, vocab)
    if space is None:
        space = torch.full((need + 16,), 255, device="cuda:0", dtype=torch.uint8)
    out = [torch.full((n + 1,), -7, device="cuda:0", dtype=t)
           for t in (torch.int32, torch.float32, torch.int32)]
    rc = L.dsv4_gpu_sample_d(out[0].data_ptr(), out[1].data_ptr() if prob else None,
                             out[2].data_ptr() if kept else None,
                             buf.data_ptr() + shift * buf.element_size(), int(bf), n, vocab,
                             stride, ctypes.byref(rules), space.data_ptr(), need,
                             dc.stream() if st is None else st)
    assert rc == 0
    torch.cuda.synchronize()
    assert (space[need:] == 255).all()
    got = [o.cpu().numpy() for o in out]
    assert all(g[n] == -7 for g in got)
    return [g[:n] for g in got]


# --------------------------------------------------------------- attention
class Batch:
    """Requests of lens positions, of which their last news[i] are the step's tokens,
    over a paged device cache; positions before `prefix` hold the same rows in all of
    them (whole pages are shared, the rest copied)."""

    def __init__(self, seed, lens, news, h, dqk, fmt, bf, page=16, prefix=0, scale=1.0, stride=None,
                 spare=3, room=0):
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.news = [int(v) for v in lens], [int(v) for v in news]
        self.h, self.dqk, self.fmt, self.bf, self.page, self.prefix = h, dqk, fmt, bf, page, prefix
        width = max([-(-n // page) for n in self.lens] + [1]) + 1
        own = prefix // page
        need = own + sum(max(0, -(-n // page) - own) for n in self.lens) + spare
        order = rng.permutation(need).astype(np.int32)
        t = self.table = np.full((len(self.lens), width), -1, np.int32)
        used = own
        for i, n in enumerate(self.lens):
            k = -(-n // page)
            t[i, :min(own, width)] = order[:min(own, width)]
            t[i, own:k] = order[used:used + max(0, k - own)]
            used += max(0, k - own)
        self.rows = need * page
        x = rng.standard_normal((self.rows, dqk))
        whole = [i for i, n in enumerate(self.lens) if n > prefix]
        for i, n in enumerate(self.lens):
            for p in range(own * page, min(n, prefix)):
                x[self.row(i, p)] = x[self.row(whole[0], p)] if whole else 0.25
        self.x, s = dc.stored(x, fmt)
        self.stride = stride or dqk
        self.cache, self.ks = dc.cache_of(self.x, fmt, self.stride, s)
        self.first = np.concatenate([[0], np.cumsum(self.news)]).astype(np.int32)
        self.tokens = int(self.first[-1])
        self.max_tok = self.tokens + room
        q = (rng.standard_normal((self.max_tok, h, dqk)) * scale).astype(np.float32)
        self.q = dc.bf16(q) if bf else q
        self.dq = dc.to_fmt(self.q, bf)
        self.dev = {k: dc.dev(np.asarray(v, np.int32)) for k, v in
                    dict(len=self.lens, pages=t, first=self.first).items()}

    def row(self, i, p):
        return int(self.table[i, p // self.page]) * self.page + p % self.page

    def struct(self, dsv4, **kw):
        d = self.dev
        a = dict(length=d["len"], pages=d["pages"], first=d["first"], page=self.page,
                 max_tok=self.max_tok, prefix=self.prefix)
        a.update(kw)
        return reqs(dsv4, **a)

    def buffers(self, dsv4, dv):
        import torch
        L, h, n = dsv4.lib(), self.h, len(self.lens)
        self.plan = torch.full((L.dsv4_gpu_reqs_plan_bytes(n, self.max_tok, h) + 16,), 255,
                               device="cuda:0", dtype=torch.uint8)
        self.space = torch.full((L.dsv4_gpu_reqs_attn_scratch_bytes(
            int(self.bf), h, self.dqk, dv, self.fmt, n, self.max_tok) + 16,), 255, device="cuda:0",
            dtype=torch.uint8)
        self.o = torch.full((self.max_tok + 1, h, dv), 99.0, device="cuda:0", dtype=self.dq.dtype)
        return self.o

    def make_plan(self, dsv4, dv, window=0, st=None, **kw):
        return dsv4.lib().dsv4_gpu_reqs_plan_d(
            self.plan.data_ptr(), self.plan.numel() - 16, ctypes.byref(self.struct(dsv4, **kw)),
            int(self.bf), self.h, self.dqk, dv, self.fmt, window, dc.stream() if st is None else st)

    def attend(self, dsv4, dv, window=0, sink=None, scale=1.0, st=None, **kw):
        return dsv4.lib().dsv4_gpu_reqs_attn_d(
            self.o.data_ptr(), self.dq.data_ptr(), int(self.bf), self.h, self.dqk, dv,
            self.cache.data_ptr(), dc.ptr(self.ks), self.fmt, self.stride, self.rows,
            ctypes.byref(self.struct(dsv4, **kw)), self.plan.data_ptr(), self.plan.numel() - 16,
            window, dc.ptr(sink), ctypes.c_float(scale), self.space.data_ptr(),
            self.space.numel() - 16, dc.stream() if st is None else st)

    def call(self, dsv4, dv, window=0, sink=None, scale=1.0):
        """Plan and attention; what lies behind the buffers checked."""
        import torch
        self.buffers(dsv4, dv)
        assert self.make_plan(dsv4, dv, window) == 0
        assert self.attend(dsv4, dv, window, sink, scale) == 0
        torch.cuda.synchronize()
        assert (self.plan[-16:] == 255).all() and (self.space[-16:] == 255).all()
        got = dc.host(self.o)
        assert (got[self.tokens:] == 99).all()
        return got[:self.tokens]

    def sees(self, i, window):
        """[tokens][positions] of request i."""
        n, k = self.lens[i], self.news[i]
        p, r = np.arange(n - k, n)[:, None], np.arange(n)[None, :]
        return (r <= p) & ((p - r < window) if window else True)

    def want(self, dv, window=0, sink=None, scale=1.0, x=None, gone=None):
        """(o, sum of |weight value|) in 64 bits; gone: cache rows that are not there."""
        x = self.x if x is None else x
        o, size = np.zeros((self.tokens, self.h, dv)), np.zeros((self.tokens, self.h, dv))
        for i, n in enumerate(self.lens):
            f0, f1 = self.first[i], self.first[i + 1]
            if f0 == f1:
                continue
            p = np.arange(n)
            page = self.table[i, p // self.page].astype(np.int64)
            at = page * self.page + p % self.page
            see = self.sees(i, window)
            there = (page >= 0) & (at < self.rows)
            see &= there[None, :]
            if gone is not None:
                see &= ~gone[np.where(there, at, 0)][None, :]
            o[f0:f1], size[f0:f1] = dc.attention(self.q[f0:f1], x[np.where(there, at, 0)], see, sink,
                                                 np.float32(scale), dv)
        return o, size
