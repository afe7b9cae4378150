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
