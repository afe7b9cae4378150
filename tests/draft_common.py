"""The operators on drafted tokens (rotary positions, cache rows written and
read back, tree attention, logit rules) from their definitions in 64 bits, in
numpy, and the device-side helpers their tests share."""
import ctypes

import numpy as np

import common

U32 = 2.0 ** -24                              # half a step of f32
U16 = 2.0 ** -8                               # of bf16


def bf16(a):
    """To the nearest bf16, as f32 (NaN and infinities kept)."""
    a = np.asarray(a, np.float32)
    return np.where(np.isfinite(a), common.bf16_round(np.where(np.isfinite(a), a, 0)), a)


def tables(positions, dim, base=10000.0):
    f = base ** (-np.arange(0, dim, 2) / dim)
    a = np.arange(positions)[:, None] * f
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def rotate(x, cos, sin, pos, off, dim, halves, inverse=False):
    """x [nt][heads][hd] rotated in 64 bits, and the bound that f32's two
    products and one sum per element put on the error."""
    x = np.asarray(x, np.float64)
    out, slack = x.copy(), np.zeros_like(x)
    i = np.arange(dim // 2)
    a, b = (off + i, off + i + dim // 2) if halves else (off + 2 * i, off + 2 * i + 1)
    ok = (pos >= 0) & (pos < cos.shape[0])
    c = np.where(ok[:, None], cos.astype(np.float64)[np.where(ok, pos, 0)], np.nan)[:, None, :]
    s = np.where(ok[:, None], sin.astype(np.float64)[np.where(ok, pos, 0)], np.nan)[:, None, :]
    if inverse:
        s = -s
    with np.errstate(invalid="ignore"):
        out[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
        out[:, :, b] = x[:, :, a] * s + x[:, :, b] * c
        size = [np.abs(x[:, :, a] * c) + np.abs(x[:, :, b] * s),
                np.abs(x[:, :, a] * s) + np.abs(x[:, :, b] * c)]
    # |fl(fl(p) + fl(q)) - (p + q)| <= u (|p| + |q|) + u |p + q| (1 + u)
    slack[:, :, a], slack[:, :, b] = 2.01 * U32 * size[0], 2.01 * U32 * size[1]
    return out, slack


def e4m3_round(v):
    """The e4m3 value nearest to v (|v| <= 448), ties to even."""
    v = np.asarray(v, np.float64)
    e = np.clip(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -20))), -6, 8)
    step = np.exp2(e - 3)
    return np.rint(v / step) * step


def row_scales(x):
    """The least power of two, 2^-126 at least, that brings each row's largest
    finite magnitude to 448 or less; 1 for a row of zeros."""
    top = np.where(np.isfinite(x), np.abs(x), 0).max(1).astype(np.float64)
    m, e = np.frexp(top / 448.0)              # top / 448 = m 2^e, m in [1/2, 1)
    s = np.exp2(np.maximum(np.where(m == 0.5, e - 1, e), -126).astype(np.float64))
    return np.where(top == 0, 1.0, s)


def stored(x, fmt):
    """(values, scales or None) of rows x as a cache format holds them."""
    x = np.asarray(x, np.float32)
    if fmt == 0:
        return x.astype(np.float64), None
    if fmt == 1:
        return bf16(x).astype(np.float64), None
    s = row_scales(x)
    with np.errstate(invalid="ignore"):
        v = np.where(np.isfinite(x), e4m3_round(np.where(np.isfinite(x), x, 0) / s[:, None]),
                     np.nan) * s[:, None]
    return v, s


def words(rng, nt):
    """A drafted tree's visibility: each parent one of the four before."""
    w = []
    for t in range(nt):
        p = t - 1 - int(rng.integers(0, 4))
        w.append((w[p] if p >= 0 else 0) | 1 << t)
    return w


def visible(words_, nt, ctx, window):
    """[nt][ctx + nt]: the positions each token sees."""
    if words_ is None:
        words_ = [(2 << t) - 1 for t in range(nt)]
    full = (1 << nt) - 1
    place = [ctx + bin(words_[t] & full & ~(1 << t)).count("1") for t in range(nt)]
    see = np.zeros((nt, ctx + nt), bool)
    for t in range(nt):
        see[t, max(0, place[t] - window + 1) if window else 0:ctx] = True
        for j in range(nt):
            see[t, ctx + j] = words_[t] >> j & 1 and not (
                window and place[t] - place[j] >= window)
    return see


def attention(q, rows, see, sink, scale, dv):
    """(o, sum of |weight * value|) of q [nt][h][dqk] over rows [n][dqk] in 64
    bits, each token over the rows it sees."""
    nt, h, _ = q.shape
    o, size = np.zeros((nt, h, dv)), np.zeros((nt, h, dv))
    for t in range(nt):
        r = rows[see[t]].astype(np.float64)
        if not len(r):
            continue
        s = q[t].astype(np.float64) @ r.T * scale
        m = s.max(1, keepdims=True)
        e = np.exp(s - m)
        d = e.sum(1, keepdims=True)
        if sink is not None:
            d = d + np.exp(sink.astype(np.float64)[:, None] - m)
        o[t] = e / d @ r[:, :dv]
        size[t] = e / d @ np.abs(r[:, :dv])
    return o, size


def logit_rules(x, ids, drafts, words_, rep, freq, pres, bias, allow):
    """The rules in f32, each step rounded, and the head's scan over the
    allowed tokens. allow: [rows or 1][vocab] bool, or None."""
    x = np.asarray(x, np.float32)
    nt, vocab = x.shape
    f = np.float32
    out, pick = np.empty_like(x), np.empty(nt, np.int32)
    base = np.bincount([i for i in ids if 0 <= i < vocab], minlength=vocab)
    for t in range(nt):
        n = base.copy()
        w = (2 << t) - 1 if words_ is None else words_[t]
        for j in range(nt if drafts is not None else 0):
            if w >> j & 1 and 0 <= drafts[j] < vocab:
                n[drafts[j]] += 1
        y = x[t].copy()
        hit = n > 0
        with np.errstate(invalid="ignore", over="ignore"):
            y[hit] = np.where(y[hit] > 0, y[hit] / f(rep), y[hit] * f(rep))
            y[hit] -= n[hit].astype(f) * f(freq) + f(pres)
            if bias is not None:
                y += bias
        ok = np.ones(vocab, bool) if allow is None else allow[t % allow.shape[0]]
        y[~ok] = -np.inf
        out[t] = y
        c = np.nonzero(ok)[0]
        if not len(c):
            pick[t] = -1
        elif np.isnan(y[c[0]]):
            pick[t] = c[0]
        else:
            pick[t] = c[np.nanargmax(y[c])]
    return out, pick


# ------------------------------------------------------------- device side
def dev(a):
    import torch
    a = np.ascontiguousarray(a)
    if a.dtype == np.uint64:
        a = a.view(np.int64)
    if a.dtype == np.uint32:
        a = a.view(np.int32)
    return torch.from_numpy(a).to("cuda:0")


def to_fmt(a, bf):
    """f32 values on the device as f32 or bf16."""
    import torch
    t = dev(np.asarray(a, np.float32))
    return t.to(torch.bfloat16) if bf else t


def host(t):
    return t.float().cpu().numpy()


def ptr(t):
    return None if t is None else t.data_ptr()


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def rope_struct(dsv4, cos, sin, dim, off, halves):
    return dsv4.Rope(cos=cos.data_ptr(), sin=sin.data_ptr(), max_pos=cos.shape[0], dim=dim,
                     offset=off, layout=dsv4.ROPE_HALVES if halves else dsv4.ROPE_PAIRS)


def cache_of(values, fmt, stride=None, scales=None):
    """A device cache of the rows `values` (as stored() gives them), with row
    pitch `stride`, and its scales."""
    import torch
    n, d = values.shape
    stride = stride or d
    data = np.full((n, stride), 7.0)
    if fmt == 2:
        data[:, :d] = values / scales[:, None]
        t = torch.from_numpy(data).to(torch.float32).to(torch.float8_e4m3fn)
        return t.view(torch.uint8).to("cuda:0"), dev(scales.astype(np.float32))
    data[:, :d] = values
    return to_fmt(data, fmt == 1), None


def cache_values(cache, fmt, scales):
    import torch
    if fmt != 2:
        return host(cache).astype(np.float64)
    v = cache.view(torch.float8_e4m3fn).float().cpu().numpy().astype(np.float64)
    return v * scales.cpu().numpy().astype(np.float64)[:, None]


def tree(dsv4, q, bf, kv, ks, fmt, rows, dqk, dv, ctx, words_=None, window=0, pages=None,
         page=0, n_pages=None, sink=None, scale=1.0, stride=None, space=None, st=None):
    """dsv4_gpu_tree_attn_d on device tensors (q [nt][h][dqk]); (rc, o)."""
    import torch
    L = dsv4.lib()
    nt, h = q.shape[:2]
    o = torch.full((nt, h, dv), 99.0, device="cuda:0", dtype=q.dtype)
    if space is None:
        n = L.dsv4_gpu_tree_attn_scratch_bytes(int(bf), nt, h, dqk, dv, fmt, ctx, window)
        space = torch.full((max(n, 16),), 255, device="cuda:0", dtype=torch.uint8)
    if n_pages is None:
        n_pages = 0 if pages is None else pages.numel()
    rc = L.dsv4_gpu_tree_attn_d(
        o.data_ptr(), q.data_ptr(), int(bf), nt, h, dqk, dv, kv.data_ptr(), ptr(ks), fmt,
        stride or dqk, rows, ptr(pages), n_pages, page, ctx, ptr(words_), window, ptr(sink),
        ctypes.c_float(scale), space.data_ptr(), space.numel(), stream() if st is None else st)
    return rc, o
