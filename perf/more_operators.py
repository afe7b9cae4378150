"""The calls of a step that serves a batch of requests over a paged latent KV
cache, as cases that can be timed and checked: page tables and row maps from
the requests' lengths, attention of every request's tokens over its pages with
a shared prefix computed once for all, and sampling with temperature, top-k,
top-p and min-p from given random numbers.

  own                  False: plain torch; True: the backend's entry points
  listed()             the named cases
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  inputs and buffers, on the GPU
  run(state)           one pass; returns its outputs
  work(case)           bytes and operations a pass cannot do without
  exact(case, seed)    the outputs in 64 bits

Activations are N(0, 1), cache rows N(0, 1) in their stored format, logits
N(0, 2) with some tens of likely tokens far above the rest.
"""
import ctypes
import importlib.util
import math
import os
import random
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
KV = {"f32": 0, "bf16": 1, "fp8": 2}          # DSV4_GPU_KV_*
WF = {"f32": 0, "bf16": 1}                    # DSV4_WF32, DSV4_WBF16
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2, "fp8": 1}
_pkg = None


def backend():
    """The package's binding, its library loaded and the device up."""
    global _pkg
    if _pkg is None:
        if "dsv4_amd" not in sys.modules:
            spec = importlib.util.spec_from_file_location(
                "dsv4_amd", os.path.join(ROOT, "deepseek-v4-in-c_amd", "__init__.py"))
            mod = importlib.util.module_from_spec(spec)
            sys.modules["dsv4_amd"] = mod
            spec.loader.exec_module(mod)
        sys.modules["dsv4_amd"].init()
        _pkg = sys.modules["dsv4_amd"]
    return _pkg


# ---------------------------------------------------------------- cases
def listed():
    return [
        # A decode step of a batch: a token each, a new page now and then.
        dict(name="tables_decode_64", op="tables", n_req=64, ctx=8192, new="one", page=64,
             prefix=0, ended=2),
        # Many requests whose prompts start, next to ones that decode and end.
        dict(name="tables_prompts_1000", op="tables", n_req=1000, ctx=4096, new="prompts",
             page=16, prefix=1024, ended=100),
        # A few short requests, a token each: the smallest attention call.
        dict(name="attn_decode_8x64_1000_bf16", op="attn", n_req=8, h=64, dqk=576, dv=512,
             ctx=1000, new="one", prefix=0, kv="bf16", q="f32", window=0, page=64, sink=True),
        # A batch of chats behind one long system prompt.
        dict(name="attn_prefix_64x64_32768_bf16", op="attn", n_req=64, h=64, dqk=576, dv=512,
             ctx=2000, new="one", prefix=32768, kv="bf16", q="bf16", window=0, page=64,
             sink=True),
        # A large batch of ragged lengths that share nothing, FP8 cache.
        dict(name="attn_ragged_128x128_32768_fp8", op="attn", n_req=128, h=128, dqk=512, dv=512,
             ctx=32768, new="one", prefix=0, kv="fp8", q="bf16", window=0, page=64, sink=True),
        # Drafted tokens of every request behind a shared prefix, f32 queries.
        dict(name="attn_drafts_24x64_4096_fp8", op="attn", n_req=24, h=64, dqk=576, dv=512,
             ctx=500, new="drafts", prefix=4096, kv="fp8", q="f32", window=0, page=64,
             sink=False),
        # Odd sizes: few heads, narrow rows, small pages, a sliding window.
        dict(name="attn_window_33x5_777_f32", op="attn", n_req=33, h=5, dqk=72, dv=40, ctx=777,
             new="drafts", prefix=50, kv="f32", q="f32", window=128, page=16, sink=False),
        # Pieces of prompts beside requests that decode.
        dict(name="attn_prompts_16x64_4096_bf16", op="attn", n_req=16, h=64, dqk=576, dv=512,
             ctx=4096, new="prompts", prefix=0, kv="bf16", q="bf16", window=0, page=64,
             sink=True),
        # One request's token: latency.
        dict(name="sample_1x129280_p", op="sample", n=1, vocab=129280, fmt="f32", rules="p"),
        # A batch with the usual limits.
        dict(name="sample_64x129280_kp", op="sample", n=64, vocab=129280, fmt="f32",
             rules="kp"),
        # A large batch of bf16 logits, no limit but a floor on the probability.
        dict(name="sample_256x129280_bf16", op="sample", n=256, vocab=129280, fmt="bf16",
             rules="floor"),
        # Each row with rules of its own, greedy ones among them; an odd vocabulary.
        dict(name="sample_37x32003_mixed", op="sample", n=37, vocab=32003, fmt="f32",
             rules="mixed"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "attn", "attn", "attn", "attn", "sample", "sample", "sample"])
    if op == "tables":
        return dict(op=op, n_req=_log(rng, 1, 1000), ctx=_log(rng, 1, 8192),
                    new=rng.choice(["one", "drafts", "prompts"]),
                    page=rng.choice([1, 16, 64, rng.randint(2, 100)]),
                    prefix=rng.choice([0, rng.randint(1, 2000)]), ended=rng.randint(0, 20))
    if op == "sample":
        vocab = rng.choice([129280, _log(rng, 1000, 200000)])
        return dict(op=op, n=min(_log(rng, 1, 256), (1 << 25) // vocab), vocab=vocab,
                    fmt=rng.choice(["f32", "f32", "bf16"]),
                    rules=rng.choice(["none", "p", "kp", "floor", "mixed"]))
    dqk, dv = rng.choice([(576, 512), (512, 512), (192, 128), (128, 128),
                          (rng.randint(20, 576),) * 2])
    case = dict(op=op, n_req=_log(rng, 1, 128), h=rng.choice([16, 32, 64, 128, rng.randint(1, 40)]),
                dqk=dqk, dv=min(dv, 512), ctx=_log(rng, 1, 32768),
                new=rng.choice(["one", "one", "drafts", "prompts"]),
                prefix=rng.choice([0, 0, _log(rng, 32, 32768)]),
                kv=rng.choice(["f32", "bf16", "bf16", "fp8", "fp8"]), q=rng.choice(["f32", "bf16"]),
                window=rng.choice([0, 0, 0, 128]), page=rng.choice([16, 64, rng.randint(1, 100)]),
                sink=rng.random() < 0.6)
    while work(case)["flops"] > 1.0e12 or sum(n for n, _ in _lengths(case)) > 2000000:
        case["ctx"], case["n_req"] = max(1, case["ctx"] // 2), max(1, case["n_req"] * 3 // 4)
        if case["prefix"] > 32:
            case["prefix"] //= 2
    return case


def _lengths(case):
    """(length with the step's tokens, the step's tokens) of every request, a
    part of the case: own lengths are spread over their logarithm. A prompt's
    piece takes up to 700 tokens, for one request of five or so."""
    rng = random.Random(case["n_req"] * 7919 + case["ctx"] * 31 + case["prefix"])
    out = []
    for i in range(case["n_req"]):
        before = case["prefix"] + _log(rng, 1, case["ctx"]) - 1
        if case["new"] == "one":
            n = 1
        elif case["new"] == "drafts" or rng.random() < 0.8:
            n = rng.randint(1, 8) if case["new"] == "drafts" else 1
        else:
            n = _log(rng, 9, 700)
        out.append((before + n, n))
    return out


# ------------------------------------------------------------- the inputs
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1009 + salt)
    return g


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale


def _ints(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def _cache(g, rows, dim, fmt):
    """rows of N(0, 1) in a cache format: (stored data, row scales or None).
    FP8: e4m3 codes under the row's power-of-two scale."""
    v = _normal(g, rows, dim)
    if fmt != "fp8":
        return v.to(DT[fmt]), None
    s = torch.exp2(torch.ceil(torch.log2(v.abs().amax(1) / 448.0)))
    return (v / s[:, None]).to(torch.float8_e4m3fn).view(torch.uint8), s


def _prepare_tables(s, case, g, rng):
    """Page tables of the positions in use, the free pages in a ring, and what
    the step brings; pages before the end of the prefix are all requests'."""
    P, n_req, shared = case["page"], case["n_req"], case["prefix"] // case["page"]
    lens = _lengths(case)
    ended = set(rng.sample(range(n_req), min(case["ended"], n_req // 2)))
    width = max(-(-n // P) for n, _ in lens) + 2
    need = shared + sum(-(-n // P) - shared for n, _ in lens) + 64
    order = torch.randperm(need, generator=g, device=DEV).tolist()
    head, used = order[:shared], shared
    table = np.full((n_req, width), -1, np.int32)
    for i, (n, new) in enumerate(lens):
        have = -(-(n - new) // P)
        table[i, :shared] = head
        table[i, shared:have] = order[used:used + max(0, have - shared)]
        used += max(0, have - shared)
    ring = np.full(need, -1, np.int32)
    at = rng.randrange(need)
    free = order[used:]
    ring[(at + np.arange(len(free))) % need] = free
    s["in_use"] = _ints([n - new for n, new in lens])
    s["new"] = _ints([-1 if i in ended else new for i, (_, new) in enumerate(lens)])
    s["table"], s["ring"], s["free"] = _ints(table), _ints(ring), _ints([at, len(free)])
    s["max_tok"] = sum(new for _, new in lens)
    s["len"], s["free_out"] = torch.empty_like(s["in_use"]), torch.empty_like(s["free"])
    s["first"] = torch.empty(n_req + 1, device=DEV, dtype=torch.int32)
    s["rows"], s["pos"], s["req"] = (torch.empty(s["max_tok"], device=DEV, dtype=torch.int32)
                                     for _ in range(3))


def _prepare_attn(s, case, g):
    P, n_req, prefix = case["page"], case["n_req"], case["prefix"]
    lens = _lengths(case)
    shared = prefix // P
    width = max(-(-n // P) for n, _ in lens)
    n_pages = shared + sum(-(-n // P) - shared for n, _ in lens)
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((n_req, width), -1, device=DEV, dtype=torch.int32)
    table[:, :shared] = order[:shared]
    used = shared
    for i, (n, _) in enumerate(lens):
        k = -(-n // P) - shared
        table[i, shared:shared + k] = order[used:used + k]
        used += k
    s["kv_rows"] = n_pages * P
    s["cache"], s["scales"] = _cache(g, s["kv_rows"], case["dqk"], case["kv"])
    if prefix % P:                            # the prefix's end lies in pages of their own
        at = torch.arange(prefix // P * P, prefix, device=DEV) % P
        for i in range(1, n_req):
            src = int(table[0, shared]) * P + at
            dst = int(table[i, shared]) * P + at
            s["cache"][dst] = s["cache"][src]
            if s["scales"] is not None:
                s["scales"][dst] = s["scales"][src]
    s["lengths"] = lens                       # which the program that schedules them has
    s["table"], s["len"] = table, _ints([n for n, _ in lens])
    s["first"] = _ints([0] + np.cumsum([n for _, n in lens]).tolist())
    tokens = sum(n for _, n in lens)
    s["max_tok"] = tokens
    s["qx"] = _normal(g, tokens, case["h"], case["dqk"], scale=1.5).to(DT[case["q"]])
    s["sinks"] = _normal(g, case["h"]) if case["sink"] else None
    s["out"] = torch.empty(tokens, case["h"], case["dv"], device=DEV, dtype=DT[case["q"]])
    s["scale"] = 1.0 / math.sqrt(case["dqk"])


def _prepare_sample(s, case, g, rng):
    n, vocab = case["n"], case["vocab"]
    x = _normal(g, n, vocab, scale=2.0)
    k = min(vocab, 48)                        # the likely tokens
    at = torch.randint(0, vocab, (n, k), generator=g, device=DEV)
    x.scatter_add_(1, at, 4.0 + 4.0 * _normal(g, n, k).abs())
    s["x"] = x.to(DT[case["fmt"]])
    rules = case["rules"]
    t, tk, tp, mp = [], [], [], []
    for _ in range(n):
        r = rng.choice(["none", "p", "kp", "floor", "greedy"]) if rules == "mixed" else rules
        t.append({"greedy": 0.0, "none": 1.0}.get(r, round(rng.uniform(0.5, 1.3), 3)))
        tk.append(rng.choice([20, 50, 50, 64, 200]) if r == "kp" else 0)
        tp.append(round(rng.uniform(0.8, 0.99), 3) if r in ("p", "kp") else 1.0)
        mp.append(round(rng.uniform(0.01, 0.1), 3) if r == "floor" else 0.0)
    for name, v in (("temperature", t), ("top_p", tp), ("min_p", mp)):
        s[name] = torch.tensor(v, device=DEV, dtype=torch.float32)
    s["top_k"] = _ints(tk)
    s["u"] = torch.rand(n, generator=g, device=DEV, dtype=torch.float32)
    s["pick"], s["kept"] = (torch.empty(n, device=DEV, dtype=torch.int32) for _ in range(2))
    s["prob"] = torch.empty(n, device=DEV)


def prepare(case, seed):
    g, rng = _gen(seed, 5), random.Random(seed)
    s = dict(case)
    if case["op"] == "tables":
        _prepare_tables(s, case, g, rng)
    elif case["op"] == "attn":
        _prepare_attn(s, case, g)
    else:
        _prepare_sample(s, case, g, rng)
    return s


# ------------------------------------------------------------ the plain forms
def _plain_tables(s):
    P, width, cap = s["page"], s["table"].shape[1], s["ring"].shape[0]
    have, new = s["in_use"].long(), s["new"].long()
    up = lambda n: (n + P - 1) // P
    ok = (new > 0) & (have + new <= width * P)
    need = torch.where(ok, up(have + new) - up(have), 0)
    ok &= (need == 0) | (need.cumsum(0) <= s["free"][1])
    ok &= torch.where(ok, new, 0).cumsum(0) <= s["max_tok"]
    tok, need = torch.where(ok, new, 0), torch.where(ok, need, 0)
    s["first"][0] = 0
    s["first"][1:] = tok.cumsum(0)
    s["len"].copy_(torch.where(new < 0, 0, have + tok))
    # the taken pages, in order of request and entry
    head, count = s["free"][0].long(), s["free"][1].long()
    who = torch.repeat_interleave(torch.arange(s["n_req"], device=DEV), need)
    k = torch.arange(who.shape[0], device=DEV)
    entry = up(have)[who] + k - (need.cumsum(0) - need)[who]
    s["table"][who, entry] = s["ring"][(head + k) % cap]
    # the ended requests' own pages go behind the others
    back = torch.where(new < 0, (up(have) - s["prefix"] // P).clamp(min=0), 0)
    who = torch.repeat_interleave(torch.arange(s["n_req"], device=DEV), back)
    j = torch.arange(who.shape[0], device=DEV)
    entry = s["prefix"] // P + j - (back.cumsum(0) - back)[who]
    s["ring"][(head + count + j) % cap] = s["table"][who, entry]
    taken = k.shape[0]
    s["free_out"][0] = (head + taken) % cap
    s["free_out"][1] = count - taken + j.shape[0]
    # every token's row, position and request
    req = torch.repeat_interleave(torch.arange(s["n_req"], device=DEV), tok)
    t = torch.arange(req.shape[0], device=DEV)
    pos = have[req] + t - s["first"].long()[req]
    for name, v in (("rows", s["table"][req, pos // P].long() * P + pos % P), ("pos", pos),
                    ("req", req)):
        s[name].fill_(-1)
        s[name][:t.shape[0]] = v.to(torch.int32)
    return _table_outputs(s)


def _table_outputs(s):
    return {k: s[k] for k in ("first", "len", "table", "ring", "free_out", "rows", "pos", "req")}


def _plain_attn(s):
    P, h, t0 = s["page"], s["h"], 0
    for i, (n, new) in enumerate(s["lengths"]):
        lo = max(0, n - new + 1 - s["window"]) if s["window"] else 0
        at = torch.arange(lo, n, device=DEV)
        rows = s["table"][i].long()[at // P] * P + at % P
        k = s["cache"][rows]
        k = k.float() if s["scales"] is None else \
            k.view(torch.float8_e4m3fn).float() * s["scales"][rows][:, None]
        q = s["qx"][t0:t0 + new].float().view(new * h, -1)
        p = (q @ k.t()).view(new, h, -1) * s["scale"]
        pos = torch.arange(n - new, n, device=DEV)
        hide = at[None, :] > pos[:, None]
        if s["window"]:
            hide |= pos[:, None] - at[None, :] >= s["window"]
        p.masked_fill_(hide[:, None, :], -math.inf)
        top = p.amax(-1, keepdim=True)
        p.sub_(top).exp_()
        total = p.sum(-1)
        if s["sinks"] is not None:
            total = total + torch.exp(s["sinks"] - top[..., 0])
        o = (p.view(new * h, -1) @ k[:, :s["dv"]]).view(new, h, -1) / total[..., None]
        s["out"][t0:t0 + new] = o.to(s["out"].dtype)
        t0 += new
    return s["out"]


def _plain_sample(s):
    """In 64 bits: which side of top-p's border a token lies on, and the token
    that u falls on, are differences of long sums."""
    n, vocab = s["x"].shape
    v, order = torch.sort(s["x"].float(), dim=1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    z = (v.double() - v[:, :1].double()) / torch.where(greedy, 1.0, t)
    w = torch.exp(z)
    rank = torch.arange(vocab, device=DEV)[None, :]
    top_k = s["top_k"].long()[:, None]
    limit = torch.where(greedy, 1, torch.where(top_k > 0, top_k, vocab))
    w = torch.where(rank < limit, w, 0.0)
    run = w.cumsum(1)
    before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], 1)
    top_p = s["top_p"].double()[:, None]
    keep = (top_p >= 1) | (before < top_p * run[:, -1:])
    keep &= (w >= s["min_p"].double()[:, None]) & (rank < limit)
    keep |= rank == 0
    w = torch.where(keep, w, 0.0)
    run = w.cumsum(1)
    over = run > s["u"].double()[:, None] * run[:, -1:]
    at = over.to(torch.int32).argmax(1, keepdim=True)
    s["pick"].copy_(order.gather(1, at)[:, 0])
    s["prob"].copy_((w.gather(1, at) / run[:, -1:])[:, 0])
    s["kept"].copy_(keep.sum(1))
    return s["pick"], s["prob"], s["kept"]


# ----------------------------------------------------------------- a pass
def _at(t):
    return None if t is None else t.data_ptr()


def _buffer(s, name, bytes_):
    """A workspace, which a program keeps beside its other buffers."""
    if name not in s:
        s[name] = torch.empty(max(16, bytes_()), device=DEV, dtype=torch.uint8)
    return s[name].data_ptr(), s[name].numel()


def _own(s):
    D = backend()
    L, op = D.lib(), s["op"]
    st = torch.cuda.current_stream().cuda_stream or None
    if op == "sample":
        n, vocab = s["x"].shape
        rules = D.Sampling(temperature=s["temperature"].data_ptr(), top_k=s["top_k"].data_ptr(),
                           top_p=s["top_p"].data_ptr(), min_p=s["min_p"].data_ptr(),
                           u=s["u"].data_ptr())
        space = _buffer(s, "space", lambda: L.dsv4_gpu_sample_scratch_bytes(n, vocab))
        rc = L.dsv4_gpu_sample_d(s["pick"].data_ptr(), s["prob"].data_ptr(),
                                 s["kept"].data_ptr(), s["x"].data_ptr(), WF[s["fmt"]], n, vocab,
                                 vocab, ctypes.byref(rules), *space, st)
        out = s["pick"], s["prob"], s["kept"]
    else:
        reqs = D.Reqs(len=s["len"].data_ptr(), pages=s["table"].data_ptr(),
                      first=s["first"].data_ptr(), n_req=s["n_req"], max_pages=s["table"].shape[1],
                      page_rows=s["page"], max_tok=s["max_tok"], n_prefix=s["prefix"])
    if op == "tables":
        rc = L.dsv4_gpu_reqs_tables_d(ctypes.byref(reqs), s["in_use"].data_ptr(),
                                      s["new"].data_ptr(), s["ring"].data_ptr(),
                                      s["ring"].shape[0], s["free"].data_ptr(),
                                      s["free_out"].data_ptr(), s["rows"].data_ptr(),
                                      s["pos"].data_ptr(), s["req"].data_ptr(), st)
        out = _table_outputs(s)
    elif op == "attn":
        shape = (WF[s["q"]], s["h"], s["dqk"], s["dv"])
        plan = _buffer(s, "plan", lambda: L.dsv4_gpu_reqs_plan_bytes(s["n_req"], s["max_tok"],
                                                                     s["h"]))
        space = _buffer(s, "space", lambda: L.dsv4_gpu_reqs_attn_scratch_bytes(
            *shape, KV[s["kv"]], s["n_req"], s["max_tok"]))
        rc = L.dsv4_gpu_reqs_plan_d(*plan, ctypes.byref(reqs), *shape, KV[s["kv"]], s["window"],
                                    st)
        rc = rc or L.dsv4_gpu_reqs_attn_d(s["out"].data_ptr(), s["qx"].data_ptr(), *shape,
                                          s["cache"].data_ptr(), _at(s["scales"]), KV[s["kv"]],
                                          s["dqk"], s["kv_rows"], ctypes.byref(reqs), *plan,
                                          s["window"], _at(s["sinks"]), s["scale"], *space, st)
        out = s["out"]
    if rc != 0:
        raise RuntimeError("%s: the call was refused" % op)
    return out


def run(s):
    if own:
        return _own(s)
    return dict(tables=_plain_tables, attn=_plain_attn, sample=_plain_sample)[s["op"]](s)


# ------------------------------------------------------- bytes and operations
def work(case):
    if case["op"] == "sample":
        n, v = case["n"], case["vocab"]
        return dict(bytes=n * (v * SIZE[case["fmt"]] + 32), flops=4 * n * v)
    lens = _lengths(case)
    if case["op"] == "tables":
        P = case["page"]
        new = sum(n for _, n in lens)
        taken = sum(-(-n // P) - -(-(n - k) // P) for n, k in lens)
        return dict(bytes=16 * case["n_req"] + 12 * new + 8 * taken, flops=4 * new)
    h, dqk, dv, window, prefix = (case[k] for k in ("h", "dqk", "dv", "window", "prefix"))
    seen = sum(min(p + 1, window) if window else p + 1 for n, k in lens for p in range(n - k, n))
    lo = [max(0, n - k + 1 - window) if window else 0 for n, k in lens]
    rows = max(0, prefix - min(lo)) + sum(n - max(a, prefix) for (n, _), a in zip(lens, lo))
    tokens = sum(k for _, k in lens)
    return dict(bytes=rows * (dqk * SIZE[case["kv"]] + 4 * (case["kv"] == "fp8")) +
                tokens * h * (dqk + dv) * SIZE[case["q"]],
                flops=2 * h * (dqk + dv) * seen)


# ----------------------------------------------------------- in 64 bits
def _exact_tables(s):
    """Request by request, as a scheduler on the host would do it."""
    P, cap = s["page"], s["ring"].shape[0]
    have, new = s["in_use"].tolist(), s["new"].tolist()
    table, ring = s["table"].cpu().numpy().copy(), s["ring"].cpu().numpy().copy()
    head, count = s["free"].tolist()
    first, length, taken, back, asked = [0], [], 0, [], 0
    rows, pos, req = [], [], []
    full = False
    for i in range(s["n_req"]):
        n = max(0, new[i])
        a, b = -(-have[i] // P), -(-(have[i] + n) // P)
        fits = b <= table.shape[1]
        if n and fits:
            asked += b - a
        if not fits or b > a and asked > count:
            n = 0
        full = full or len(rows) + n > s["max_tok"]
        if full:
            n = 0
        if n:
            for e in range(a, b):
                table[i, e] = ring[(head + taken) % cap]
                taken += 1
        for p in range(have[i], have[i] + n):
            rows.append(int(table[i, p // P]) * P + p % P)
            pos.append(p)
            req.append(i)
        first.append(len(rows))
        if new[i] < 0:
            back += table[i, s["prefix"] // P:a].tolist()
        length.append(0 if new[i] < 0 else have[i] + n)
    for j, page in enumerate(back):
        ring[(head + count + j) % cap] = page
    rest = [-1] * (s["max_tok"] - len(rows))
    out = dict(first=first, len=length, table=table, ring=ring,
               free_out=[(head + taken) % cap, count - taken + len(back)], rows=rows + rest,
               pos=pos + rest, req=req + rest)
    return {k: torch.from_numpy(np.asarray(v, np.int32)) for k, v in out.items()}


def _exact_attn(s):
    P, h = s["page"], s["h"]
    data = s["cache"].view(torch.float8_e4m3fn) if s["kv"] == "fp8" else s["cache"]
    out, t0 = [], 0
    for i, (n, new) in enumerate(s["lengths"]):
        pages = s["table"][i, :-(-n // P)].long()
        rows = (pages[:, None] * P + torch.arange(P, device=DEV)).flatten()[:n]
        lo = max(0, n - new + 1 - s["window"]) if s["window"] else 0
        rows = rows[lo:]
        k = data.view(torch.uint8).view(data.shape[0], -1)[rows].view(data.dtype).double()
        if s["scales"] is not None:
            k *= s["scales"].double()[rows, None]
        z = torch.mm(s["qx"][t0:t0 + new].double().reshape(new * h, -1), k.t().contiguous())
        z.mul_(s["scale"])
        bias = np.zeros((new, n - lo))
        for j in range(new):
            p = n - new + j
            bias[j, p + 1 - lo:] = -np.inf
            if s["window"]:
                bias[j, :max(0, p - s["window"] + 1 - lo)] = -np.inf
        z.view(new, h, -1).add_(torch.from_numpy(bias).to(DEV)[:, None, :])
        lse = torch.logsumexp(z, 1)
        if s["sinks"] is not None:
            lse = torch.logaddexp(lse, s["sinks"].double().repeat(new))
        z.sub_(lse[:, None]).exp_()
        out.append(torch.mm(z, k[:, :s["dv"]].contiguous()).view(new, h, -1))
        t0 += new
    return torch.cat(out)


def _exact_sample(s):
    """The pick's probability, row by row on the host; picks and counts are
    whole numbers."""
    rows = s["x"].double().cpu().numpy()
    prob = np.empty(len(rows))
    names = ("temperature", "top_k", "top_p", "min_p", "u")
    rules = zip(*(s[k].double().cpu().numpy() for k in names))
    for i, (t, k, p, floor, u) in enumerate(rules):
        x = np.sort(rows[i])[::-1]
        if t <= 0:
            x, t = x[:1], 1.0
        if k > 0:
            x = x[:int(k)]
        e = np.exp((x - x[0]) / t)
        c = np.cumsum(e)
        kept = len(e) if p >= 1 else 1 + int(np.searchsorted(c[:-1], p * c[-1], side="left"))
        kept = max(1, min(kept, int((e >= floor).sum())))
        at = min(kept - 1, int(np.searchsorted(c[:kept], u * c[kept - 1], side="right")))
        prob[i] = e[at] / c[kept - 1]
    return None, torch.from_numpy(prob), None


def exact(case, seed):
    s = prepare(case, seed)
    return dict(tables=_exact_tables, attn=_exact_attn, sample=_exact_sample)[case["op"]](s)
