"""The calls of a step that verifies drafted tokens over a latent KV cache, as
cases that can be timed and checked: rotary positions for many tokens, rows
quantised into the cache as they are written and read back, attention of a
tree of drafted tokens over the cache, and the rules a request puts on its
logits with the greedy pick.

  own                  False: plain torch; True: the backend's entry points
  listed()             the named cases
  draw(rng)            one more case of the same ranges
  prepare(case, seed)  inputs and buffers, on the GPU
  run(state)           one pass; returns its outputs
  work(case)           bytes and operations a pass cannot do without
  exact(case, seed)    the outputs in 64 bits

Activations are N(0, 1), cache rows N(0, 1) in their stored format, logits
N(0, 3); the RoPE tables are those of a base of 160000.
"""
import ctypes
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
KV = {"f32": 0, "bf16": 1, "fp8": 2}          # DSV4_GPU_KV_*
WF = {"f32": 0, "bf16": 1}                    # DSV4_WF32, DSV4_WBF16
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
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
        # One token's queries of a layer (64 heads of 512, the last 64
        # elements rotated, neighbouring pairs): decode, where latency counts.
        dict(name="rope_decode_1x64x512", op="rope", nt=1, heads=64, hd=512, dim=64, off=448,
             layout="pairs", fmt="f32", inverse=False),
        # A prompt's queries in the other layout, the whole head rotated back.
        dict(name="rope_prompt_4099x64x128", op="rope", nt=4099, heads=64, hd=128, dim=128,
             off=0, layout="halves", fmt="bf16", inverse=True),
        # One token's latent row, rotated and quantised into its cache row.
        dict(name="append_decode_1x576_fp8", op="append", n=1, rows=2048, dim=576, fmt="f32",
             kv="fp8", scatter=True, rope=64),
        # A prompt's latent rows into the rows its pages gave it.
        dict(name="append_prompt_6000x512_fp8", op="append", n=6000, rows=6144, dim=512,
             fmt="f32", kv="fp8", scatter=True, rope=64),
        # The rows an indexer selected, widened for the sparse attention.
        dict(name="read_2048x576_fp8", op="read", n=2048, rows=32768, dim=576, kv="fp8",
             fmt="bf16", scatter=True),
        # A long cache read back whole.
        dict(name="read_131072x576_fp8", op="read", n=131072, rows=131072, dim=576, kv="fp8",
             fmt="f32", scatter=False),
        # One token over a short context: the smallest attention call.
        dict(name="tree_decode_1x64_1500_bf16", op="tree", nt=1, h=64, dqk=576, dv=512,
             ctx=1500, kv="bf16", q="f32", tree=False, window=0, page=0, sink=True),
        # A ragged tree of 13 drafts under a sliding window, few heads.
        dict(name="tree_13x5_777_window_f32", op="tree", nt=13, h=5, dqk=72, dv=40, ctx=777,
             kv="f32", q="f32", tree=True, window=128, page=16, sink=False),
        # A tree of 16 drafts over a long paged FP8 cache.
        dict(name="tree_16x64_32768_fp8", op="tree", nt=16, h=64, dqk=512, dv=512, ctx=32768,
             kv="fp8", q="f32", tree=True, window=0, page=64, sink=True),
        # The widest call: 64 tokens of 128 heads in bf16 over 131072 rows.
        dict(name="tree_64x128_131072_bf16", op="tree", nt=64, h=128, dqk=576, dv=512,
             ctx=131072, kv="bf16", q="bf16", tree=True, window=0, page=0, sink=True),
        # One token's logits: penalties over its history, a grammar mask.
        dict(name="logits_1x129280", op="logits", nt=1, vocab=129280, hist=1000, draft=False,
             bias=False, allow="row"),
        # Every row of a drafted tree, with its path's tokens penalised too.
        dict(name="logits_64x129280", op="logits", nt=64, vocab=129280, hist=16384, draft=True,
             bias=True, allow="row"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["rope", "append", "read", "tree", "tree", "tree", "logits", "logits"])
    if op == "rope":
        hd = rng.choice([64, 128, 192, 512, 576])
        dim = rng.choice([d for d in (32, 64, 128, hd) if d <= hd])
        heads = rng.randint(1, 128)
        return dict(op=op, nt=_log(rng, 1, max(1, (1 << 25) // (heads * hd))), heads=heads,
                    hd=hd, dim=dim, off=rng.choice([0, hd - dim]),
                    layout=rng.choice(["pairs", "halves"]), fmt=rng.choice(["f32", "bf16"]),
                    inverse=rng.random() < 0.5)
    if op == "append":
        dim = rng.choice([128, 512, 576, _log(rng, 32, 600)])
        n = _log(rng, 1, 3800000 // dim - 70)
        return dict(op=op, n=n, rows=n + rng.randint(0, 64), dim=dim,
                    fmt=rng.choice(["f32", "bf16"]), kv=rng.choice(["f32", "bf16", "fp8", "fp8"]),
                    scatter=rng.random() < 0.6, rope=rng.choice([0, 32]))
    if op == "read":
        n = _log(rng, 1, 65536)
        return dict(op=op, n=n, rows=n + _log(rng, 1, 65536),
                    dim=rng.choice([128, 512, 576, _log(rng, 32, 600)]),
                    kv=rng.choice(["f32", "bf16", "fp8", "fp8"]),
                    fmt=rng.choice(["f32", "bf16"]), scatter=rng.random() < 0.6)
    if op == "logits":
        return dict(op=op, nt=rng.choice([1, rng.randint(2, 64)]),
                    vocab=rng.choice([129280, _log(rng, 1000, 200000)]),
                    hist=_log(rng, 1, 131072), draft=rng.random() < 0.5,
                    bias=rng.random() < 0.5, allow=rng.choice(["", "row", "all"]))
    nt = 1 if rng.random() < 0.25 else rng.randint(2, 64)
    h = rng.choice([16, 32, 64, 128, rng.randint(1, 40)])
    dqk, dv = rng.choice([(576, 512), (512, 512), (192, 128), (128, 128),
                          (rng.randint(20, 576),) * 2])
    dv = min(dv, 512)
    ctx = _log(rng, 1, 131072)
    ctx = max(1, min(ctx, (1 << 39) // (nt * h * (dqk + dv))))
    return dict(op=op, nt=nt, h=h, dqk=dqk, dv=dv, ctx=ctx,
                kv=rng.choice(["f32", "bf16", "bf16", "fp8", "fp8"]),
                q=rng.choice(["f32", "bf16"]), tree=rng.random() < 0.7,
                window=rng.choice([0, 0, 128]), page=rng.choice([0, 16, 64]),
                sink=rng.random() < 0.6)


# ------------------------------------------------------------- the inputs
def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1009 + salt)
    return g


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale


def _cache(g, rows, dim, fmt):
    """rows of N(0, 1) in a cache format: (stored data, row scales or None).
    FP8: e4m3 codes under the row's power-of-two scale."""
    v = _normal(g, rows, dim)
    if fmt != "fp8":
        return v.to(DT[fmt]), None
    s = torch.exp2(torch.ceil(torch.log2(v.abs().amax(1) / 448.0)))
    return (v / s[:, None]).to(torch.float8_e4m3fn).view(torch.uint8), s


def _tables(positions, dim):
    """cos and sin of the first `positions` positions, [positions][dim / 2]."""
    f = 160000.0 ** (-torch.arange(0, dim, 2, device=DEV, dtype=torch.float64) / dim)
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _ancestors(rng, nt):
    """A drafted tree: each token's parent is one of the four before it (or
    none); bit j of word t is set where t sees draft j."""
    words = []
    for t in range(nt):
        p = t - 1 - rng.randrange(4)
        words.append((words[p] if p >= 0 else 0) | 1 << t)
    return torch.from_numpy(np.array(words, np.uint64).view(np.int64)).to(DEV)


def _rope(s, dim, off, layout):
    s["cos"], s["sin"] = _tables(8192, dim)
    s.update(dim=dim, off=off, halves=layout == "halves")


def prepare(case, seed):
    import random
    g, rng = _gen(seed, 3), random.Random(seed)
    op = case["op"]
    s = dict(case)
    if op == "rope":
        shape = (case["nt"], case["heads"], case["hd"])
        s["x"] = _normal(g, *shape).to(DT[case["fmt"]])
        s["pos"] = torch.randint(0, 8192, (case["nt"],), generator=g, device=DEV,
                                 dtype=torch.int32)
        s["out"] = torch.empty_like(s["x"])
        _rope(s, case["dim"], case["off"], case["layout"])
    elif op in ("append", "read"):
        n, rows, dim = case["n"], case["rows"], case["dim"]
        s["cache"], s["scales"] = _cache(g, rows, dim, case["kv"])
        order = torch.randperm(rows, generator=g, device=DEV)[:n].to(torch.int32)
        s["at"] = order.contiguous() if case["scatter"] else None
        s["row0"] = 0 if case["scatter"] else rows - n
        s["width"] = dim
        if op == "append":
            s["x"] = _normal(g, n, dim).to(DT[case["fmt"]])
            s["pos"] = torch.arange(n, device=DEV, dtype=torch.int32) % 8192
            if case["rope"]:
                _rope(s, case["rope"], dim - case["rope"], "pairs")
        else:
            s["out"] = torch.empty(n, dim, device=DEV, dtype=DT[case["fmt"]])
    elif op == "tree":
        nt, h, page = case["nt"], case["h"], case["page"]
        total = case["ctx"] + nt
        n_pages = -(-total // page) if page else 0
        rows = n_pages * page if page else total
        s["cache"], s["scales"] = _cache(g, rows, case["dqk"], case["kv"])
        s["pages"] = None
        if page:
            s["pages"] = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        s["rows"], s["n_pages"] = rows, n_pages
        s["qx"] = _normal(g, nt, h, case["dqk"], scale=1.5).to(DT[case["q"]])
        s["mask"] = _ancestors(rng, nt) if case["tree"] else None
        s["sinks"] = _normal(g, h) if case["sink"] else None
        s["out"] = torch.empty(nt, h, case["dv"], device=DEV, dtype=DT[case["q"]])
        s["scale"] = 1.0 / math.sqrt(case["dqk"])
    else:
        nt, vocab = case["nt"], case["vocab"]
        s["x"] = _normal(g, nt, vocab, scale=3.0)
        # text repeats itself: a history's ids come from a fifth of the vocabulary
        s["ids"] = torch.randint(0, max(1, vocab // 5), (case["hist"],), generator=g,
                                 device=DEV, dtype=torch.int32)
        s["drafts"] = s["mask"] = s["dense"] = s["words"] = None
        if case["draft"]:
            s["drafts"] = torch.randint(0, vocab, (nt,), generator=g, device=DEV,
                                        dtype=torch.int32)
            s["mask"] = _ancestors(rng, nt)
        if case["bias"]:
            s["dense"] = _normal(g, vocab)
        if case["allow"]:
            rows = nt if case["allow"] == "row" else 1
            s["words"] = torch.randint(-1 << 31, 1 << 31, (rows, -(-vocab // 32)), generator=g,
                                       device=DEV, dtype=torch.int64).to(torch.int32)
        s["out"] = torch.empty(nt, vocab, device=DEV)
        s["pick"] = torch.empty(nt, device=DEV, dtype=torch.int32)
        s.update(repetition=1.1, frequency=0.2, presence=0.3)
    return s


# ------------------------------------------------------------ the plain forms
def _rotate(x, s, pos, inverse):
    """x [..., heads, width] in 32 bits with its rotated part turned."""
    half = s["dim"] // 2
    c = s["cos"][pos.long()][:, None, :]
    n = s["sin"][pos.long()][:, None, :]
    n = -n if inverse else n
    part = x[..., s["off"]:s["off"] + s["dim"]]
    if s["halves"]:
        a, b = part[..., :half], part[..., half:]
        turned = torch.cat([a * c - b * n, a * n + b * c], -1)
    else:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
    return torch.cat([x[..., :s["off"]], turned, x[..., s["off"] + s["dim"]:]], -1)


def _stored(s):
    """The cache's rows as the values they stand for, in 32 bits."""
    if s["scales"] is None:
        return s["cache"].float()
    return s["cache"].view(torch.float8_e4m3fn).float() * s["scales"][:, None]


def _plain_append(s):
    x = s["x"].float()
    if s["rope"]:
        x = _rotate(x[:, None, :], s, s["pos"], False)[:, 0, :]
    at = torch.arange(s["row0"], s["row0"] + s["n"], device=DEV) if s["at"] is None \
        else s["at"].long()
    if s["kv"] != "fp8":
        s["cache"][at] = x.to(s["cache"].dtype)
        return s["cache"]
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(1)
    m, e = torch.frexp(top.double() / 448.0)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-126)
    scale = torch.where(top == 0, 1.0, torch.exp2(e.double())).float()
    s["cache"][at] = (x / scale[:, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    s["scales"][at] = scale
    return s["cache"].view(torch.float8_e4m3fn), s["scales"]


def _plain_read(s):
    at = torch.arange(s["row0"], s["row0"] + s["n"], device=DEV) if s["at"] is None \
        else s["at"].long()
    rows = s["cache"][at]
    if s["scales"] is None:
        return rows.float().to(s["out"].dtype)
    return (rows.view(torch.float8_e4m3fn).float() * s["scales"][at][:, None]).to(s["out"].dtype)


def _visible(s):
    """[nt][ctx + nt]: which rows a token sees."""
    nt, ctx = s["nt"], s["ctx"]
    j = torch.arange(nt, device=DEV)
    if s["mask"] is None:
        tree = j[None, :] <= j[:, None]
    else:
        tree = ((s["mask"][:, None] >> j[None, :]) & 1).bool()
    see = torch.cat([torch.ones(nt, ctx, device=DEV, dtype=torch.bool), tree], 1)
    if s["window"]:
        depth = ctx + (tree & (j[None, :] != j[:, None])).sum(1)
        at = torch.cat([torch.arange(ctx, device=DEV), depth])
        see &= depth[:, None] - at[None, :] < s["window"]
    return see


def _plain_tree(s):
    nt, h, page = s["nt"], s["h"], s["page"]
    n = torch.arange(s["ctx"] + nt, device=DEV)
    k = _stored(s)
    if page:
        k = k[s["pages"].long()[n // page] * page + n % page]
    p = (s["qx"].float().view(nt * h, -1) @ k.t()).view(nt, h, -1) * s["scale"]
    p.masked_fill_(~_visible(s)[:, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p.sub_(top).exp_()
    total = p.sum(-1)
    if s["sinks"] is not None:
        total = total + torch.exp(s["sinks"] - top[..., 0])
    o = (p.view(nt * h, -1) @ k[:, :s["dv"]]).view(nt, h, -1)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    return o.to(s["out"].dtype)


def _plain_logits(s):
    nt, vocab = s["nt"], s["vocab"]
    seen = torch.zeros(nt, vocab, device=DEV)
    seen += torch.zeros(vocab, device=DEV).index_add_(
        0, s["ids"].long(), torch.ones(s["hist"], device=DEV))
    if s["drafts"] is not None:
        j = torch.arange(nt, device=DEV)
        on = ((s["mask"][:, None] >> j[None, :]) & 1).float()
        seen.index_add_(1, s["drafts"].long(), on)
    x = s["x"]
    y = torch.where(seen > 0, torch.where(x > 0, x / s["repetition"], x * s["repetition"]), x)
    y = torch.where(seen > 0, y - (seen * s["frequency"] + s["presence"]), y)
    if s["dense"] is not None:
        y = y + s["dense"]
    if s["words"] is not None:
        v = torch.arange(vocab, device=DEV)
        ok = ((s["words"][:, v // 32] >> (v % 32)) & 1).bool()
        y = torch.where(ok, y, -math.inf)
    return y, y.argmax(1).to(torch.int32)


# ----------------------------------------------------------------- a pass
def _at(t):
    return None if t is None else t.data_ptr()


def _buffer(s, bytes_):
    """The call's workspace, which a program keeps beside its other buffers."""
    if "space" not in s:
        s["space"] = torch.empty(max(16, bytes_), device=DEV, dtype=torch.uint8)
    return s["space"].data_ptr(), s["space"].numel()


def _rope_struct(D, s):
    return D.Rope(cos=s["cos"].data_ptr(), sin=s["sin"].data_ptr(), max_pos=s["cos"].shape[0],
                  dim=s["dim"], offset=s["off"],
                  layout=D.ROPE_HALVES if s["halves"] else D.ROPE_PAIRS)


def _own(s):
    D = backend()
    L, op = D.lib(), s["op"]
    st = torch.cuda.current_stream().cuda_stream or None
    if op == "rope":
        pitch = s["heads"] * s["hd"]
        rc = L.dsv4_gpu_rope_n_d(s["out"].data_ptr(), pitch, s["x"].data_ptr(), pitch,
                                 WF[s["fmt"]], s["pos"].data_ptr(), s["nt"], s["heads"], s["hd"],
                                 ctypes.byref(_rope_struct(D, s)), int(s["inverse"]), st)
        out = s["out"]
    elif op == "append":
        rope = ctypes.byref(_rope_struct(D, s)) if s["rope"] else None
        rc = L.dsv4_gpu_kv_append_d(s["cache"].data_ptr(), _at(s["scales"]), KV[s["kv"]],
                                    s["width"], s["rows"], s["x"].data_ptr(), WF[s["fmt"]],
                                    s["width"], s["n"], s["width"], _at(s["at"]), s["row0"],
                                    rope, s["pos"].data_ptr(), st)
        out = s["cache"] if s["kv"] != "fp8" else (s["cache"].view(torch.float8_e4m3fn),
                                                   s["scales"])
    elif op == "read":
        rc = L.dsv4_gpu_kv_read_d(s["out"].data_ptr(), WF[s["fmt"]], s["width"],
                                  s["cache"].data_ptr(), _at(s["scales"]), KV[s["kv"]],
                                  s["width"], s["rows"], _at(s["at"]), s["row0"], s["n"],
                                  s["width"], st)
        out = s["out"]
    elif op == "tree":
        shape = (WF[s["q"]], s["nt"], s["h"], s["dqk"], s["dv"])
        space = _buffer(s, 0 if "space" in s else L.dsv4_gpu_tree_attn_scratch_bytes(
            *shape, KV[s["kv"]], s["ctx"], s["window"]))
        rc = L.dsv4_gpu_tree_attn_d(s["out"].data_ptr(), s["qx"].data_ptr(), *shape,
                                    s["cache"].data_ptr(), _at(s["scales"]), KV[s["kv"]],
                                    s["dqk"], s["rows"], _at(s["pages"]), s["n_pages"],
                                    s["page"], s["ctx"], _at(s["mask"]), s["window"],
                                    _at(s["sinks"]), s["scale"], *space, st)
        out = s["out"]
    else:
        words = s["words"]
        rules = D.LogitRules(hist=s["ids"].data_ptr(), n_hist=s["hist"], draft=_at(s["drafts"]),
                             mask=_at(s["mask"]), repetition=s["repetition"],
                             frequency=s["frequency"], presence=s["presence"],
                             bias=_at(s["dense"]), allow=_at(words),
                             allow_stride=words.shape[1] if s["allow"] == "row" else 0)
        space = _buffer(s, L.dsv4_gpu_logits_scratch_bytes(s["nt"], s["vocab"]))
        rc = L.dsv4_gpu_logits_adjust_d(s["out"].data_ptr(), s["pick"].data_ptr(),
                                        s["x"].data_ptr(), s["nt"], s["vocab"], s["vocab"],
                                        ctypes.byref(rules), *space, st)
        out = (s["out"], s["pick"])
    if rc != 0:
        raise RuntimeError("%s: the call was refused" % op)
    return out


def run(s):
    if own:
        return _own(s)
    if s["op"] == "rope":
        return _rotate(s["x"].float(), s, s["pos"], s["inverse"]).to(s["x"].dtype)
    return dict(append=_plain_append, read=_plain_read, tree=_plain_tree,
                logits=_plain_logits)[s["op"]](s)


# ------------------------------------------------------- bytes and operations
SIZE = {"f32": 4, "bf16": 2, "fp8": 1}


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["nt"] * case["heads"]
        return dict(bytes=2 * n * case["hd"] * SIZE[case["fmt"]] + 4 * case["nt"] * (1 + case["dim"]),
                    flops=3 * n * case["dim"])
    if op in ("append", "read"):
        n, d = case["n"], case["dim"]
        b = n * d * (SIZE[case["fmt"]] + SIZE[case["kv"]])
        b += 4 * n * ((case["kv"] == "fp8") + bool(case["scatter"]))
        if op == "append" and case["rope"]:
            b += 4 * n * (1 + case["rope"])
        return dict(bytes=b, flops=2 * n * d)
    if op == "tree":
        nt, h, dqk, dv = case["nt"], case["h"], case["dqk"], case["dv"]
        ctx = min(case["ctx"], case["window"]) if case["window"] else case["ctx"]
        drafts = 2 if case["tree"] else (nt + 1) / 2           # seen of its own kind
        rows = ctx + nt
        b = rows * (dqk * SIZE[case["kv"]] + 4 * (case["kv"] == "fp8"))
        return dict(bytes=b + nt * h * (dqk + dv) * SIZE[case["q"]],
                    flops=2 * nt * h * (dqk + dv) * (ctx + drafts))
    nt, v = case["nt"], case["vocab"]
    b = 8 * nt * v + 4 * case["hist"] + 4 * v * bool(case["bias"])
    if case["allow"]:
        b += 4 * -(-v // 32) * (nt if case["allow"] == "row" else 1)
    return dict(bytes=b, flops=4 * nt * v)


# ----------------------------------------------------------- in 64 bits
def _e4m3(v):
    """The e4m3 value nearest to v (|v| <= 448), ties to the even code."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -9))).clamp(-6, 8)
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _turn64(x, cos, sin, pos, off, dim, halves, sign):
    """Each rotated pair as a complex number times cos + i sin."""
    z = x.clone()
    w = torch.complex(cos.double()[pos.long()], sign * sin.double()[pos.long()])
    first = torch.arange(dim // 2, device=DEV) if halves else torch.arange(0, dim, 2, device=DEV)
    second = first + (dim // 2 if halves else 1)
    t = torch.complex(x[:, :, off + first], x[:, :, off + second]) * w[:, None, :]
    z[:, :, off + first], z[:, :, off + second] = t.real, t.imag
    return z


def _value64(s):
    if s["kv"] == "fp8":
        return s["cache"].view(torch.float8_e4m3fn).double() * s["scales"].double()[:, None]
    return s["cache"].double()


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _turn64(s["x"].double(), s["cos"], s["sin"], s["pos"], case["off"], case["dim"],
                       case["layout"] == "halves", -1.0 if case["inverse"] else 1.0)
    if op in ("append", "read"):
        rows = torch.arange(case["n"], device=DEV) + s["row0"]
        if s["at"] is not None:
            rows = s["at"].long()
        if op == "read":
            return _value64(s).index_select(0, rows)
        x = s["x"].double()
        if case["rope"]:
            x = _turn64(x[:, None, :], s["cos"], s["sin"], s["pos"], case["dim"] - case["rope"],
                        case["rope"], False, 1.0)[:, 0, :]
        if case["kv"] != "fp8":
            return s["cache"].double().index_copy(0, rows, x)
        # the smallest power of two that brings the row's largest under 448
        power = torch.ceil(torch.log2(x.abs().amax(1) / 448.0))
        scale = torch.exp2(power)
        codes = s["cache"].view(torch.float8_e4m3fn).double()
        return (codes.index_copy(0, rows, _e4m3(x / scale[:, None])),
                s["scales"].double().index_copy(0, rows, scale))
    if op == "tree":
        nt, h, ctx = case["nt"], case["h"], case["ctx"]
        k = _value64(s)
        if case["page"]:
            k = k.view(s["n_pages"], case["page"], -1)[s["pages"].long()].flatten(0, 1)
        k = k[:ctx + nt].contiguous()
        # the rows each token sees, from its word alone
        words = [(1 << t + 1) - 1 for t in range(nt)] if s["mask"] is None else \
            [int(w) & (1 << 64) - 1 for w in s["mask"].tolist()]
        bias = np.zeros((nt, ctx + nt))
        place = [ctx + bin(words[t] & ~(1 << t)).count("1") for t in range(nt)]
        for t in range(nt):
            if case["window"]:
                bias[t, :max(0, min(ctx, place[t] - case["window"] + 1))] = -np.inf
            for j in range(nt):
                far = case["window"] and place[t] - place[j] >= case["window"]
                if far or not words[t] >> j & 1:
                    bias[t, ctx + j] = -np.inf
        z = torch.mm(s["qx"].double().reshape(nt * h, -1), k.t().contiguous())
        z.mul_(s["scale"])
        z.view(nt, h, -1).add_(torch.from_numpy(bias).to(DEV)[:, None, :])
        if s["sinks"] is not None:
            lse = torch.logaddexp(torch.logsumexp(z, 1), s["sinks"].double().repeat(nt))
        else:
            lse = torch.logsumexp(z, 1)
        z.sub_(lse[:, None]).exp_()
        return torch.mm(z, k[:, :case["dv"]].contiguous()).view(nt, h, -1)
    nt, vocab = case["nt"], case["vocab"]
    ids, x = s["ids"].cpu().numpy(), s["x"].double().cpu().numpy()
    base = np.bincount(ids, minlength=vocab)
    drafts = None if s["drafts"] is None else s["drafts"].cpu().numpy()
    words = None if s["words"] is None else s["words"].cpu().numpy().view(np.uint8)
    out = np.empty((nt, vocab))
    # the penalties' own values are floats of 32 bits
    rep, freq, pres = (float(np.float32(s[k])) for k in ("repetition", "frequency", "presence"))
    for t in range(nt):
        count = base.copy()
        for j in range(nt if drafts is not None else 0):
            if int(s["mask"][t]) >> j & 1:
                count[drafts[j]] += 1
        hit = count > 0
        row = x[t].copy()
        row[hit] = np.where(row[hit] > 0, row[hit] / rep, row[hit] * rep)
        row[hit] -= freq * count[hit] + pres
        if s["dense"] is not None:
            row += s["dense"].double().cpu().numpy()
        if words is not None:
            w = words[t if case["allow"] == "row" else 0]
            row[np.unpackbits(w, bitorder="little")[:vocab] == 0] = -np.inf
        out[t] = row
    return torch.from_numpy(out), None
