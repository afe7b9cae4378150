"""The operators on batches of requests refuse what they do not take before any
launch, do nothing for a length of zero, and report a failed launch. CPU only:
nothing is launched."""
import hip_shim

CHILD = r"""
buf = np.zeros(1 << 12, np.uint8)
p = (buf.ctypes.data + 255) // 256 * 256                     # nothing reads it
assert L.dsv4_gpu_init() == 0
BIG = 1 << 40


def reqs(**kw):
    r = dict(len=p, pages=p, first=p, n_req=3, max_pages=4, page_rows=16, max_tok=5, n_prefix=0)
    r.update(kw)
    return ctypes.byref(D.Reqs(**r))


def rules(**kw):
    r = dict(temperature=p, top_k=p, top_p=p, min_p=p, u=p)
    r.update(kw)
    return ctypes.byref(D.Sampling(**r))


BATCHES = [dict(r=None)] + [dict(r=reqs(**kw)) for kw in (
    dict(n_req=-1), dict(n_req=4097), dict(max_pages=0), dict(page_rows=0), dict(page_rows=-1),
    dict(max_pages=1 << 16, page_rows=(1 << 14) + 1), dict(max_tok=-1), dict(max_tok=(1 << 20) + 1),
    dict(n_prefix=-1), dict(len=None), dict(pages=None), dict(first=None))]
TABLES = dict(r=reqs(), len=p, new=p, ring=p, cap=64, free=p, out=p, rows=p, pos=p, req=p, st=None)
PLAN = dict(plan=p, pb=BIG, r=reqs(), fmt=0, h=4, dqk=64, dv=32, kf=2, window=0, st=None)
ATTN = dict(o=p, q=p, fmt=0, h=4, dqk=64, dv=32, kv=p, ks=p, kf=2, stride=64, rows=8, r=reqs(), plan=p,
            pb=BIG, window=0, sink=None, scale=1.0, space=p, sb=BIG, st=None)
SHAPES = [dict(fmt=2), dict(fmt=-1), dict(kf=3), dict(kf=-1), dict(h=0), dict(h=4097), dict(dqk=0, dv=0),
          dict(dv=0), dict(dv=65), dict(dqk=577), dict(dqk=576, dv=513), dict(window=-1),
          dict(r=reqs(max_tok=1 << 17), h=2049), dict(plan=None), dict(plan=p + 8),
          dict(pb=L.dsv4_gpu_reqs_plan_bytes(3, 5, 4) - 1)]
SAMPLE = dict(pick=p, prob=p, kept=p, x=p, fmt=0, n=2, vocab=100, stride=100, s=rules(), space=p,
              bytes=BIG, st=None)
CALLS = {
    "dsv4_gpu_reqs_tables_d": (TABLES, BATCHES + [
        dict(len=None), dict(new=None), dict(ring=None), dict(cap=0), dict(cap=(1 << 30) + 1),
        dict(free=None), dict(out=None)],
        [dict(r=reqs(max_tok=100000)), dict(r=reqs(n_req=4096)), dict(rows=None, pos=None, req=None),
         dict(r=reqs(n_req=0, len=None, pages=None), len=None, new=None)]),
    "dsv4_gpu_reqs_plan_d": (PLAN, [k for k in BATCHES if k != dict(r=BATCHES[-2]["r"])] + SHAPES,
        [dict(r=reqs(pages=None)), dict(r=reqs(n_req=0, len=None)), dict(r=reqs(max_tok=0)),
         dict(pb=L.dsv4_gpu_reqs_plan_bytes(3, 5, 4))]),
    "dsv4_gpu_reqs_attn_d": (ATTN, BATCHES[:10] + [dict(r=reqs(pages=None))] + SHAPES + [
        dict(o=None), dict(q=None), dict(kv=None), dict(ks=None), dict(stride=63), dict(rows=0),
        dict(dqk=576, dv=512, stride=575), dict(space=None), dict(space=p + 8),
        dict(sb=L.dsv4_gpu_reqs_attn_scratch_bytes(0, 4, 64, 32, 2, 3, 5) - 1)],
        [dict(kf=0, ks=None), dict(kf=1, ks=None, fmt=1), dict(r=reqs(len=None, first=None)),
         dict(sb=L.dsv4_gpu_reqs_attn_scratch_bytes(0, 4, 64, 32, 2, 3, 5))]),
    "dsv4_gpu_sample_d": (SAMPLE, [
        dict(pick=None), dict(x=None), dict(fmt=2), dict(fmt=-1), dict(n=-1), dict(n=65537),
        dict(vocab=0), dict(vocab=(1 << 22) + 1, stride=BIG), dict(stride=99), dict(s=None),
        dict(s=rules(u=None)), dict(space=None), dict(space=p + 8),
        dict(bytes=L.dsv4_gpu_sample_scratch_bytes(2, 100) - 1)],
        [dict(fmt=1), dict(prob=None, kept=None), dict(n=65536),
         dict(s=rules(temperature=None, top_k=None, top_p=None, min_p=None)),
         dict(bytes=L.dsv4_gpu_sample_scratch_bytes(2, 100))]),
}
NOTHING = {"dsv4_gpu_reqs_attn_d": dict(r=reqs(max_tok=0), o=None, q=None, kv=None, plan=None, pb=0,
                                        space=None, sb=0),
           "dsv4_gpu_sample_d": dict(n=0, pick=None, x=None, space=None, bytes=0)}
for name, (good, bad, also) in CALLS.items():
    f = getattr(L, name)

    def call(**kw):
        return f(*dict(good, **kw).values())

    for kw in [{}] + also:
        shim.shim_reset(-1, 0)
        assert call(**kw) == 0 and shim.shim_launches() >= 1, (name, kw)
        n = shim.shim_launches()
        for at in range(n):
            shim.shim_reset(at, 0)
            assert call(**kw) == -1, (name, kw, at)
    for kw in bad:
        shim.shim_reset(-1, 0)
        assert call(**kw) == -1, (name, kw)
        assert shim.shim_launches() == 0, (name, kw)
    if name in NOTHING:
        shim.shim_reset(-1, 0)
        assert call(**NOTHING[name]) == 0 and shim.shim_launches() == 0, name

# a workspace for the most rows or tokens serves fewer
size = L.dsv4_gpu_sample_scratch_bytes
for n in (1, 2, 63, 64, 65, 1000):
    last = 0
    for vocab in (1, 63, 64, 65, 8191, 8192, 8193, 16385, 32769, 129280, 1 << 22):
        assert size(n, vocab) >= max(last, size(n - 1, vocab)), (n, vocab)
        last = size(n, vocab)
for a, b in ((0, 1), (1, 2), (63, 64), (1000, 1001), (4095, 4096)):
    for h in (1, 5, 64, 128):
        for tok in (0, 1, 64, 1000, 1023, 1024, 4096, 100000):
            plan, space = L.dsv4_gpu_reqs_plan_bytes, L.dsv4_gpu_reqs_attn_scratch_bytes
            assert plan(a, tok, h) <= min(plan(b, tok, h), plan(a, tok + 1, h), plan(a, tok, h + 1))
            shape = (0, h, 576, 512, 2)
            assert 0 < space(*shape, a, tok) <= min(space(*shape, b, tok), space(*shape, a, tok + 1))
assert L.dsv4_gpu_reqs_plan_bytes(4097, 1, 1) == L.dsv4_gpu_reqs_plan_bytes(1, 1 << 18, 2048) == 0
assert L.dsv4_gpu_reqs_attn_scratch_bytes(0, 4, 576, 577, 2, 3, 5) == 0
assert size(0, 100) == size(65537, 100) == size(1, 0) == size(1, (1 << 22) + 1) == 0
print("done")
"""


def test_refusals(tmp_path):
    assert hip_shim.run(tmp_path, CHILD).endswith("done\n")
