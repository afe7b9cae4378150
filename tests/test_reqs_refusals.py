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
SAMPLE = dict(pick=p, prob=p, kept=p, x=p, fmt=0, n=2, vocab=100, stride=100, s=rules(), space=p,
              bytes=BIG, st=None)
CALLS = {
    "dsv4_gpu_reqs_tables_d": (TABLES, BATCHES + [
        dict(len=None), dict(new=None), dict(ring=None), dict(cap=0), dict(cap=(1 << 30) + 1),
        dict(free=None), dict(out=None)],
        [dict(r=reqs(max_tok=100000)), dict(r=reqs(n_req=4096)), dict(rows=None, pos=None, req=None),
         dict(r=reqs(n_req=0, len=None, pages=None), len=None, new=None)]),
    "dsv4_gpu_sample_d": (SAMPLE, [
        dict(pick=None), dict(x=None), dict(fmt=2), dict(fmt=-1), dict(n=-1), dict(n=65537),
        dict(vocab=0), dict(vocab=(1 << 22) + 1, stride=BIG), dict(stride=99), dict(s=None),
        dict(s=rules(u=None)), dict(space=None), dict(space=p + 8),
        dict(bytes=L.dsv4_gpu_sample_scratch_bytes(2, 100) - 1)],
        [dict(fmt=1), dict(prob=None, kept=None), dict(n=65536),
         dict(s=rules(temperature=None, top_k=None, top_p=None, min_p=None)),
         dict(bytes=L.dsv4_gpu_sample_scratch_bytes(2, 100))]),
}
NOTHING = {"dsv4_gpu_sample_d": dict(n=0, pick=None, x=None, space=None, bytes=0)}
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
assert size(0, 100) == size(65537, 100) == size(1, 0) == size(1, (1 << 22) + 1) == 0
print("done")
"""


def test_refusals(tmp_path):
    assert hip_shim.run(tmp_path, CHILD).endswith("done\n")
