"""The operators on drafted tokens refuse what they do not take before any
launch, do nothing for a length of zero, and report a failed launch. CPU only:
nothing is launched."""
import hip_shim

CHILD = r"""
buf = np.zeros(1 << 12, np.uint8)
p = (buf.ctypes.data + 255) // 256 * 256                     # nothing reads it
assert L.dsv4_gpu_init() == 0


def rope(**kw):
    r = dict(cos=p, sin=p, max_pos=8, dim=32, offset=0, layout=0)
    r.update(kw)
    return ctypes.byref(D.Rope(**r))


def rules(**kw):
    r = dict(hist=p, n_hist=8, repetition=1.0)
    r.update(kw)
    return ctypes.byref(D.LogitRules(**r))


BIG = 1 << 40
ROPE = dict(out=p, os=256, x=p, xs=256, fmt=0, pos=p, nt=2, heads=4, hd=64, rope=rope(), inv=0,
            st=None)
APPEND = dict(kv=p, ks=p, fmt=2, stride=64, rows=8, x=p, xf=0, xs=64, n=2, dim=64, at=p, row0=0,
              rope=rope(), pos=p, st=None)
READ = dict(out=p, of=0, os=64, kv=p, ks=p, fmt=2, stride=64, rows=8, at=p, row0=0, n=2, dim=64,
            st=None)
TREE = dict(o=p, q=p, fmt=0, nt=2, h=4, dqk=64, dv=32, kv=p, ks=p, kf=2, stride=64, rows=8,
            pages=None, n_pages=0, page=0, ctx=6, mask=p, window=0, sink=None, scale=1.0, space=p,
            bytes=BIG, st=None)
LOGITS = dict(out=p, pick=p, x=p, nt=2, vocab=100, stride=100, rules=rules(), space=p, bytes=BIG,
              st=None)
CALLS = {
    "dsv4_gpu_rope_n_d": (ROPE, [
        dict(out=None), dict(x=None), dict(pos=None), dict(nt=-1), dict(heads=0), dict(hd=0),
        dict(fmt=2), dict(fmt=-1), dict(xs=255), dict(os=255), dict(x=p + 0, out=p, os=512),
        dict(rope=None), dict(rope=rope(cos=None)), dict(rope=rope(sin=None)),
        dict(rope=rope(max_pos=0)), dict(rope=rope(dim=31)), dict(rope=rope(dim=0)),
        dict(rope=rope(dim=-2)), dict(rope=rope(offset=-1)), dict(rope=rope(offset=33)),
        dict(rope=rope(dim=66)), dict(rope=rope(layout=2)), dict(rope=rope(offset=2 ** 31 - 1)),
        dict(heads=1 << 16, hd=1 << 16, xs=BIG, os=BIG), dict(nt=(1 << 30) + 1)], dict(nt=0)),
    "dsv4_gpu_kv_append_d": (APPEND, [
        dict(kv=None), dict(ks=None), dict(fmt=3), dict(fmt=-1), dict(stride=63), dict(rows=0),
        dict(x=None), dict(xf=2), dict(xs=63), dict(n=-1), dict(dim=0),
        dict(dim=16385, stride=16385, xs=16385), dict(at=None, row0=7), dict(at=None, row0=-1),
        dict(at=None, row0=2 ** 31 - 1), dict(pos=None), dict(rope=rope(dim=66)),
        dict(rope=rope(layout=-1)), dict(rope=rope(cos=None)), dict(n=(1 << 30) + 1)], dict(n=0)),
    "dsv4_gpu_kv_read_d": (READ, [
        dict(kv=None), dict(ks=None), dict(fmt=3), dict(stride=63), dict(rows=0), dict(out=None),
        dict(of=2), dict(os=63), dict(n=-1), dict(dim=0), dict(dim=16385, stride=16385, os=16385),
        dict(at=None, row0=7), dict(at=None, row0=-1), dict(n=(1 << 30) + 1)], dict(n=0)),
    "dsv4_gpu_tree_attn_d": (TREE, [
        dict(o=None), dict(q=None), dict(kv=None), dict(ks=None), dict(fmt=2), dict(kf=3),
        dict(nt=-1), dict(nt=65), dict(h=0), dict(h=4097), dict(dqk=0, dv=0), dict(dv=0),
        dict(dv=65), dict(dqk=577, stride=577), dict(dqk=576, dv=513, stride=576),
        dict(stride=63), dict(rows=0), dict(pages=p, page=0), dict(pages=p, page=4, n_pages=-1),
        dict(ctx=-1), dict(ctx=2 ** 31 - 1), dict(window=-1)], dict(nt=0)),
    "dsv4_gpu_logits_adjust_d": (LOGITS, [
        dict(x=None), dict(nt=-1), dict(nt=65), dict(vocab=0), dict(vocab=(1 << 30) + 1,
        stride=BIG), dict(stride=99), dict(rules=None), dict(rules=rules(n_hist=-1)),
        dict(rules=rules(n_hist=(1 << 30) + 1)),
        dict(rules=rules(hist=None)), dict(rules=rules(repetition=0.0)),
        dict(rules=rules(repetition=-1.0)), dict(rules=rules(repetition=float("nan"))),
        dict(rules=rules(allow=p, allow_stride=3)), dict(rules=rules(allow=p, allow_stride=-1)),
        dict(space=None), dict(space=p + 8), dict(bytes=0)], dict(nt=0)),
}
for name, (good, bad, nothing) in CALLS.items():
    f = getattr(L, name)

    def call(**kw):
        return f(*dict(good, **kw).values())

    shim.shim_reset(-1, 0)
    assert call() == 0 and shim.shim_launches() >= 1, name
    n = shim.shim_launches()
    for at in range(n):
        shim.shim_reset(at, 0)
        assert call() == -1, (name, at)
    for kw in bad:
        shim.shim_reset(-1, 0)
        assert call(**kw) == -1, (name, kw)
        assert shim.shim_launches() == 0, (name, kw)
    shim.shim_reset(-1, 0)
    assert call(**nothing) == 0 and shim.shim_launches() == 0, name

# a long attention call asks for a workspace, whole and aligned
shape = (0, 1, 64, 576, 512, 1, 100000, 0)
need = L.dsv4_gpu_tree_attn_scratch_bytes(*shape)
big = dict(TREE, nt=1, h=64, dqk=576, dv=512, kf=1, stride=576, rows=100001, ctx=100000)
f = L.dsv4_gpu_tree_attn_d
assert f(*big.values()) == 0
if need:
    for kw in (dict(space=None), dict(space=p + 8), dict(bytes=need - 1)):
        shim.shim_reset(-1, 0)
        assert f(*dict(big, **kw).values()) == -1 and shim.shim_launches() == 0, kw
    assert f(*dict(big, bytes=need).values()) == 0
last = 0
for ctx in list(range(0, 3000, 37)) + [2 ** k for k in range(12, 30)]:
    n = L.dsv4_gpu_tree_attn_scratch_bytes(0, 3, 64, 512, 512, 2, ctx, 0)
    assert n >= last, ctx
    last = n
assert L.dsv4_gpu_tree_attn_scratch_bytes(0, 65, 64, 512, 512, 2, 100, 0) == 0
assert L.dsv4_gpu_logits_scratch_bytes(65, 100) == 0
# picks only where they are asked for: then no workspace is
assert L.dsv4_gpu_logits_adjust_d(*dict(LOGITS, pick=None, space=None, bytes=0).values()) == 0
print("done")
"""


def test_refusals(tmp_path):
    assert hip_shim.run(tmp_path, CHILD).endswith("done\n")
