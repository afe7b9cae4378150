"""The workspaces of the operators on drafted tokens: what a program may ask for
once and then use for every smaller call. CPU only: nothing is launched."""
import hip_shim

COMMON = r"""
buf = np.zeros(1 << 12, np.uint8)
p = (buf.ctypes.data + 255) // 256 * 256                     # nothing reads it
assert L.dsv4_gpu_init() == 0
size = L.dsv4_gpu_tree_attn_scratch_bytes


def tree(shape, bytes):
    fmt, nt, h, dqk, dv, kf, ctx, window = shape
    shim.shim_reset(-1, 0)
    return L.dsv4_gpu_tree_attn_d(p, p, fmt, nt, h, dqk, dv, p, p, kf, dqk, ctx + nt, None, 0, 0,
                                  ctx, p, window, None, 1.0, p, bytes, None)
"""


def test_a_windows_workspace_serves_every_shorter_context(tmp_path):
    """The bytes do not fall as the context grows, whatever the window, and a
    call with those of the longest is taken at each shorter length."""
    child = COMMON + r"""
for fmt, nt, h, dqk, dv, kf in ((0, 1, 64, 576, 512, 2), (1, 13, 64, 128, 128, 1),
                                (0, 64, 3, 512, 512, 0)):
    for window in (1, 31, 32, 33, 100, 128, 5000):
        ctxs = list(range(0, 6000)) + [65536 + k for k in range(-70, 70)]
        last = 0
        for ctx in ctxs:
            n = size(fmt, nt, h, dqk, dv, kf, ctx, window)
            assert n >= last, (fmt, nt, window, ctx, n, last)
            last = n
        for ctx in ctxs[::7] + ctxs[-140:]:
            assert tree((fmt, nt, h, dqk, dv, kf, ctx, window), last) == 0, (fmt, nt, window, ctx)
print("done")
"""
    assert hip_shim.run(tmp_path, child).endswith("done\n")


def test_a_window_longer_than_the_context_is_no_window(tmp_path):
    """Up to the largest number there is: the same bytes, and where the cache is
    split without a window (two launches) it is split with one."""
    child = COMMON + r"""
for fmt, nt, h, dqk, dv, kf in ((0, 1, 64, 576, 512, 1), (1, 13, 64, 128, 128, 2),
                                (0, 64, 3, 512, 512, 0)):
    for ctx in (0, 1, 33, 1000, 32768, 100000):
        want = size(fmt, nt, h, dqk, dv, kf, ctx, 0)
        assert tree((fmt, nt, h, dqk, dv, kf, ctx, 0), want) == 0
        launches = shim.shim_launches()
        assert launches == 2 or ctx < 32768
        for window in (2 ** 31 - 1, 2 ** 31 - 1 - nt, 2 ** 31 - nt, 2 ** 30, ctx + 4096):
            assert size(fmt, nt, h, dqk, dv, kf, ctx, window) == want, (ctx, window)
            assert tree((fmt, nt, h, dqk, dv, kf, ctx, window), want) == 0
            assert shim.shim_launches() == launches, (ctx, window)
print("done")
"""
    assert hip_shim.run(tmp_path, child).endswith("done\n")


def test_a_trees_workspace_serves_smaller_trees(tmp_path):
    """The attention's bytes do not fall as tokens or heads are added, and calls
    of fewer are taken with those of the most; a call of one split takes any."""
    child = COMMON + r"""
for fmt, dqk, dv, kf in ((0, 576, 512, 1), (0, 512, 512, 0), (1, 576, 512, 1), (1, 128, 128, 2)):
    for ctx, window in ((100000, 0), (3000, 0), (70000, 128), (40, 0)):
        for hs in ((1, 5, 16, 40, 64, 65, 128, 1000, 4096), (64,)):
            prev = {}
            for h in hs:
                last = 0
                for nt in range(1, 65):
                    n = size(fmt, nt, h, dqk, dv, kf, ctx, window)
                    assert n >= last, (fmt, h, nt, ctx, window, n, last)
                    assert n >= prev.get(nt, 0), (fmt, h, nt, ctx, window)
                    last = prev[nt] = n
                for nt in range(1, 65, 3 if len(hs) > 1 else 1):
                    assert tree((fmt, nt, h, dqk, dv, kf, ctx, window), last) == 0, (h, nt, ctx)
# one split: nothing is written to a workspace
for shape in ((0, 64, 4096, 576, 512, 1, 100000, 0), (0, 1, 16, 64, 64, 1, 20, 0)):
    assert tree(shape, 0) == 0 and shim.shim_launches() == 1, shape
print("done")
"""
    assert hip_shim.run(tmp_path, child).endswith("done\n")


def test_the_logits_workspace_serves_fewer_rows(tmp_path):
    """The bytes do not fall as rows or the vocabulary grow; calls of fewer rows
    are taken with those of the most."""
    child = COMMON + r"""
size = L.dsv4_gpu_logits_scratch_bytes
prev = [0] * 65
for vocab in (1, 100, 1023, 1024, 1025, 2049, 32000, 129280, 200001):
    last = 0
    for nt in range(1, 65):
        n = size(nt, vocab)
        assert n >= last and n >= prev[nt], (nt, vocab, n, last, prev[nt])
        last = prev[nt] = n
    for nt in range(1, 65):
        for hist in (0, 100, 100000):
            r = D.LogitRules(hist=p, n_hist=hist, repetition=1.5)
            assert L.dsv4_gpu_logits_adjust_d(p, p, p, nt, vocab, vocab, ctypes.byref(r), p, last,
                                              None) == 0, (nt, vocab)
print("done")
"""
    assert hip_shim.run(tmp_path, child).endswith("done\n")
