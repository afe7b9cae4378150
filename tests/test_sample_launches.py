"""Launches of the sampling and of a batch's attention at the most rows and tokens that
their calls may name. CPU only: nothing is launched."""
import hip_shim
from test_draft_lengths import GRIDS

CHILD = r"""
buf = np.zeros(1 << 12, np.uint8)
p = (buf.ctypes.data + 255) // 256 * 256                     # nothing reads it
assert L.dsv4_gpu_init() == 0
BIG = 1 << 45


def grids():
    t, g = ctypes.c_double(), ctypes.c_longlong()
    shim.shim_grids(ctypes.byref(t), ctypes.byref(g))
    return t.value, g.value


rules = ctypes.byref(D.Sampling(temperature=p, top_k=p, top_p=p, min_p=p, u=p))
for n, vocab in ((1, 1), (65536, 129280), (65536, 1 << 18), (16383, 1 << 22), (16384, 1 << 22),
                 (16385, 1 << 22), (65536, 1 << 20), (65535, 1 << 22), (65536, 1 << 22)):
    for fmt in (0, 1):
        shim.shim_reset(-1, 0)
        grids()
        assert L.dsv4_gpu_sample_d(p, p, p, p, fmt, n, vocab, vocab, rules, p, BIG, None) == 0
        # a dimension of a launch has fewer than 2^32 threads
        t, g = grids()
        assert t < 2.0 ** 32, ("sample", n, vocab, t)
        # and each slice of 8192 logits and each row has its workgroup
        assert g == n * -(-vocab // 8192) + n, ("sample", n, vocab, g)
for h, tok in ((1, 1), (256, 1 << 20), (4096, 1 << 16)):
    r = ctypes.byref(D.Reqs(len=p, pages=p, first=p, n_req=4096, max_pages=1 << 20, page_rows=1 << 10,
                            max_tok=tok, n_prefix=64))
    for kv in (0, 1, 2):
        for fmt in (0, 1):
            shim.shim_reset(-1, 0)
            grids()
            assert L.dsv4_gpu_reqs_plan_d(p, BIG, r, fmt, h, 576, 512, kv, 0, None) == 0
            assert L.dsv4_gpu_reqs_attn_d(p, p, fmt, h, 576, 512, p, p, kv, 576, 8, r, p, BIG, 0, None,
                                          ctypes.c_float(1), p, BIG, None) == 0
            assert grids()[0] < 2.0 ** 32, ("attn", h, tok)
print("done")
"""


def test_launches_of_the_most_rows(tmp_path, monkeypatch):
    old = hip_shim.SOURCE.index("int __hipPushCallConfiguration")
    end = hip_shim.SOURCE.index("}\n", old) + 2
    source = hip_shim.SOURCE[:old] + GRIDS + hip_shim.SOURCE[end:]
    # these kernels have no second argument to keep
    keep = "    if (launches == 1) arg1 = *(void **)a[1];\n"
    assert keep in source
    monkeypatch.setattr(hip_shim, "SOURCE", source.replace(keep, "    (void)a;\n"))
    assert hip_shim.run(tmp_path, CHILD).endswith("done\n")
