"""The operators on drafted tokens at the most rows that their calls may name.
CPU only: nothing is launched."""
import hip_shim

# the launches' dimensions, which the shim lets go
GRIDS = r"""
static double most_threads;
static long long groups;
void shim_grids(double *t, long long *g)
{
    *t = most_threads; *g = groups;
    most_threads = 0; groups = 0;
}
int __hipPushCallConfiguration(D3 g, D3 b, size_t l, void *s)
{
    const double x = (double)g.x * b.x, y = (double)g.y * b.y;
    (void)l; (void)s;
    if (x > most_threads) most_threads = x;
    if (y > most_threads) most_threads = y;
    groups += (long long)g.x * g.y;
    return 0;
}
"""

CHILD = r"""
buf = np.zeros(1 << 12, np.uint8)
p = (buf.ctypes.data + 255) // 256 * 256                     # nothing reads it
assert L.dsv4_gpu_init() == 0


def grids():
    t, g = ctypes.c_double(), ctypes.c_longlong()
    shim.shim_grids(ctypes.byref(t), ctypes.byref(g))
    return t.value, g.value


rope = D.Rope(cos=p, sin=p, max_pos=8, dim=2, offset=0, layout=0)
MOST = 1 << 30
for n in (1, 4096, 4097, 100000, (1 << 26) - 1, 1 << 26, (1 << 26) + 5, MOST - 1, MOST):
    for at in (None, p):
        shim.shim_reset(-1, 0)
        grids()
        assert L.dsv4_gpu_kv_append_d(p, p, 2, 8, MOST, p, 0, 8, n, 8, at, 0, None, None, None) == 0
        # a dimension of a launch has fewer than 2^32 threads
        t, g = grids()
        assert t < 2.0 ** 32, ("append", n, t)
        # and a list costs each of its workgroups no more than 2^17 entries: not the square
        # of what the call may name
        if at and n > 1 << 17:
            assert shim.shim_launches() >= n >> 17, ("append", n, shim.shim_launches())
        shim.shim_reset(-1, 0)
        assert L.dsv4_gpu_kv_read_d(p, 0, 8, p, p, 2, 8, MOST, at, 0, n, 8, None) == 0
        assert grids()[0] < 2.0 ** 32, ("read", n)
    shim.shim_reset(-1, 0)
    assert L.dsv4_gpu_rope_n_d(p, 8, p, 8, 0, p, n, 1, 8, ctypes.byref(rope), 0, None) == 0
    assert grids()[0] < 2.0 ** 32, ("rope", n)
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


EMPTY = r"""
p = np.zeros(64, np.uint8).ctypes.data
assert L.dsv4_gpu_init() == 0
rope = D.Rope(cos=p, sin=p, max_pos=8, dim=2, offset=0, layout=0)
rules = D.LogitRules(repetition=1.0)
calls = {                                                    # (of 0, with a wrong size or rule)
    "dsv4_gpu_rope_n_d": [(None, 8, None, 8, 0, None, 0, 1, hd, ctypes.byref(rope), 0, None)
                          for hd in (8, 1)],
    "dsv4_gpu_kv_append_d": [(None, None, 2, 8, 4, None, 0, 8, 0, 8, None, row0,
                              ctypes.byref(rope), None, None) for row0 in (4, 5)],
    "dsv4_gpu_kv_read_d": [(None, 0, 8, None, None, 2, 8, 4, None, row0, 0, 8, None)
                           for row0 in (4, 5)],
    "dsv4_gpu_tree_attn_d": [(None, None, 0, 0, 1, 8, dv, None, None, 2, 8, 4, None, 0, 0, 3, None,
                              0, None, 1.0, None, 0, None) for dv in (8, 9)],
    "dsv4_gpu_logits_adjust_d": [(None, None, None, 0, 8, 8, r, None, 0, None)
                                 for r in (ctypes.byref(rules), None)],
}
for name, (good, bad) in calls.items():
    shim.shim_reset(-1, 0)
    assert getattr(L, name)(*good) == 0, name
    assert getattr(L, name)(*bad) == -1, name
    assert shim.shim_launches() == 0, name
print("done")
"""


def test_a_length_of_zero_needs_no_buffers(tmp_path):
    """Its sizes, types, ranges and rules are checked as ever."""
    assert hip_shim.run(tmp_path, EMPTY).endswith("done\n")
