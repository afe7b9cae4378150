"""A plan (dsv4_gpu_reqs_plan_d) serves the sizes, formats and window that it was made for,
and with any other dsv4_gpu_reqs_attn_d makes all of o NaN."""
import ctypes

import numpy as np
import pytest

import draft_common as dc
import reqs_common as rc

pytestmark = pytest.mark.gpu

MADE = dict(fmt=1, h=4, dqk=160, dv=100, kf=1, window=0, n_req=3, max_pages=6, page=16, max_tok=8,
            prefix=0)
OTHER = [dict(fmt=0), dict(h=3), dict(h=5), dict(dqk=256), dict(dqk=161), dict(dqk=300), dict(dqk=100),
         dict(dv=112), dict(dv=99), dict(dv=64), dict(kf=0), dict(kf=2), dict(window=9), dict(n_req=2),
         dict(max_pages=5), dict(page=8), dict(max_tok=7), dict(max_tok=9), dict(prefix=16)]


@pytest.mark.parametrize("other", range(-1, len(OTHER)))
def test_a_plan_of_other_sizes(gpu, dsv4, other):
    import torch
    L = dsv4.lib()
    now = dict(MADE, **(OTHER[other] if other >= 0 else {}))
    rows, width, most = 400, 304, 9              # room for every one of the sizes
    d = {k: dc.dev(np.asarray(v, np.int32)) for k, v in dict(
        len=[40, 50, 7], first=[0, 2, 5, 6], pages=np.arange(18).reshape(3, 6)).items()}

    def batch(m):
        return dsv4.Reqs(len=d["len"].data_ptr(), pages=d["pages"].data_ptr(),
                         first=d["first"].data_ptr(), n_req=m["n_req"], max_pages=m["max_pages"],
                         page_rows=m["page"], max_tok=m["max_tok"], n_prefix=m["prefix"])

    plan = torch.zeros(max(L.dsv4_gpu_reqs_plan_bytes(m["n_req"], m["max_tok"], m["h"])
                           for m in (MADE, now)), device="cuda:0", dtype=torch.uint8)
    space = torch.zeros(L.dsv4_gpu_reqs_attn_scratch_bytes(
        now["fmt"], now["h"], now["dqk"], now["dv"], now["kf"], now["n_req"], now["max_tok"]),
        device="cuda:0", dtype=torch.uint8)
    dt = torch.bfloat16 if now["fmt"] else torch.float32
    q = torch.randn(most, now["h"], now["dqk"], device="cuda:0").to(dt)
    x, scales = dc.stored(np.random.default_rng(1).standard_normal((rows, width)), now["kf"])
    cache, ks = dc.cache_of(x, now["kf"], scales=scales)
    o = torch.full((now["max_tok"] + 1, now["h"], now["dv"]), 99.0, device="cuda:0", dtype=dt)
    a = MADE
    assert L.dsv4_gpu_reqs_plan_d(plan.data_ptr(), plan.numel(), ctypes.byref(batch(a)), a["fmt"],
                                  a["h"], a["dqk"], a["dv"], a["kf"], a["window"], dc.stream()) == 0
    a = now
    assert L.dsv4_gpu_reqs_attn_d(
        o.data_ptr(), q.data_ptr(), a["fmt"], a["h"], a["dqk"], a["dv"], cache.data_ptr(), dc.ptr(ks),
        a["kf"], width, rows, ctypes.byref(batch(a)), plan.data_ptr(), plan.numel(), a["window"], None,
        ctypes.c_float(0.1), space.data_ptr(), space.numel(), dc.stream()) == 0
    torch.cuda.synchronize()
    got = dc.host(o)
    assert (got[a["max_tok"]:] == 99).all()
    if other < 0:
        assert np.isfinite(got).all() and (got[6:] == 99).all()
    else:
        assert np.isnan(got[:a["max_tok"]]).all(), OTHER[other]
