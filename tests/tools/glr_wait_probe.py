"""Run by tests/test_gpu_glr.py in a process of its own with HIERTCN_LIB = libhiertcn_gfx950_testhooks.so (the only build that reads HIERTCN_GLR_TEST_POLLS): the
workgroups of a chained recurrence publish nothing and look that often for each other's words.  Every launch ends, what depends on a word that never came is NaN,
everything else is what it always is, and the next call is as good as ever."""
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
import torch

from hiertcn_amd.glr import glr_scan, glr_scan_backward
from tests.test_gpu_glr import inputs

assert os.environ.get("HIERTCN_LIB", "").endswith("testhooks.so")
TILE = 128                  # steps of a chained tile, at least: eight segments of 16


def run(g, x, dh, state, ds, mask, record=None):
    h, s, rec = glr_scan(g, x, state, mask=mask, want_record=True)
    dg, dx, d0 = glr_scan_backward(g, x, dh, rec if record is None else record, mask=mask, dstate_out=ds)
    torch.cuda.synchronize()
    return h, s, rec, dg, dx, d0


for B, T, D, dtype in ((1, 40000, 64, torch.float32), (2, 40000, 256, torch.bfloat16)):      # one and two channels a lane
    for cut in (False, True):
        g, x, dh, state, ds, _, _ = inputs(B, T, D, dtype, seed=5, ragged=False, resets=False, layout="plain")
        mask = None
        if cut:                                                              # one reset near each end
            mask = torch.ones(B, T, device="cuda")
            mask[:, 20] = mask[:, T - 10] = 0
        want = run(g, x, dh, state, ds, mask)
        assert all(torch.isfinite(v.float()).all() for v in want)
        for polls in ("0", "200"):
            print("polls", polls, B, T, D, "cut" if cut else "", flush=True)
            os.environ["HIERTCN_GLR_TEST_POLLS"] = polls
            t0 = time.time()
            try:
                h, s, rec, dg, dx, d0 = run(g, x, dh, state, ds, mask, record=want[2])
            finally:
                os.environ.pop("HIERTCN_GLR_TEST_POLLS")
            assert time.time() - t0 < 20
            known = h[:, :TILE]
            assert torch.equal(known, want[0][:, :TILE]) and torch.isnan(h[:, T // 2]).all()
            assert torch.equal(dg[:, -8:], want[3][:, -8:]) and torch.equal(dx[:, -8:], want[4][:, -8:]) and torch.isnan(dx[:, T // 2]).all()
            if cut:         # behind the last reset (backward: in front of the first) nothing depends on the missing words
                assert torch.isnan(h[:, T - 11]).all() and torch.equal(h[:, T - 10:], want[0][:, T - 10:]) and torch.equal(s, want[1])
                assert torch.isnan(dx[:, 20]).all() and torch.equal(dx[:, :20], want[4][:, :20]) and torch.equal(d0, want[5])
            else:
                assert torch.isnan(h[:, -1]).all() and torch.isnan(s).all() and torch.isnan(dx[:, 0]).all() and torch.isnan(d0).all()
            again = run(g, x, dh, state, ds, mask)
            assert all(torch.equal(a, b) for a, b in zip(again, want))
print("glr_wait_probe ok")
