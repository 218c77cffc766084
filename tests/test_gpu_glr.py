"""The gated linear recurrence (hiertcn_amd/glr.py, csrc/glr.hip) against its 64-bit restatement, step by step."""
import numpy as np
import pytest
import torch

from oracle import sequence_oracle as SO

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}    # half a step of the output's type
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}              # ... near its zero


def inputs(B, T, D, dtype, seed=0, ragged=True, resets=True, layout="halves"):
    rng = np.random.default_rng(seed)
    gate = np.clip(rng.standard_normal((B, T, D)) + 1.5, -8, 8)
    cand = np.clip(rng.standard_normal((B, T, D)), -8, 8)
    to = lambda v: torch.tensor(v, dtype=torch.float32).to(dtype).cuda()  # noqa: E731
    g, x = to(gate), to(cand)
    if layout == "halves":
        p = torch.cat([g, x], -1)
        g, x = p[..., :D], p[..., D:]
    elif layout == "time_major":
        g, x = (v.transpose(0, 1).contiguous().transpose(0, 1) for v in (g, x))
    elif layout == "shifted":          # addresses that allow one element at a time only
        p = torch.empty(B * T * D + 1, dtype=dtype, device="cuda")
        p[1:] = g.reshape(-1)
        g = p[1:].view(B, T, D)
    dh, state, ds = to(rng.standard_normal((B, T, D))), torch.tensor(rng.standard_normal((B, D)), dtype=torch.float32).cuda(), torch.tensor(rng.standard_normal((B, D)), dtype=torch.float32).cuda()
    lens = rng.integers(0, T + 1, B)
    if B > 2:
        lens[:3] = [0, T, min(1, T)]
    lengths = torch.tensor(lens, dtype=torch.int32).cuda() if ragged else None
    mask = torch.tensor((rng.random((B, T)) > 0.1), dtype=torch.float32).cuda() if resets else None
    return g, x, dh, state, ds, mask, lengths


def reference(g, x, state, mask, lengths, act, dh=None, ds=None):
    n = lambda t: None if t is None else t.double().cpu().numpy()  # noqa: E731
    return SO.glr(n(g), n(x), n(state), n(mask), None if lengths is None else lengths.cpu().numpy(), act, n(dh), n(ds))


def close(got, ref, name, dtype):
    want, err = ref[name], ref[name + "_err"]
    d = np.abs(got.double().cpu().numpy() - want)
    allowed = err * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + TINY[dtype]
    bad = d > allowed
    assert not bad.any(), (name, int(bad.sum()), float((d / allowed).max()), np.argwhere(bad)[:3].tolist())


def check(g, x, dh, state, ds, mask, lengths, act):
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    h, s, rec = glr_scan(g, x, state, mask=mask, lengths=lengths, cand_act=act, want_record=True)
    h2, s2, _ = glr_scan(g, x, state, mask=mask, lengths=lengths, cand_act=act)
    assert torch.equal(h, h2) and torch.equal(s, s2)
    dproj = torch.full((*g.shape[:2], 2 * g.shape[2]), 7.0, dtype=g.dtype, device="cuda")
    D = g.shape[2]
    dg, dx, d0 = glr_scan_backward(g, x, dh, rec, mask=mask, lengths=lengths, cand_act=act, dstate_out=ds, dgate=dproj[..., :D], dcand=dproj[..., D:])
    ref = reference(g, x, state, mask, lengths, act, dh, ds)
    close(h, ref, "h", g.dtype)
    close(s, ref, "state", torch.float32)
    close(dg, ref, "dgate", g.dtype)
    close(dx, ref, "dcand", g.dtype)
    close(d0, ref, "dstate", torch.float32)


SHAPES = [(1, 1, 1), (3, 1, 64), (5, 7, 130), (2, 8, 96), (4, 9, 33), (3, 257, 64), (33, 40, 70), (2, 1031, 66), (1, 2500, 5), (600, 24, 128), (7, 513, 200)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, dtype):
    check(*inputs(*shape, dtype, seed=sum(shape)), "tanh" if shape[1] % 2 else "none")


@pytest.mark.parametrize("layout", ["halves", "time_major", "shifted", "plain"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(layout, dtype):
    check(*inputs(4, 70, 64, dtype, seed=3, layout=layout), "tanh")


@pytest.mark.parametrize("ragged,resets", [(False, False), (True, False), (False, True)])
def test_without_lengths_or_resets(ragged, resets):
    check(*inputs(4, 300, 66, torch.float32, seed=5, ragged=ragged, resets=resets), "tanh")


@pytest.mark.parametrize("shape", [(1, 40000, 64), (2, 16411, 130)], ids=str)
def test_a_long_time_axis_over_many_workgroups(shape):
    check(*inputs(*shape, torch.float32, seed=9, ragged=shape[0] > 1), "none")


def test_many_lanes():
    check(*inputs(3000, 12, 192, torch.bfloat16, seed=11), "tanh")


def test_the_gradient_against_differences_of_the_definition():
    """d loss along a direction, from the definition in 64 bits alone, against the kernel's gradients."""
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    g, x, dh, state, ds, mask, lengths = inputs(3, 45, 34, torch.float32, seed=21)
    _, _, rec = glr_scan(g, x, state, mask=mask, lengths=lengths, want_record=True)
    dg, dx, d0 = glr_scan_backward(g, x, dh, rec, mask=mask, lengths=lengths, dstate_out=ds)
    n = lambda t: t.double().cpu().numpy()  # noqa: E731
    rng = np.random.default_rng(1)
    dirs = [rng.standard_normal(n(v).shape) for v in (g, x, state)]
    step = 1e-5

    def loss(k):
        r = SO.glr(n(g) + k * dirs[0], n(x) + k * dirs[1], n(state) + k * dirs[2], n(mask), lengths.cpu().numpy(), "tanh")
        return (r["h"] * n(dh)).sum() + (r["state"] * n(ds)).sum()

    num = (loss(step) - loss(-step)) / (2 * step)
    ana = (n(dg) * dirs[0]).sum() + (n(dx) * dirs[1]).sum() + (n(d0) * dirs[2]).sum()
    # the kernel's elements are within their bounds (1e-5 of their size, test_forward_and_backward); differences: step^2 and 2^-52 / step of sums of ~1e2
    scale = np.sqrt((n(dg) ** 2).sum() + (n(dx) ** 2).sum() + (n(d0) ** 2).sum())
    assert abs(num - ana) < 1e-4 * scale, (num, ana)


def test_steps_equal_the_scan():
    """Serving: one step after the other, in place, with lanes that drop out -- the same states as the scan to its bound."""
    from hiertcn_amd.glr import glr_step
    B, T, D = 6, 19, 128
    g, x, _, state, _, mask, lengths = inputs(B, T, D, torch.bfloat16, seed=31)
    ref = reference(g, x, state, mask, lengths, "tanh")
    s = state.clone()
    for t in range(T):
        h, s2 = glr_step(g[:, t], x[:, t], s, mask=mask[:, t].contiguous(), active=(lengths > t).to(torch.int32), state_out=s)
        assert s2 is s
        d = np.abs(h.double().cpu().numpy() - ref["h"][:, t])
        assert (d <= ref["h_err"][:, t] * 2 + HALF[torch.bfloat16] * np.abs(ref["h"][:, t]) + 1e-37).all(), t
    close(s, ref, "state", torch.float32)


def test_in_place_state_of_a_split_time_axis():
    from hiertcn_amd.glr import glr_scan
    g, x, _, state, _, mask, lengths = inputs(1, 30000, 64, torch.float32, seed=41, ragged=False)
    h, s, _ = glr_scan(g, x, state, mask=mask)
    mine = state.clone()
    h2, s2, _ = glr_scan(g, x, mine, mask=mask, state_out=mine)
    assert s2 is mine and torch.equal(mine, s) and torch.equal(h, h2)


@pytest.mark.parametrize("T", [5, 300, 20000])
def test_nan_and_infinity(T):
    """Behind a sequence's end nothing is read; a reset cuts a state that is NaN or infinite; nothing else does, however small the gates' product."""
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    B, D = 3, 64
    g, x, dh, state, ds, _, _ = inputs(B, T, D, torch.float32, seed=51, ragged=False, resets=False)
    n = T // 2
    lengths = torch.tensor([n, T, T], dtype=torch.int32, device="cuda")
    clean = glr_scan(g, x, state, lengths=lengths, want_record=True)
    cg = glr_scan_backward(g, x, dh, clean[2], lengths=lengths, dstate_out=ds)
    g2, x2, dh2 = g.clone(), x.clone(), dh.clone()
    for v in (g2, x2, dh2):
        v[0, n:] = float("nan")
    out = glr_scan(g2, x2, state, lengths=lengths, want_record=True)
    og = glr_scan_backward(g2, x2, dh2, out[2], lengths=lengths, dstate_out=ds)
    assert all(torch.equal(a, b) for a, b in zip(out[:2] + og, clean[:2] + cg))
    assert (out[0][0, n:] == 0).all() and (og[0][0, n:] == 0).all()
    # a reset at step 2 of lane 1 cuts the NaN state, lane 2 keeps it to the end although its gates are all but closed
    bad = state.clone()
    bad[1:] = float("nan")
    bad[1, 1] = float("inf")
    mask = torch.ones(B, T, device="cuda")
    mask[1, 2] = 0
    shut = g.clone()
    shut[2] = -30.0
    h, s, _ = glr_scan(shut, x, bad, mask=mask)
    assert torch.isnan(h[2]).all() and torch.isnan(s[2]).all()
    assert not torch.isfinite(h[1, :2]).any() and torch.isfinite(h[1, 2:]).all() and torch.isfinite(s[1]).all()


def test_lengths_outside_the_range_are_clamped():
    from hiertcn_amd.glr import glr_scan
    g, x, _, state, _, _, _ = inputs(3, 11, 16, torch.float32, seed=61)
    a = glr_scan(g, x, state, lengths=torch.tensor([-5, 400, 3], dtype=torch.int32, device="cuda"))
    b = glr_scan(g, x, state, lengths=torch.tensor([0, 11, 3], dtype=torch.int32, device="cuda"))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[1][0], state[0]) and (a[0][0] == 0).all()


def test_empty_calls():
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    e = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    s0 = torch.randn(3, 8, device="cuda")
    h, s, rec = glr_scan(e(3, 0, 8), e(3, 0, 8), s0, want_record=True)
    assert h.shape == (3, 0, 8) and torch.equal(s, s0)
    _, _, d0 = glr_scan_backward(e(3, 0, 8), e(3, 0, 8), e(3, 0, 8), rec, dstate_out=s0)
    assert torch.equal(d0, s0)
    assert (glr_scan(e(3, 0, 8), e(3, 0, 8))[1] == 0).all() and glr_scan(e(0, 5, 8), e(0, 5, 8))[1].shape == (0, 8)


def test_broadcast_inputs():
    """Gates that all lanes share (stride 0) are read as they are; the gradient of each use comes back, for the caller to sum."""
    check_g = torch.randn(1, 20, 64, device="cuda")
    g = check_g.expand(4, 20, 64)
    _, x, dh, state, ds, mask, lengths = inputs(4, 20, 64, torch.float32, seed=71)
    check(g, x, dh, state, ds, mask, lengths, "tanh")


def test_graph_replays_and_another_stream():
    """A captured forward + backward replayed with new data, eager calls of other shapes between the replays, and a second graph beside it."""
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    args = inputs(4, 500, 64, torch.bfloat16, seed=81)
    args2 = inputs(1, 20000, 64, torch.bfloat16, seed=82)

    def step(a):
        g, x, dh, state, ds, mask, lengths = a
        h, s, rec = glr_scan(g, x, state, mask=mask, lengths=lengths, want_record=True)
        return (h, s, *glr_scan_backward(g, x, dh, rec, mask=mask, lengths=lengths, dstate_out=ds))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [v.clone() for v in step(args)]
        step(args2)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in (args, args2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(a))
        graphs.append(gr)
    for k in range(3):
        for gr in graphs:
            gr.replay()
        step(inputs(2, 40 + k, 32, torch.float32, seed=k))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[0], eager))
        assert all(torch.equal(a, b) for a, b in zip(outs[1], step(args2)))
        args[0].copy_(args[0] * 0.9)
        eager = [v.clone() for v in step(args)]


def test_offsets_behind_2_to_the_32():
    """B * T * D > 2^32 elements: the rows behind it are computed like any other."""
    from hiertcn_amd.glr import glr_scan
    B, T, D = 5, 1 << 20, 1024
    g = torch.empty(B, T, D, dtype=torch.bfloat16, device="cuda")
    assert g.numel() > 2 ** 32
    part = torch.randn(1, 1, D, device="cuda")
    g.copy_(part)
    x = torch.ones(1, 1, D, dtype=torch.bfloat16, device="cuda").expand(B, T, D)
    state = torch.zeros(B, D, device="cuda")
    h, s, _ = glr_scan(g, x, state, cand_act="none", lengths=torch.tensor([1, 2, 3, 4, T], dtype=torch.int32, device="cuda"))
    assert (h[4, T - 1] - 1).abs().max() < 1e-2 and (s[4] - 1).abs().max() < 1e-4 and (h[3, 4:1000] == 0).all() and (h[3, T - 1] == 0).all()
    tail = glr_scan(g[4:, :40], x[4:, :40], state[4:], cand_act="none")[0]
    assert torch.equal(h[4, :40], tail[0])


def test_a_wait_that_cannot_be_met_gives_up():
    """Long recurrences hand states from workgroup to workgroup; with words that never come (tests/tools/glr_wait_probe.py, the test-hooks build) the launch ends and
    what could not be learnt is NaN."""
    import os
    import subprocess
    import sys
    from hiertcn_amd.build import LIB_TESTHOOKS
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "tests", "tools", "glr_wait_probe.py")], env=dict(os.environ, HIERTCN_LIB=LIB_TESTHOOKS), capture_output=True, text=True,
                       timeout=110)
    assert r.returncode == 0 and "glr_wait_probe ok" in r.stdout, r.stdout[-2000:] + r.stderr[-4000:]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(3, 50, 64), (1, 3000, 64), (700, 6, 128)], ids=str)
def test_gradients_of_saturated_candidates(shape, dtype):
    """|cand| of 5 to 20: the slope of tanh there is 2e-4 to 2e-17 and the gradient as exact, relative to itself, as anywhere."""
    g, x, dh, state, ds, mask, lengths = inputs(*shape, dtype, seed=91)
    size = 5 + 15 * torch.rand(x.shape, generator=torch.Generator().manual_seed(4))
    x = torch.where(torch.rand(x.shape, generator=torch.Generator().manual_seed(5)) < 0.5, -size, size).to(dtype).cuda()
    check(g, x, dh, state, ds, mask, lengths, "tanh")


@pytest.mark.parametrize("shape", [(3, 40, 64), (1, 2000, 64), (700, 6, 128)], ids=str)
@pytest.mark.parametrize("size", [8, 30, 80])
def test_gates_far_open_and_shut(size, shape):
    """fp32 gates of up to +-80: the small one of u and 1 - u is as exact, relative to itself, as the other.  (Its exponential is within 3 half steps + 1/20 of |x|; 1 + e,
    the reciprocal, the product: 5 more, 12 in all at |gate| = 80; the bound counts 16.)"""
    g, x, dh, state, ds, mask, lengths = inputs(*shape, torch.float32, seed=93)
    g = (size * (2 * torch.rand(g.shape, generator=torch.Generator().manual_seed(size)) - 1)).cuda()
    check(g, x, dh, state, ds, mask, lengths, "tanh")


@pytest.mark.parametrize("resets", [False, True])
@pytest.mark.parametrize("T", [12, 300, 20000])
def test_an_infinite_state_stays_infinite(T, resets):
    """Gates of 1e-13 all along (16 of them multiply to less than fp32 holds): h = u inf + (1 - u) c is infinite at every step, forward and backward, until a reset."""
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    B, D = 2, 64
    g, x, dh, state, ds, _, _ = inputs(B, T, D, torch.float32, seed=95, ragged=False, resets=False)
    g = torch.full_like(g, -30.0)
    mask = torch.ones(B, T, device="cuda") if resets else None
    if resets:
        mask[1, T - 3] = 0
    bad, dbad = state.clone(), ds.clone()
    bad[:, ::2], dbad[:, 1::2] = float("inf"), float("-inf")
    h, s, rec = glr_scan(g, x, bad, mask=mask, want_record=True)
    rows = h[1, :T - 3] if resets else h[1]
    assert torch.isposinf(h[0, :, ::2]).all() and torch.isposinf(s[0, ::2]).all() and torch.isposinf(rows[:, ::2]).all() and torch.isfinite(h[:, :, 1::2]).all()
    if resets:
        assert torch.isfinite(h[1, T - 3:]).all() and torch.isfinite(s[1]).all()
    _, dx, d0 = glr_scan_backward(g, x, dh, glr_scan(g, x, state, mask=mask, want_record=True)[2], mask=mask, dstate_out=dbad)
    assert torch.isneginf(dx[0, :, 1::2]).all() and torch.isneginf(d0[0, 1::2]).all() and torch.isfinite(dx[:, :, ::2]).all()
    if resets:
        assert torch.isneginf(dx[1, T - 3:, 1::2]).all() and torch.isfinite(dx[1, :T - 3]).all() and torch.isfinite(d0[1]).all()


# Two channels a lane from 8192 waves on (B * ceil(D / 128) * ceil(T / 16)): one wave a sequence; several tiles of waves one behind the other; chained workgroups.
WIDE = [(2100, 64, 128, 60), (310, 450, 130, 14), (2, 33000, 256, 1)]


FORMS = [("tanh", True), ("none", False), ("tanh", False), ("none", True)]


@pytest.mark.parametrize("shape,act,resets", [(s, *f) for s in WIDE for f in FORMS[:2 if s[1] > 1000 else 4]], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_two_channels_a_lane(shape, dtype, act, resets):
    """Every `every`-th sequence against 64 bits; the others against the same sequences called by themselves (one channel a lane), to both calls' bounds."""
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    B, T, D, every = shape
    assert B * -(-D // 128) * -(-T // 16) >= 8192
    g, x, dh, state, ds, mask, lengths = inputs(B, T, D, dtype, seed=T, resets=resets)
    h, s, rec = glr_scan(g, x, state, mask=mask, lengths=lengths, cand_act=act, want_record=True)
    dg, dx, d0 = glr_scan_backward(g, x, dh, rec, mask=mask, lengths=lengths, cand_act=act, dstate_out=ds)
    pick = torch.arange(0, B, every, device="cuda")
    of = lambda v: None if v is None else v[pick]  # noqa: E731
    ref = reference(of(g), of(x), of(state), of(mask), of(lengths), act, of(dh), of(ds))
    for got, name, dt in ((h, "h", dtype), (s, "state", torch.float32), (dg, "dgate", dtype), (dx, "dcand", dtype), (d0, "dstate", torch.float32)):
        close(got[pick], ref, name, dt)
    assert torch.isfinite(h.float()).all() and torch.isfinite(rec).all()
    if T < 1000:
        n = 8192 // (-(-D // 128) * -(-T // 16)) // 2       # few enough for one channel a lane
        for at in range(0, B - n, 3 * n):
            cut = slice(at, at + n)
            one = glr_scan(g[cut], x[cut], state[cut], mask=None if mask is None else mask[cut], lengths=None if lengths is None else lengths[cut], cand_act=act)
            # |h| <= max |c|, |state| <= 8.  A step adds at most 19 half steps of fp32 of that (the oracle's EPS_GATE + 3 EPS) and 16 of c's, and gates of at most 1 let no
            # earlier error grow: both calls are within 35 T half steps of 8, and a rounding of the type
            off = 2 * 35 * T * HALF[torch.float32] * 8
            assert (one[0].double() - h[cut].double()).abs().max() <= off + 2 * HALF[dtype] * 8
            assert (one[1] - s[cut]).abs().max() <= off
