"""AdamW over many tensors (hiertcn_amd/adamw.py, csrc/adamw.hip): 32-bit states against the formula in 64 bits, 8-bit states to the bit against the same single
fp32 operations in NumPy."""
import numpy as np
import pytest
import torch

from oracle import sequence_oracle as SO

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
B1, B2, E = 0.9, 0.999, 1e-8
SIZES = [1, 3, 255, 256, 257, 1000, 4096, 70001]


def tensors(sizes, seed, gdtype=torch.float32, offset=0):
    rng = np.random.default_rng(seed)

    def one(k, scale, dt=torch.float32):
        buf = torch.empty(k + offset, dtype=dt, device="cuda")
        buf[offset:] = torch.tensor(scale * rng.standard_normal(k), dtype=torch.float32).to(dt)
        return buf[offset:]
    return [one(k, 0.1) for k in sizes], [one(k, 0.01, gdtype) for k in sizes], rng


@pytest.mark.parametrize("gdtype,offset", [(torch.float32, 0), (torch.bfloat16, 0), (torch.float16, 0), (torch.float32, 1), (torch.bfloat16, 3)])
def test_32_bit_states(gdtype, offset):
    from hiertcn_amd.adamw import AdamW
    params, grads, rng = tensors(SIZES, 1, gdtype, offset)
    copies = [p.to(torch.bfloat16 if i % 2 else torch.float16) if i != 3 else None for i, p in enumerate(params)]
    decay = [0.1 * (i % 3) for i in range(len(SIZES))]
    opt = AdamW(params, lr=3e-3, betas=(B1, B2), eps=E, weight_decay=decay, copies=copies)
    ref = [(p.double().cpu().numpy(), np.zeros(k), np.zeros(k)) for p, k in zip(params, SIZES)]
    err = [(np.zeros(k), np.zeros(k), np.zeros(k)) for k in SIZES]
    for t in range(1, 6):
        gs = 0.5 if t % 2 else torch.tensor([0.25], device="cuda")
        opt.step(grads, lr=3e-3 * t, grad_scale=gs)
        for i, g in enumerate(grads):
            gn = g.double().cpu().numpy() * float(gs)
            p, m, v = ref[i]
            ep, em, ev = err[i]
            # fp32: constants, products and sums are half a step off each; the update m / (sqrt(v) c + eps) carries the errors of both states
            lr = 3e-3 * t
            p2, m2, v2 = SO.adamw64(p, gn, m, v, t, lr, B1, B2, E, float(np.float32(decay[i])))
            em = B1 * em + 3 * EPS * (np.abs(B1 * m) + np.abs(0.1 * gn)) + EPS * np.abs(m2)
            ev = B2 * ev + 3 * EPS * np.abs(B2 * v) + 4 * EPS * 0.001 * gn ** 2 + EPS * v2
            root = np.sqrt(v2 / (1 - B2 ** t)) + E
            upd = lr / (1 - B1 ** t) * m2 / root
            with np.errstate(all="ignore"):
                rel = np.where(v2 > 0, 0.5 * ev / v2, 0) + 8 * EPS
            ep = ep + 2 * EPS * np.abs(p) + np.abs(upd) * rel + lr / (1 - B1 ** t) * em / root + EPS * np.abs(p2)
            ref[i], err[i] = (p2, m2, v2), (ep, em, ev)
    assert opt.t == 5
    for i in range(len(SIZES)):
        for got, want, e, name in zip((params[i], opt.m[i], opt.v[i]), ref[i], err[i], "pmv"):
            d = np.abs(got.double().cpu().numpy() - want)
            assert (d <= 1.01 * e + 1e-37).all(), (name, i, float((d / (e + 1e-37)).max()))
        if copies[i] is not None:
            assert torch.equal(copies[i], params[i].to(copies[i].dtype))


@pytest.mark.parametrize("gdtype,offset", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 0)])
def test_8_bit_states_to_the_bit(gdtype, offset):
    from hiertcn_amd.adamw import AdamW
    sizes = SIZES + [5, 0, 300]
    params, grads, rng = tensors(sizes, 2, gdtype, offset)
    grads[5].zero_()                       # a tensor that never gets a gradient
    grads[6][:256] = 1e-30                 # a block below the smallest scale
    opt = AdamW(params, grads, lr=1e-2, betas=(B1, B2), eps=E, weight_decay=0.05, state_bits=8, seed=77)
    host = [(p.cpu().numpy(), np.zeros(k, np.int8), np.zeros(k, np.uint8), np.zeros(-(-k // 256), np.float32), np.zeros(-(-k // 256), np.float32)) for p, k in zip(params, sizes)]
    for t in range(1, 8):
        for g in grads:
            g.mul_(-0.7)
        opt.step()
        for i, g in enumerate(grads):
            p, qm, qv, sm, sv = host[i]
            if p.size:
                host[i] = SO.adamw8(p, g.float().cpu().numpy(), qm, qv, sm, sv, t, 1e-2, B1, B2, E, 0.05, 77, i)
        for i in range(len(sizes)):
            p, qm, qv, sm, sv = host[i]
            for name, got, want in (("m", opt.m[i], qm), ("v", opt.v[i], qv), ("m_scale", opt.m_scale[i], sm), ("v_scale", opt.v_scale[i], sv)):
                assert np.array_equal(got.cpu().numpy(), want), (t, i, name, np.argwhere(got.cpu().numpy() != want)[:4].tolist())
            # (the division of the update may be contracted on neither side: equal up to its last step)
            assert (np.abs(params[i].cpu().numpy() - p) <= 4 * EPS * (np.abs(p) + 1e-2)).all(), (t, i)
    m, v = opt.moments()
    for i in range(len(sizes)):
        if sizes[i]:
            assert np.array_equal(m[i].cpu().numpy(), SO.decode(host[i][1], host[i][3], False)) and np.array_equal(v[i].cpu().numpy(), SO.decode(host[i][2], host[i][4], True))
    assert (opt.m[5] == 0).all() and (opt.v[5] == 0).all() and (opt.m_scale[6][0] == 0)


def test_more_tensors_than_a_launch_takes():
    from hiertcn_amd.adamw import AdamW
    params, grads, _ = tensors([1 + 37 * i for i in range(130)], 3)
    some = [None if i % 11 == 0 else g for i, g in enumerate(grads)]
    before = [p.clone() for p in params]
    AdamW(params, some, lr=1e-3).step()
    for i, (p, b, g) in enumerate(zip(params, before, grads)):
        if i % 11 == 0:
            assert torch.equal(p, b)
        else:       # the first step moves by lr * sign(g), to fp32
            assert (p - (b - 1e-3 * g / (g.abs() + 1e-8))).abs().max() < 1e-6


def test_state_round_trip_and_determinism():
    from hiertcn_amd.adamw import AdamW
    for bits in (8, 32):
        params, grads, _ = tensors([1000, 333], 5)
        a = AdamW(params, grads, lr=1e-3, state_bits=bits, seed=5)
        for _ in range(3):
            a.step()
        twin = [p.clone() for p in params]
        b = AdamW(twin, grads, lr=1e-3, state_bits=bits)
        b.load_state_dict(a.state_dict())
        for _ in range(3):
            a.step()
            b.step()
        assert a.t == b.t == 6 and all(torch.equal(x, y) for x, y in zip(params + a.m + a.v, twin + b.m + b.v))


def test_nan_gradient_stays_in_its_block():
    from hiertcn_amd.adamw import AdamW
    params, grads, _ = tensors([1024], 7)
    opt = AdamW(params, grads, state_bits=8)
    opt.step()
    grads[0][300] = float("nan")
    opt.step()
    m, v = opt.moments()
    assert torch.isnan(params[0][300]) and torch.isfinite(params[0][:300]).all() and torch.isfinite(params[0][301:]).all()
    assert not torch.isfinite(m[0][256:512]).any() and torch.isfinite(m[0][:256]).all() and torch.isfinite(v[0][512:]).all()


def test_a_captured_step_is_refused():
    from hiertcn_amd._lib import HierTCNError
    from hiertcn_amd.adamw import AdamW
    params, grads, _ = tensors([1000], 9)
    opt = AdamW(params, grads)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(HierTCNError, match="captured"):
        with torch.cuda.graph(graph):
            params[0].add_(0.0)
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert opt.t == 2


def test_8_bit_states_follow_32_bit_ones():
    """Gradients of constant size: v tends to g^2.  A step of v is narrower than its codes (4 / q >= 1.6 %), so rounding to nearest would hold it where it
    is; with the expectation kept it arrives: the mean of 2560 within 1 % (they scatter by less than a code, 2.7 %, each), each within four codes."""
    from hiertcn_amd.adamw import AdamW
    k = 64 * 40
    g = (torch.rand(k, device="cuda") + 0.5) * 1e-2
    p = torch.zeros(k, device="cuda")
    opt = AdamW([p], [g], lr=1e-6, state_bits=8, seed=1)
    for _ in range(3000):
        opt.step()
    _, v = opt.moments()
    ratio = (v[0] / (g * g * (1 - B2 ** 3000))).double()
    assert abs(float(ratio.mean()) - 1) < 0.01 and float((ratio - 1).abs().max()) < 0.11, (float(ratio.mean()), float(ratio.min()), float(ratio.max()))


def test_the_same_tensor_twice_is_refused():
    from hiertcn_amd._lib import HierTCNError
    from hiertcn_amd.adamw import AdamW
    p = [torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")]
    half = torch.zeros(100, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(HierTCNError, match="overlap"):
        AdamW([p[0], p[0]])
    with pytest.raises(HierTCNError, match="overlap"):
        AdamW(p, copies=[half, half])
    opt = AdamW(p)
    with pytest.raises(HierTCNError, match="overlap"):
        opt.set_state([opt.m[0], opt.m[0]], opt.v, 0)


def test_elements_behind_2_to_the_32():
    """A tensor of 2^32 + 700 elements: its last blocks and its first ones step as the formula says, and their random bits take the high word of the index."""
    from hiertcn_amd.adamw import AdamW
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("60 GiB of device memory")
    n, tail, lr = 2 ** 32 + 700, 956, 1e-2
    p = torch.full((n,), 0.5, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    rng = np.random.default_rng(4)
    ends = torch.tensor(rng.standard_normal((2, tail)), dtype=torch.float32).to(torch.bfloat16)
    g[:tail], g[n - tail:] = ends[0].cuda(), ends[1].cuda()
    opt = AdamW([p], [g], lr=lr, betas=(B1, B2), eps=E, state_bits=8, seed=9)
    opt.step()
    opt.step()
    start = n - tail                                       # a multiple of 256: whole blocks, on both sides of 2^32
    assert start % 256 == 0 and start < 2 ** 32 < n
    for at, grad in ((0, ends[0]), (start, ends[1])):
        q = np.full(tail, 0.5, np.float32)
        qm, qv, blocks = np.zeros(tail, np.int8), np.zeros(tail, np.uint8), -(-tail // 256)
        sm, sv = np.zeros(blocks, np.float32), np.zeros(blocks, np.float32)
        for t in (1, 2):
            whole = SO.mix
            try:                                           # the oracle's bits of elements at .. at + tail - 1
                SO.mix = lambda numel, tensor, t, seed, at=at: _bits(at + np.arange(numel, dtype=np.uint64), t, seed)
                q, qm, qv, sm, sv = SO.adamw8(q, grad.float().numpy(), qm, qv, sm, sv, t, lr, B1, B2, E, 0.0, 9, 0)
            finally:
                SO.mix = whole
        b0 = at // 256
        for got, want in ((opt.m[0][at:at + tail], qm), (opt.v[0][at:at + tail], qv), (opt.m_scale[0][b0:b0 + blocks], sm), (opt.v_scale[0][b0:b0 + blocks], sv)):
            assert np.array_equal(got.cpu().numpy(), want), at
        assert (np.abs(p[at:at + tail].cpu().numpy() - q) <= 4 * EPS * (np.abs(q) + 1e-2)).all()
    assert (p[tail:start] == 0.5).all()


def _bits(e, t, seed):
    u = np.uint32
    with np.errstate(over="ignore"):
        key = u((seed * 0x9E3779B1 + t * 0x6A09E667) & 0xFFFFFFFF) + (e >> np.uint64(32)).astype(u) * u(0x1F83D9AB)
        x = e.astype(u) * u(0x9E3779B1) + key
        x = (x ^ (x >> u(16))) * u(0x3C6EF373)
        x = (x ^ (x >> u(15))) * u(0x510E527F)
        return x ^ (x >> u(16))


def test_states_of_the_callers_own():
    from hiertcn_amd._lib import HierTCNError
    from hiertcn_amd.adamw import AdamW
    params, grads, _ = tensors([300, 7], 12)
    twin = [p.clone() for p in params]
    m, v = ([torch.zeros_like(p) for p in params] for _ in range(2))
    a, b = AdamW(params, grads, state=(m, v)), AdamW(twin, grads)
    for _ in range(2):
        a.step()
        b.step()
    assert all(torch.equal(x, y) for x, y in zip(params + m + v, twin + b.m + b.v)) and a.m[0] is m[0]
    with pytest.raises(HierTCNError):
        AdamW(params, grads, state=(m, v), state_bits=8)
    with pytest.raises(HierTCNError):
        AdamW(params, grads, state=(m[:1], v))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_refused_binding_leaves_the_optimizer_as_it_was(bits):
    """Gradients or states that are refused half-way: the next step works on the ones from before, not on a part of the refused ones."""
    from hiertcn_amd._lib import HierTCNError
    from hiertcn_amd.adamw import AdamW
    params, grads, _ = tensors([500, 60], 13)
    twin = [p.clone() for p in params]
    a, b = AdamW(params, grads, state_bits=bits, seed=3), AdamW(twin, grads, state_bits=bits, seed=3)
    bad = [torch.full((500,), float("nan"), device="cuda"), torch.zeros(61, device="cuda")]
    with pytest.raises(HierTCNError, match=r"grads\[1\]"):
        a.step(bad)
    z = [torch.zeros_like(x) for x in a.m]
    kw = {} if bits == 32 else dict(m_scale=[torch.zeros_like(x) for x in a.m_scale], v_scale=[torch.zeros_like(x) for x in a.v_scale])
    with pytest.raises(HierTCNError, match=r"v\[1\]"):
        a.set_state(z, [torch.zeros_like(a.v[0]), torch.zeros_like(a.v[1])[:-1]], 0, **kw)
    assert a.t == 0
    a.step()
    b.step()
    assert all(torch.equal(x, y) for x, y in zip(params + a.m + a.v, twin + b.m + b.v)) and not any(x.any() for x in z)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_moved(bits):
    """p.data = other memory between steps, as loading and resharding do: the step goes there, and what held the parameter before is not written any more."""
    from hiertcn_amd.adamw import AdamW
    params, grads, _ = tensors([700, 300], 15)
    twin = [p.clone() for p in params]
    copies, tcopies = ([torch.empty_like(p, dtype=torch.bfloat16) for p in params] for _ in range(2))
    a, b = AdamW(params, grads, copies=copies, state_bits=bits, seed=3), AdamW(twin, [g.clone() for g in grads], copies=tcopies, state_bits=bits, seed=3)
    a.step()
    b.step()
    old = [p.data for p in params]
    kept = [o.clone() for o in old]
    for p, g, c in zip(params, grads, copies):
        p.data, g.data, c.data = p.data.clone(), g.data.clone(), c.data.clone()
    a.step()
    b.step()
    assert all(torch.equal(x, y) for x, y in zip(params + copies + list(a.m), twin + tcopies + list(b.m)))
    assert all(torch.equal(o, k) for o, k in zip(old, kept)) and not torch.equal(params[0], kept[0])


def test_a_tensor_of_more_blocks_than_a_launch_takes():
    """2^34 + 700 elements: 2^24 + 1 workgroups, more than a launch may have.  First, middle and last blocks of the step and of the decoded moments as the formula says."""
    from hiertcn_amd.adamw import AdamW
    if torch.cuda.mem_get_info()[0] < 170 << 30:
        pytest.skip("170 GiB of device memory")
    n, lr = 2 ** 34 + 700, 1e-2
    p = torch.full((n,), 0.5, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    edge = 2 ** 33                                         # where the second piece of the step begins
    spots = [(0, 512), (edge - 512, 1024), (2 ** 34 - 256, 956)]
    rng = np.random.default_rng(6)
    grads = []
    for at, k in spots:
        grads.append(torch.tensor(rng.standard_normal(k), dtype=torch.float32).to(torch.bfloat16))
        g[at:at + k] = grads[-1].cuda()
    opt = AdamW([p], [g], lr=lr, betas=(B1, B2), eps=E, state_bits=8, seed=9)
    opt.step()
    for (at, k), grad in zip(spots, grads):
        blocks = -(-k // 256)
        zero = np.zeros(blocks, np.float32)
        whole = SO.mix
        try:
            SO.mix = lambda numel, tensor, t, seed, at=at: _bits(at + np.arange(numel, dtype=np.uint64), t, seed)
            q, qm, qv, sm, sv = SO.adamw8(np.full(k, 0.5, np.float32), grad.float().numpy(), np.zeros(k, np.int8), np.zeros(k, np.uint8), zero, zero, 1, lr, B1, B2, E, 0.0, 9, 0)
        finally:
            SO.mix = whole
        b0 = at // 256
        for got, want in ((opt.m[0][at:at + k], qm), (opt.v[0][at:at + k], qv), (opt.m_scale[0][b0:b0 + blocks], sm), (opt.v_scale[0][b0:b0 + blocks], sv)):
            assert np.array_equal(got.cpu().numpy(), want), at
        assert (np.abs(p[at:at + k].cpu().numpy() - q) <= 4 * EPS * (np.abs(q) + 1e-2)).all()
    assert (p[512:edge - 512] == 0.5).all() and (p[edge + 512:2 ** 34 - 256] == 0.5).all()
