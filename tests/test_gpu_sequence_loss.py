"""The preference and policy losses (hiertcn_amd/sequence_loss.py, csrc/seq_loss.hip) and their gradients against their 64-bit restatement."""
import numpy as np
import pytest
import torch

from oracle import sequence_oracle as SO

pytestmark = pytest.mark.gpu
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def make(n, T, V, dtype, seed=0, layout="plain"):
    rng = np.random.default_rng(seed)
    z = torch.tensor(np.clip(2 * rng.standard_normal((n, T, V)), -10, 10), dtype=torch.float32).to(dtype)
    ids = rng.integers(1, max(V, 2), (n, T)) if V > 1 else np.ones((n, T), int)
    lens = rng.integers(0, T + 1, n)
    lens[0] = T
    if n > 2:
        lens[1] = 0
    ids = (ids * (np.arange(T) < lens[:, None])).astype(np.int32)
    if T > 2:
        ids[0, 1] = -3          # no answers either
        ids[0, 2] = V
    if layout == "padded":       # rows of a wider buffer
        buf = torch.full((n, T, V + 5), float("nan"), dtype=dtype)
        buf[..., :V] = z
        z = buf.cuda()[..., :V]
    elif layout == "shifted":
        buf = torch.empty(n * T * V + 3, dtype=dtype)
        buf[3:] = z.reshape(-1)
        z = buf.cuda()[3:].view(n, T, V)
    else:
        z = z.cuda()
    return z, torch.tensor(ids).cuda(), rng


def n64(t):
    return t.double().cpu().numpy()


def close(got, ref, name, dtype=torch.float32):
    want, err = np.asarray(ref[name]), np.asarray(ref[name + "_err"])
    d = np.abs(n64(got) - want)
    allowed = err * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + TINY[dtype]
    assert not (d > allowed).any(), (name, float((d / allowed).max()), np.argwhere(d > allowed)[:3].tolist())


SHAPES = [(2, 1, 2), (4, 3, 7), (2, 5, 1009), (6, 4, 777), (2, 3, 20778), (2, 2, 70001), (30, 40, 64), (2, 1, 540001)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_preference(shape, dtype):
    from hiertcn_amd.sequence_loss import preference_loss, sequence_logp
    z, ids, rng = make(*shape, dtype, seed=sum(shape))
    kind = ("sigmoid", "hinge", "squared")[shape[2] % 3]
    smoothing = 0.1 if kind == "sigmoid" else 0.0
    base = SO.rows(n64(z), ids.cpu().numpy())["logp"].sum(1)
    ref = torch.tensor(base + 4 * rng.standard_normal(shape[0]), dtype=torch.float32).cuda()
    scale = 512.0 if dtype == torch.float16 else 1.0
    want = SO.preference(n64(z), ids.cpu().numpy(), n64(ref), float(np.float32(0.3)), kind, float(np.float32(smoothing)), shape[1] % 2 == 0, scale)
    out = preference_loss(z, ids, ref, beta=0.3, kind=kind, label_smoothing=smoothing, average=shape[1] % 2 == 0, grad_scale=scale)
    for k in ("loss", "pair_loss", "margin", "seq_logp", "logp"):
        close(out[k], want, k)
    close(out["dlogits"], want, "dlogits", dtype)
    # without a gradient a row is summed in other parts: the same bounds, not the same bits
    close(sequence_logp(z, ids), want, "logp")
    less = preference_loss(z, ids, ref, beta=0.3, kind=kind, label_smoothing=smoothing, average=shape[1] % 2 == 0, want_grad=False)
    assert less["dlogits"] is None
    for k in ("loss", "pair_loss", "margin", "seq_logp", "logp"):
        close(less[k], want, k)
    again = preference_loss(z, ids, ref, beta=0.3, kind=kind, label_smoothing=smoothing, average=shape[1] % 2 == 0, grad_scale=scale, dlogits=z)
    assert again["dlogits"] is z and torch.equal(z, out["dlogits"])


def policy_inputs(z, ids, rng, per_step=False):
    n, T, _ = z.shape
    lp = SO.rows(n64(z), ids.cpu().numpy())["logp"]
    # log ratios away from the clip's borders log 0.8 = -0.223 and log 1.28 = 0.247
    old = lp - rng.choice([-0.6, -0.35, -0.1, 0.0, 0.05, 0.15, 0.4, 0.9], (n, T))
    ref = lp + rng.choice([-1.0, -0.2, -0.01, 0.0, 0.03, 0.3, 1.5], (n, T))
    adv = rng.standard_normal((n, T) if per_step else n)
    adv.reshape(-1)[0] = 0.0
    to = lambda v: torch.tensor(v, dtype=torch.float32).cuda()  # noqa: E731
    return to(old), to(ref), to(adv)


@pytest.mark.parametrize("mean", ["sequence", "token"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_policy(shape, dtype, mean):
    from hiertcn_amd.sequence_loss import policy_loss
    z, ids, rng = make(*shape, dtype, seed=sum(shape) + 1)
    old, ref, adv = policy_inputs(z, ids, rng, per_step=shape[0] % 4 == 2)
    scale = 512.0 if dtype == torch.float16 else 1.0
    f = lambda v: float(np.float32(v))  # noqa: E731
    with_ref = shape[1] != 4
    want = SO.policy(n64(z), ids.cpu().numpy(), n64(old), n64(adv), n64(ref) if with_ref else None, f(0.2), f(0.28), f(0.05) if with_ref else 0.0, mean, scale)
    out = policy_loss(z, ids, old, adv, ref_logp=ref if with_ref else None, clip_low=0.2, clip_high=0.28, kl_coef=0.05 if with_ref else 0.0, mean=mean, grad_scale=scale)
    for k in ("loss", "kl", "clipped", "logp"):
        close(out[k], want, k)
    close(out["dlogits"], want, "dlogits", dtype)
    less = policy_loss(z, ids, old, adv, ref_logp=ref if with_ref else None, clip_low=0.2, clip_high=0.28, kl_coef=0.05 if with_ref else 0.0, mean=mean, want_grad=False)
    for k in ("loss", "kl", "clipped", "logp"):
        close(less[k], want, k)
    policy_loss(z, ids, old, adv, ref_logp=ref if with_ref else None, clip_low=0.2, clip_high=0.28, kl_coef=0.05 if with_ref else 0.0, mean=mean, grad_scale=scale, dlogits=z)
    assert torch.equal(z, out["dlogits"])


@pytest.mark.parametrize("layout", ["padded", "shifted"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(layout, dtype):
    """Padded rows (NaN behind them) and odd addresses; the gradient into rows of another alignment."""
    from hiertcn_amd.sequence_loss import policy_loss
    z, ids, rng = make(3, 4, 1003, dtype, seed=5, layout=layout)
    old, ref, adv = policy_inputs(z, ids, rng)
    want = SO.policy(n64(z), ids.cpu().numpy(), n64(old), n64(adv), None, float(np.float32(0.2)), float(np.float32(0.2)))
    out = policy_loss(z, ids, old, adv)
    close(out["dlogits"], want, "dlogits", dtype)
    buf = torch.full((3, 4, 1010), 3.0, dtype=dtype, device="cuda")
    policy_loss(z, ids, old, adv, dlogits=buf[..., 1:1004])
    d = (n64(buf[..., 1:1004]) - want["dlogits"])
    assert (np.abs(d) <= want["dlogits_err"] * 1.01 + HALF[dtype] * np.abs(want["dlogits"]) + 1e-37).all()
    assert (buf[..., 0] == 3).all() and (buf[..., 1004:] == 3).all()      # what lies between the rows stays


@pytest.mark.parametrize("dtype", DTYPES)
def test_masks(dtype):
    """-inf and the type's lowest value as masks, rows of nothing but -inf, NaN in rows without an answer, all sequences empty."""
    from hiertcn_amd.sequence_loss import policy_loss, preference_loss
    n, T, V = 4, 6, 300
    z, ids, rng = make(n, T, V, dtype, seed=9)
    ids[:] = torch.tensor(rng.integers(1, V, (n, T)), dtype=torch.int32)
    ids[2, 3] = 0
    z[0, :, 100:] = float("-inf")
    z[1, :, 50:] = torch.finfo(dtype).min
    ids[0:2] = ids[0:2] % 50
    z[3, 2] = float("-inf")
    z[2, 3] = float("nan")
    z[3, 3] = torch.finfo(dtype).min
    old, ref, adv = policy_inputs(z, ids, rng)
    host = n64(z)
    host[2, 3] = 0
    want = SO.policy(host, ids.cpu().numpy(), n64(old), n64(adv), n64(ref), float(np.float32(0.2)), float(np.float32(0.2)), float(np.float32(0.1)))
    out = policy_loss(z, ids, old, adv, ref_logp=ref, kl_coef=0.1)
    for k in ("loss", "kl", "clipped", "logp"):
        close(out[k], want, k)
    close(out["dlogits"], want, "dlogits", dtype)
    assert (out["dlogits"][2, 3] == 0).all() and (out["dlogits"][3, 2] == 0).all() and (out["dlogits"][0, :, 100:] == 0).all()
    assert out["logp"][3, 2] == 0 and torch.isfinite(out["dlogits"].float()).all()
    zero = torch.zeros_like(ids)
    for o in (policy_loss(z, zero, old, adv, ref_logp=ref, kl_coef=0.1), policy_loss(z, zero, old, adv, mean="token")):
        assert o["loss"] == 0 and o["kl"] == 0 and o["clipped"] == 0 and (o["dlogits"] == 0).all()
    o = preference_loss(z, zero, torch.zeros(n, device="cuda"), average=True)
    assert abs(float(o["loss"]) - np.log(2)) < 1e-6 and (o["dlogits"] == 0).all() and (o["seq_logp"] == 0).all()


def test_nan_in_an_answered_row_shows():
    from hiertcn_amd.sequence_loss import policy_loss
    z, ids, rng = make(2, 3, 1000, torch.float32, seed=13)
    ids[:] = 5
    old, ref, adv = policy_inputs(z, ids, rng)
    for bad in (float("nan"), float("inf")):
        y = z.clone()
        y[1, 1, 700] = bad
        out = policy_loss(y, ids, old, adv)
        assert torch.isnan(out["loss"]) and torch.isnan(out["dlogits"][1, 1]).any() and torch.isfinite(out["dlogits"][0]).all() and torch.isfinite(out["dlogits"][1, 0]).all()


def test_an_impossible_answer_has_a_finite_gradient():
    """The logit of an answer is -inf: its log-probability is -inf, the preference loss infinite, and the slope at its limit."""
    from hiertcn_amd.sequence_loss import preference_loss
    z, ids, _ = make(2, 1, 50, torch.float32, seed=17)
    ids[:] = 7
    z[0, 0, 7] = float("-inf")
    out = preference_loss(z, ids, torch.zeros(2, device="cuda"), beta=0.5)
    assert torch.isposinf(out["loss"]) and out["logp"][0, 0] == float("-inf")
    p = torch.softmax(z[0, 0].double(), 0)
    want = -0.5 * (torch.nn.functional.one_hot(torch.tensor(7), 50).cuda().double() - p)
    assert (out["dlogits"][0, 0].double() - want).abs().max() < 1e-6


def test_the_gradient_against_differences_of_the_definition():
    from hiertcn_amd.sequence_loss import policy_loss, preference_loss
    z, ids, rng = make(4, 5, 60, torch.float32, seed=19)
    old, ref, adv = policy_inputs(z, ids, rng)
    seq_ref = torch.tensor(rng.standard_normal(4) * 3 - 15, dtype=torch.float32).cuda()
    direction, step, idn = rng.standard_normal(z.shape), 1e-6, ids.cpu().numpy()
    f = lambda v: float(np.float32(v))  # noqa: E731
    for grad, loss in ((policy_loss(z, ids, old, adv, ref_logp=ref, kl_coef=0.5)["dlogits"],
                        lambda x: SO.policy(x, idn, n64(old), n64(adv), n64(ref), f(0.2), f(0.2), 0.5)["loss"]),
                       (preference_loss(z, ids, seq_ref, beta=0.25)["dlogits"], lambda x: SO.preference(x, idn, n64(seq_ref), 0.25, "sigmoid")["loss"])):
        num = (loss(n64(z) + step * direction) - loss(n64(z) - step * direction)) / (2 * step)
        scale = np.linalg.norm(n64(grad)) * np.linalg.norm(direction) / np.sqrt(direction.size)
        assert abs(num - (n64(grad) * direction).sum()) < 1e-4 * max(scale, 1e-3), (num, (n64(grad) * direction).sum())


def test_graph_replays():
    from hiertcn_amd.sequence_loss import policy_loss, preference_loss
    z, ids, rng = make(4, 5, 3001, torch.bfloat16, seed=23)
    old, ref, adv = policy_inputs(z, ids, rng)
    sref = torch.zeros(4, device="cuda")
    keys = ("loss", "logp", "dlogits")

    def step():
        a, b = policy_loss(z, ids, old, adv, ref_logp=ref, kl_coef=0.1), preference_loss(z, ids, sref)
        return [a[k] for k in keys] + [b[k] for k in keys]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        z.mul_(0.9)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_offsets_behind_2_to_the_32():
    from hiertcn_amd.sequence_loss import policy_loss
    n, T, V = 2, 11000, 200000
    z = torch.zeros(n, T, V, dtype=torch.bfloat16, device="cuda")
    assert z.numel() > 2 ** 32
    ids = torch.zeros(n, T, dtype=torch.int32, device="cuda")
    ids[1, T - 1] = 199999
    z[1, T - 1, 199999] = 3.0
    lp = 3.0 - np.log(V - 1 + np.exp(3.0))
    out = policy_loss(z, ids, torch.full((n, T), lp, device="cuda"), torch.ones(n, device="cuda"), dlogits=z)
    assert abs(float(out["logp"][1, T - 1]) - lp) < 1e-5 and abs(float(out["loss"]) + 1) < 1e-5
    p = np.exp(3.0) / (V - 1 + np.exp(3.0))
    assert abs(float(z[1, T - 1, 199999]) + (1 - p)) < 2 ** -8 and abs(float(z[1, T - 1, 5]) - p / np.exp(3.0)) < 2 ** -8 * p
    assert (z[0, 0] == 0).all() and (z[1, T - 2] == 0).all()


@pytest.mark.parametrize("V", [2045, 4001, 8190])
def test_many_rows_of_some_thousand_items(V):
    """4160 rows (a wave takes a row; four rounds of its loads at the longest), against the same rows in two batches of fewer (a workgroup takes a row from 2049
    items on): both within the bounds of the formula; every 97th row is compared with 64 bits."""
    from hiertcn_amd.sequence_loss import policy_loss, sequence_logp
    n, T = 1040, 4
    g = torch.Generator(device="cuda").manual_seed(V)
    z = (2 * torch.randn(n, T, V, generator=g, device="cuda")).clamp(-10, 10).to(torch.bfloat16)
    ids = torch.randint(1, V, (n, T), generator=g, device="cuda", dtype=torch.int32)
    ids[::3, 2:] = 0
    lp = sequence_logp(z, ids)
    parts = torch.cat([sequence_logp(z[:520], ids[:520]), sequence_logp(z[520:], ids[520:])])
    rows = torch.arange(0, n, 97)
    want = SO.rows(n64(z[rows]), ids[rows].cpu().numpy())
    # (a lane of 64 sums up to 128 elements: 96 half steps more than the 32 that the bound counts)
    allowed = 1.01 * (want["logp_err"] + 96 * HALF[torch.float32]) + HALF[torch.float32] * np.abs(want["logp"])
    for got in (lp, parts):
        assert (np.abs(n64(got[rows]) - want["logp"]) <= allowed).all()
    adv = torch.randn(n, generator=g, device="cuda")
    out = policy_loss(z, ids, lp, adv, grad_scale=float(n))                  # ratios of one: c = -A / answers
    p = torch.softmax(z[rows].double(), -1)
    hot = torch.zeros_like(p).scatter_(-1, ids[rows].long()[..., None], 1.0)
    live = (ids[rows] > 0).double()
    c = (-adv[rows].double()[:, None] / (ids[rows] > 0).sum(1, keepdim=True)) * live
    ref = c[..., None] * (hot - p)
    err = (out["dlogits"][rows].double() - ref).abs()
    # relative: (120 + 96) half steps of the sum and 2 (20 + 8) of the exponential, a ratio off by lp's rounding (16 half steps), bf16's half step
    assert (err <= ref.abs() * (HALF[torch.bfloat16] + 400 * HALF[torch.float32]) + 400 * HALF[torch.float32] * c.abs()[..., None]).all(), float(err.max())
    assert (out["dlogits"][::3, 2:] == 0).all()


def test_a_pair_of_very_long_sequences():
    """40000 answers a sequence of 9 items: more rows than a thread of the pair's workgroup keeps bits for.  A row's logp is within 2^-24 (120 + 2 (4 + 20) + 60) of
    itself, D within 2 T of that (1.1 at the worst), its slope within beta^2 / 4 of D's: 1e-3 of beta at beta = 1e-3 (with the rounding of c and p)."""
    from hiertcn_amd.sequence_loss import preference_loss
    T, V, beta = 40000, 9, 1e-3
    g = torch.Generator(device="cuda").manual_seed(2)
    z = (2 * torch.randn(2, T, V, generator=g, device="cuda")).clamp(-10, 10)
    ids = torch.randint(0, V, (2, T), generator=g, device="cuda", dtype=torch.int32)
    z[1, 5], z[0, 39999] = -float("inf"), -float("inf")                      # rows of no distribution, near both ends
    ids[1, 5], ids[0, 39999] = 2, 3
    ref = torch.tensor([-80000.0, -79900.0], device="cuda")
    out = preference_loss(z, ids, ref, beta=beta, grad_scale=1000.0)
    z64, hot = z.double().cpu(), torch.nn.functional.one_hot(ids.long().cpu(), V).double()
    ok = (ids.cpu() > 0) & torch.isfinite(z64[..., 0])
    lp = torch.where(ok, (torch.log_softmax(torch.nan_to_num(z64, neginf=0.0), -1) * hot).sum(-1), torch.zeros(()).double())
    s = lp.sum(1)
    bound = 228 * 2.0 ** -24 * T
    assert ((out["seq_logp"].double().cpu() - s).abs() <= bound + 2.0 ** -24 * s.abs()).all()
    D = float((s[0] - ref[0].double().cpu()) - (s[1] - ref[1].double().cpu()))
    c = 1000.0 * beta * (1 / (1 + np.exp(-beta * D)) - 1.0)
    want = torch.stack([c * (hot[0] - torch.softmax(z64[0], -1)), -c * (hot[1] - torch.softmax(z64[1], -1))])
    want = torch.where(ok[..., None], want, torch.zeros(()).double())
    got = out["dlogits"].double().cpu()
    assert (got[~ok] == 0).all() and ((got - want)[ok].abs() <= 1e-3 * abs(c) + 1000.0 * beta ** 2 / 4 * 2 * bound).all()


@pytest.mark.parametrize("A", [1.5, -1.5])
def test_an_impossible_answer_under_the_policy_loss(A):
    """The logit of an answer is -inf: ratio 0, so the clipped term is 0 (A > 0) or decided by the clamp (A < 0), and its gradient 0.  A reference that is only
    monitored (kl_coef = 0) leaves loss and gradient as they are without it, whether it masks the item too or not; with a coefficient the penalty is infinite."""
    from hiertcn_amd.sequence_loss import policy_loss
    z, ids, _ = make(2, 3, 60, torch.float32, seed=29)
    ids[:] = 7
    z[0, 1, 7] = float("-inf")
    old = torch.full((2, 3), -4.0, device="cuda")
    adv = torch.full((2,), A, device="cuda")
    plain = policy_loss(z, ids, old, adv)
    assert plain["logp"][0, 1] == float("-inf") and torch.isfinite(plain["loss"]) and (plain["dlogits"][0, 1] == 0).all() and torch.isfinite(plain["dlogits"]).all()
    lp = SO.rows(n64(z), ids.cpu().numpy())["logp"]
    ratio = np.exp(lp + 4.0)
    term = -np.minimum(ratio * A, np.clip(ratio, 1 - float(np.float32(0.2)), 1 + float(np.float32(0.2))) * A)
    assert abs(float(plain["loss"]) - term.mean(1).mean()) < 1e-5
    for there in (-3.0, float("-inf")):
        ref = torch.full((2, 3), -3.5, device="cuda")
        ref[0, 1] = there
        out = policy_loss(z, ids, old, adv, ref_logp=ref)
        assert torch.equal(out["loss"], plain["loss"]) and torch.equal(out["dlogits"], plain["dlogits"]) and torch.equal(out["clipped"], plain["clipped"])
        assert not torch.isfinite(out["kl"])
    ref[0, 1] = -3.0
    out = policy_loss(z, ids, old, adv, ref_logp=ref, kl_coef=0.1)
    assert torch.isposinf(out["loss"]) and torch.isposinf(out["kl"]) and torch.isfinite(out["dlogits"][0, 0]).all() and torch.isfinite(out["dlogits"][1]).all()


@pytest.mark.parametrize("layout", ["plain", "shifted"])
@pytest.mark.parametrize("V", [61, 4003])
def test_the_gradient_of_far_logits(V, layout):
    """fp32 logits up to 80 below their row's largest (multiples of 1/1024: differences are exact).  dz_j / dz_max = exp(z_j - z_max) for unanswered j, whatever sum and
    coefficient are: the exponential is within 3 half steps + 1/20 of |x|, dz_j and dz_max one rounding each."""
    from hiertcn_amd.sequence_loss import preference_loss
    rng = np.random.default_rng(V)
    z = torch.tensor(rng.integers(-80 * 1024, 0, (2, 2, V)) / 1024, dtype=torch.float32)
    z[..., 5] = 0.0
    ids = torch.full((2, 2), 9, dtype=torch.int32).cuda()
    if layout == "shifted":
        buf = torch.empty(z.numel() + 3, device="cuda")
        buf[3:] = z.reshape(-1).cuda()
        z = buf[3:].view(2, 2, V)
    d = n64(preference_loss(z.cuda(), ids, torch.zeros(2, device="cuda"), beta=0.5, grad_scale=2.0 ** 20)["dlogits"])
    x = n64(z)
    others = np.arange(V) != 9
    ratio, want = (d / d[..., 5:6])[..., others], np.exp(x)[..., others]
    assert (np.abs(ratio - want) <= (6 + np.abs(x[..., others]) / 20) * HALF[torch.float32] * want).all()


@pytest.mark.parametrize("aligned", [True, False])
def test_the_longest_row(aligned):
    """V = 2^31 - 4097, 16 bytes at a time and (gradient rows of another alignment) one element at a time.  2^31 ones are summed exactly up to 2^24 a thread and joined."""
    from hiertcn_amd.sequence_loss import policy_loss
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("16 GiB of device memory")
    V = 2 ** 31 - 4097
    z = torch.zeros(1, 1, V, dtype=torch.bfloat16, device="cuda")
    z[0, 0, V - 1] = 20.0
    buf = torch.full((V + 1,), 3.0, dtype=torch.bfloat16, device="cuda")
    d = (buf[:V] if aligned else buf[1:]).view(1, 1, V)
    p = np.exp(20.0) / (V - 1 + np.exp(20.0))
    ids = torch.full((1, 1), V - 1, dtype=torch.int32, device="cuda")
    out = policy_loss(z, ids, torch.full((1, 1), float(np.log(p)), device="cuda"), torch.ones(1, device="cuda"), grad_scale=2.0 ** 20, dlogits=d)
    assert abs(float(out["logp"]) - np.log(p)) < 1e-5 and abs(float(out["loss"]) + 1) < 1e-5
    each = 2.0 ** 20 * p / np.exp(20.0)
    assert abs(float(d[0, 0, V - 1]) + 2.0 ** 20 * (1 - p)) <= 2.0 ** 20 * (1 - p) * (2.0 ** -8 + 1e-5)
    head = d[0, 0, :V - 1]
    assert (head == head[0]).all() and abs(float(head[0]) - each) <= each * (2.0 ** -8 + 1e-5)
    assert float(buf[V] if aligned else buf[0]) == 3.0
