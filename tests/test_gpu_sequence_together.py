"""The sequence operators as a program uses them: a recurrent head (projection -> gated linear recurrence -> item scores) under the preference and the policy loss,
differentiated by their explicit backward calls and stepped by AdamW, against autograd in 64 bits; the losses on a model's `pred`; AdamW as a model's optimizer."""
import numpy as np
import pytest
import torch

from oracle import sequence_oracle as SO
from tests.gpu_common import make_batch, make_params, small_args

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def head64(W, O, x, ids, mask, lengths, s0, loss):
    """The same program in 64 bits on the CPU, with autograd -> loss, dW, dO, the last state"""
    W, O = W.requires_grad_(), O.requires_grad_()
    D = O.shape[1]
    p = x @ W
    u, c = torch.sigmoid(p[..., :D]), torch.tanh(p[..., D:])
    h, hs = s0, []
    for t in range(x.shape[1]):
        on = (t < lengths)[:, None]
        new = u[:, t] * torch.where(mask[:, t, None] != 0, h, torch.zeros_like(h)) + (1 - u[:, t]) * c[:, t]
        h = torch.where(on, new, h)
        hs.append(torch.where(on, new, torch.zeros_like(new)))
    z = torch.stack(hs, 1) @ O.T
    lp = torch.log_softmax(z, -1).gather(-1, ids.long().clamp(min=0)[..., None])[..., 0] * (ids > 0)
    value = loss(lp)
    value.backward()
    return float(value.detach()), W.grad, O.grad, h.detach()


@pytest.mark.parametrize("which", ["preference", "policy"])
def test_a_head_trained_for_three_steps(which):
    """Gradients: every one is a sum of at most B T V = 1.1e5 products whose factors have been through fewer than 1000 roundings each; in units of the largest
    gradient 2000 half steps hold them all.  AdamW's update moves by at most lr |dg| (1 / (sqrt(v) + eps) and its derivative: 2 / eps) for a gradient off by |dg|."""
    from hiertcn_amd.adamw import AdamW
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    from hiertcn_amd.sequence_loss import policy_loss, preference_loss, sequence_logp
    B, T, E, D, V = 6, 37, 24, 40, 501
    g = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    W, O = (0.3 * rn(E, 2 * D)).cuda(), (0.3 * rn(V, D)).cuda()
    x, s0 = rn(B, T, E).cuda(), rn(B, D).cuda()
    lengths = torch.tensor([T, 20, 0, 1, 33, 16], dtype=torch.int32).cuda()
    ids = torch.randint(1, V, (B, T), generator=g, dtype=torch.int32).cuda() * (torch.arange(T).cuda() < lengths[:, None])
    ids = ids.to(torch.int32).contiguous()
    mask = (torch.rand(B, T, generator=g) > 0.1).float().cuda()
    copies = [torch.empty_like(W, dtype=torch.bfloat16), torch.empty_like(O, dtype=torch.bfloat16)]
    eps, lr, decay = 1e-3, 2e-2, 0.1
    opt = AdamW([W, O], lr=lr, eps=eps, weight_decay=decay, copies=copies)
    c64 = lambda t: t.double().cpu()  # noqa: E731
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())

    def forward():
        p = x @ W
        h, last, record = glr_scan(p[..., :D], p[..., D:], s0, want_record=True, mask=mask, lengths=lengths, cand_act="tanh")
        return p, h, last, record, h @ O.t()

    with torch.cuda.stream(stream):          # all of it on a stream of its own
        start = sequence_logp(forward()[4], ids)
        old = start + 0.05 * rn(B, T).cuda()
        adv, ref_sum = rn(B).cuda(), start.sum(1) + rn(B).cuda()
        for step in range(1, 4):
            p, h, last, record, z = forward()
            if which == "preference":
                out = preference_loss(z, ids, ref_sum, beta=0.25, label_smoothing=0.125)
                P = B // 2

                def loss(lp):
                    s = lp.sum(1)
                    m = 0.25 * ((s[:P] - c64(ref_sum)[:P]) - (s[P:] - c64(ref_sum)[P:]))
                    return (0.875 * torch.nn.functional.softplus(-m) + 0.125 * torch.nn.functional.softplus(m)).mean()
            else:
                out = policy_loss(z, ids, old, adv, ref_logp=old, clip_low=0.5, clip_high=0.75, kl_coef=0.125)

                def loss(lp):
                    ratio, gap, a = torch.exp(lp - c64(old)), c64(old) - lp, c64(adv)[:, None]
                    term = -torch.minimum(ratio * a, ratio.clamp(0.5, 1.75) * a) + 0.125 * (torch.exp(gap) - gap - 1)
                    ok = (ids.cpu() > 0).double()
                    n = ok.sum(1)
                    return ((term * ok).sum(1) / n.clamp(min=1)).sum() / (n > 0).sum()
            dz = out["dlogits"]
            dh = dz @ O
            dO = (dz.reshape(-1, V).t() @ h.reshape(-1, D))
            dp = torch.empty_like(p)
            glr_scan_backward(p[..., :D], p[..., D:], dh, record, dgate=dp[..., :D], dcand=dp[..., D:], mask=mask, lengths=lengths, cand_act="tanh")
            dW = x.reshape(-1, E).t() @ dp.reshape(-1, 2 * D)
            stream.synchronize()
            want, wW, wO, wlast = head64(c64(W), c64(O), c64(x), ids.cpu(), mask.cpu(), lengths.cpu(), c64(s0), loss)
            assert abs(float(out["loss"]) - want) <= 2000 * U * max(1.0, abs(want)), (step, float(out["loss"]), want)
            assert (c64(last) - wlast).abs().max() <= 2000 * U
            assert torch.equal(last[2], s0[2])                                # no steps: the state as it came
            off = []
            for got, ref, name in ((dW, wW, "dW"), (dO, wO, "dO")):
                off.append(2000 * U * float(ref.abs().max()))
                assert (c64(got) - ref).abs().max() <= off[-1], (step, name, float((c64(got) - ref).abs().max()), off[-1])
            state = [(c64(q), c64(m).reshape(q.shape), c64(v).reshape(q.shape)) for q, m, v in zip((W, O), opt.m, opt.v)]
            opt.step([dW.contiguous(), dO.contiguous()])
            stream.synchronize()
            for (q, m, v), ref, got, copy, o in zip(state, (wW, wO), (W, O), copies, off):
                new = torch.tensor(SO.adamw64(q, ref, m, v, step, lr, 0.9, 0.999, eps, float(np.float32(decay)))[0])
                assert (c64(got) - new).abs().max() <= lr * 2 / eps * o + 16 * U * float(new.abs().max())
                assert torch.equal(copy, got.to(torch.bfloat16))
    torch.cuda.current_stream().wait_stream(stream)


def test_losses_on_a_models_pred():
    from hiertcn_amd import loss as L
    from hiertcn_amd import model as M
    from hiertcn_amd.model_hier import model_hier
    M.reset_scopes()
    args = small_args(N=600, d=64, H=32)
    M.set_scope("hier", M.HierTCNModel(args, make_params(args), "hier"))
    rng = np.random.default_rng(5)
    x, y, mask = make_batch(rng, 6, 3, 8, 600)
    widths = [int(max(1, (y[:, s] > 0).sum(1).max())) for s in range(3)]
    xl, yl = ([v[:, s, :w] for s, w in enumerate(widths)] for v in (x, y))
    pred, _ = model_hier(args, xl, yl, [mask[:, s:s + 1] for s in range(3)], np.zeros((6, 64), np.float32))
    ids = np.concatenate(yl, 1)
    z = pred.materialize()
    n64 = lambda t: t.double().cpu().numpy()  # noqa: E731

    def close(got, ref, names):
        for k in names:
            d = np.abs(n64(got[k]) - np.asarray(ref[k]))
            assert (d <= np.asarray(ref[k + "_err"]) * (1 + U) + U * np.abs(ref[k]) + 1e-37).all(), (k, float(d.max()))
    lp = L.calc_sequence_logp(pred, ids)
    want = SO.rows(n64(z), ids)
    close({"logp": lp}, want, ["logp"])
    ce = L.calc_loss(pred, ids)
    assert (lp + ce).abs().max() < 1e-4                                      # (the fused cross entropy of the same rows)
    ref = lp.sum(1) + torch.tensor(rng.standard_normal(6), dtype=torch.float32, device=lp.device)
    got = L.calc_preference(pred, ids.astype(np.float64), ref, beta=0.5)
    close(got, SO.preference(n64(z), ids, n64(ref), 0.5, "sigmoid"), ["loss", "pair_loss", "margin", "seq_logp", "dlogits"])
    old = lp + 0.1 * (torch.rand(lp.shape, device=lp.device) - 0.5)          # ratios within 0.95 .. 1.06: away from the clip
    adv = torch.tensor(rng.standard_normal(6), dtype=torch.float32, device=lp.device)
    got = L.calc_policy(pred, ids, old, adv, ref_logp=old, kl_coef=0.25)
    close(got, SO.policy(n64(z), ids, n64(old), n64(adv), n64(old), float(np.float32(0.2)), float(np.float32(0.2)), 0.25), ["loss", "kl", "clipped", "dlogits"])
    assert L.calc_policy(pred, ids, old, adv, want_grad=False)["dlogits"] is None and torch.equal(pred.materialize(), z)
    with pytest.raises(TypeError):
        L.calc_policy(z, ids, old, adv)
    M.reset_scopes()


@pytest.mark.parametrize("dtype,hier", [("bf16", True), ("bf16", False), ("fp32", True)])
def test_adamw_as_a_models_optimizer(dtype, hier):
    """args.optimizer = 'adamw': every variable moves by the formula from the device's own gradients (single fp32 operations: fewer than 12 half steps of the
    parameter and of an update of at most 12 lr), the device's 16-bit copies follow, the slots survive a checkpoint, and Adam's own step is untouched."""
    from hiertcn_amd.engine import Engine
    args = small_args(N=500, d=64, H=32)
    args.storage_dtype, args.optimizer, args.weight_decay = dtype, "adamw", 0.05
    lr = 1e-2
    dev = lambda a: torch.as_tensor(np.ascontiguousarray(a)).cuda().contiguous()  # noqa: E731
    rng = np.random.default_rng(1)
    x, y, mask = make_batch(rng, 6, 4 if hier else 1, 9, 500)
    if hier:
        p, batch = make_params(args), (dev(x), dev(y), dev(mask), dev(np.zeros((6, 64), np.float32)))
    else:
        from hiertcn_amd.params import init_params
        p, batch = init_params(args, 2, "tcn"), (dev(x), dev(y), None, None)
    eng = Engine(args, hier=hier, train=True)
    eng.set_weights(p)
    w = {k: v.astype(np.float64) for k, v in eng.export("weights").items()}
    m, v = ({k: np.zeros_like(a) for k, a in w.items()} for _ in range(2))
    for t in range(1, 4):
        eng.train_forward_backward(*batch)
        g = {k: a.astype(np.float64) for k, a in eng.export("grads").items()}
        eng.optimizer_step(lr)
        got = eng.export("weights")
        for k in w:
            new, m[k], v[k] = SO.adamw64(w[k], g[k], m[k], v[k], t, lr, 0.9, 0.999, 1e-8, float(np.float32(0.05)))
            assert (np.abs(got[k] - new) <= 12 * U * (np.abs(new) + 12 * lr)).all(), (k, t, float(np.abs(got[k] - new).max()))
            w[k] = got[k].astype(np.float64)
    state = eng.optimizer_state()
    assert int(state["adam_t"][0]) == 3
    twin = Engine(args, hier=hier, train=True)
    twin.set_weights(got)                    # the copies that a fresh handle makes of these masters ...
    twin.load_optimizer_state(state)
    outs = []
    for e in (eng, twin):                    # ... are the ones that the step has left
        outs.append(e.forward_eval(*batch, want_rows=True))
    assert torch.equal(outs[0]["rank"], outs[1]["rank"]) and torch.equal(outs[0]["ce"], outs[1]["ce"])
    for e in (eng, twin):
        e.grad_arena().copy_(torch.linspace(-1, 1, e.grad_arena().numel(), device="cuda"))
        e.optimizer_step(lr)
    a, b = eng.export("weights"), twin.export("weights")
    assert all(np.array_equal(a[k], b[k]) for k in a)
    # args without the attribute: Adam, to the bit
    del args.optimizer, args.weight_decay
    pair = []
    for step in ("optimizer_step", "adam_step"):
        e = Engine(args, hier=hier, train=True)
        e.set_weights(p)
        e.grad_arena().copy_(torch.linspace(-1, 1, e.grad_arena().numel(), device="cuda"))
        getattr(e, step)(lr)
        pair.append(e.export("weights"))
        e.close()
    assert all(np.array_equal(pair[0][k], pair[1][k]) for k in pair[0])
    for e in (eng, twin):
        e.close()


def test_training_with_adamw_from_the_command_line():
    from hiertcn_amd.args import make_args
    from hiertcn_amd.model import HierTCNModel
    args = make_args(["--optimizer", "adamw", "--weight_decay", "0.01", "--train"], model_type="hier", item_num=400, emb_dim=64, hidden_dim=32, tcn_channel=[64, 64],
                     model_low_type="tcn", max_activity_len=9, max_session_num=4, batch_size=6)
    model = HierTCNModel(args)
    rng = np.random.default_rng(8)
    x, y, mask = make_batch(rng, 6, 4, 9, 400)
    before = {k: v.copy() for k, v in model.params.items()}
    state = np.zeros((6, 64), np.float32)
    out = model.train_step_packed(x, y, mask, state, 1e-3)
    assert np.isfinite(out["loss"])
    after = model.params
    assert int(model.engine.optimizer_state()["adam_t"][0]) == 1
    # the first step: theta (1 - lr decay) - lr sign(g) wherever a gradient has come through (|g| / (|g| + eps) is within 1e-2 of 1 for |g| > 1e-6)
    g = model.engine.export("grads", root=model.name)
    for k in before:
        on = np.abs(g[k]) > 1e-6
        want = before[k] * (1 - 1e-5) - 1e-3 * np.sign(g[k])
        assert np.abs(after[k] - want)[on].max(initial=0.0) <= 1.1e-5 + 8 * U * np.abs(before[k]).max(), k
        quiet = g[k] == 0
        assert np.abs(after[k] - before[k] * (1 - 1e-5))[quiet].max(initial=0.0) <= 8 * U * np.abs(before[k]).max(), k
    model.engine.close()


def test_calls_on_two_streams_at_once():
    """Long recurrences (whose workgroups hand states to one another), losses and steps on two streams, queued without a wait between them: what each gives alone."""
    from hiertcn_amd.glr import glr_scan, glr_scan_backward
    from hiertcn_amd.sequence_loss import policy_loss
    g = torch.Generator(device="cuda").manual_seed(11)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    B, T, D, n, V = 3, 9001, 130, 12, 30011

    def inputs():
        return dict(p=rn(B, T, 2 * D).to(torch.bfloat16), dh=rn(B, T, D).to(torch.bfloat16), s=rn(B, D), z=rn(n, 5, V), ids=torch.randint(0, V, (n, 5), generator=g, device="cuda", dtype=torch.int32),
                    old=rn(n, 5) - 10, adv=rn(n))

    def work(q):
        gate, cand = q["p"][..., :D], q["p"][..., D:]
        h, last, record = glr_scan(gate, cand, q["s"], want_record=True)
        dg, dc, ds = glr_scan_backward(gate, cand, q["dh"], record)
        out = policy_loss(q["z"], q["ids"], q["old"], q["adv"], ref_logp=q["old"], kl_coef=0.1)
        return h, last, dg, dc, ds, out["loss"], out["dlogits"]
    sets = [inputs(), inputs()]
    alone = []
    for q in sets:
        alone.append(work(q))
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(6):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(work(sets[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for res in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(res, alone[k])), k
