"""What is measured of the sequence operators: the gated linear recurrence, the preference and policy losses with their gradients, and
the AdamW step.  `run` makes one pass of a case: with `own` through the framework's entry points, without it in elementary torch
operations in 32 bits."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}

# variables of the HierTCN model at the XING catalogue (20,778 items, emb 128, hidden 128 x 2 layers, two blocks of 128), as element counts
XING_VARIABLES = "2659584,128,49152,81920,128,81920,128,2659584,20778,65536,256,32768,128,65536,256,32768,128"
# the 300,000-item catalogue at d = 256: item table, scoring kernel and bias, projection, two conv blocks, the across-session cells
LARGE_VARIABLES = "76800000,256,196608,327680,256,327680,256,76800000,300000,262144,512,131072,256,262144,512,131072,256"


def listed():
    return [
        # serving: one more event of 32 lanes, d = 256
        {"name": "glr step 32x256 bf16", "op": "glr", "mode": "step", "B": 32, "T": 1, "D": 256, "dtype": "bf16", "act": "tanh", "ragged": False, "resets": False},
        # the training batch of the run loops: 32 lanes x 10 sessions x 20 events, the state cut at user boundaries
        {"name": "glr train 32x200x128 fp32", "op": "glr", "mode": "train", "B": 32, "T": 200, "D": 128, "dtype": "fp32", "act": "tanh", "ragged": True, "resets": True},
        # the single-level models' longest sequences (500 events), ragged
        {"name": "glr train 64x500x256 bf16", "op": "glr", "mode": "train", "B": 64, "T": 500, "D": 256, "dtype": "bf16", "act": "tanh", "ragged": True, "resets": False},
        # whole histories as one sequence: few lanes, long time axis
        {"name": "glr train 2x65536x512 bf16", "op": "glr", "mode": "train", "B": 2, "T": 65536, "D": 512, "dtype": "bf16", "act": "none", "ragged": False, "resets": True},
        # odd sizes, forward only
        {"name": "glr forward 17x1001x333 fp16", "op": "glr", "mode": "forward", "B": 17, "T": 1001, "D": 333, "dtype": "fp16", "act": "none", "ragged": True, "resets": True},
        # preference pairs on sessions of 20 events over the XING catalogue
        {"name": "preference 16x20x20778 bf16", "op": "preference", "n": 16, "T": 20, "V": 20778, "dtype": "bf16", "kind": "sigmoid", "ragged": True},
        # ... over the 300,000-item catalogue, in the 32 bits that the materialised logits have
        {"name": "preference 8x30x300000 fp32", "op": "preference", "n": 8, "T": 30, "V": 300000, "dtype": "fp32", "kind": "squared", "ragged": True},
        # the smallest policy batch
        {"name": "policy 4x5x1009 fp32", "op": "policy", "n": 4, "T": 5, "V": 1009, "dtype": "fp32", "mean": "token", "ragged": False},
        # 64 sessions of 30 events over the 300,000-item catalogue
        {"name": "policy 64x30x300000 bf16", "op": "policy", "n": 64, "T": 30, "V": 300000, "dtype": "bf16", "mean": "sequence", "ragged": True},
        # the optimizer over the XING model's variables
        {"name": "adamw xing 32-bit", "op": "adamw", "sizes": XING_VARIABLES, "bits": 32, "grad": "fp32", "copy": "none"},
        # ... over the large catalogue's, states in 8 bits, 16-bit gradients and a 16-bit copy for the forward pass
        {"name": "adamw 300k 8-bit", "op": "adamw", "sizes": LARGE_VARIABLES, "bits": 8, "grad": "bf16", "copy": "bf16"},
        # many small tensors of odd sizes
        {"name": "adamw 48 small 8-bit", "op": "adamw", "sizes": ",".join(str(1 + (i * 977) % 5003) for i in range(48)), "bits": 8, "grad": "fp32", "copy": "fp16"},
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["glr", "glr", "preference", "policy", "adamw"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "glr":
        B, T, D = _between(rng, 1, 512), _between(rng, 1, 65536), _between(rng, 16, 1024)
        most = 2 * 65536 * 512 // SIZE[dtype]
        while B * T * D > most:
            B, T, D = max(1, B // 2), max(1, int(T * 0.7)), max(16, int(D * 0.9))
        mode = rng.choice(["train", "train", "forward"] + (["step"] if T < 64 else []))
        return {"op": "glr", "mode": mode, "B": B, "T": 1 if mode == "step" else T, "D": D, "dtype": dtype,
                "act": rng.choice(["tanh", "none"]), "ragged": rng.random() < 0.6, "resets": rng.random() < 0.5}
    if op == "adamw":
        sizes = [_between(rng, 1, 4_000_000) for _ in range(_between(rng, 1, 60))]
        return {"op": "adamw", "sizes": ",".join(map(str, sizes)), "bits": rng.choice([8, 32]), "grad": dtype, "copy": rng.choice(["none", "bf16", "fp16"])}
    n, T, V = _between(rng, 1, 128), _between(rng, 1, 512), _between(rng, 64, 300000)
    most = (16 if op == "preference" else 64) * 30 * 300000 // SIZE[dtype]
    while n * T * V > most:
        n, T, V = max(1, n // 2), max(1, int(T * 0.7)), max(64, int(V * 0.9))
    more = {"kind": rng.choice(["sigmoid", "hinge", "squared"])} if op == "preference" else {"mean": rng.choice(["sequence", "token"])}
    return {"op": op, "n": n, "T": T, "V": V, "dtype": dtype, "ragged": rng.random() < 0.6, **more}


# ---- what a user's program has in hand ------------------------------------------------------------------------------------------------------
BETA, SMOOTH = 0.1, 0.05          # preference: temperature of the pair, label smoothing of the sigmoid form
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.05
LR, B1, B2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
GRAD_SCALE = {"fp32": 1.0, "bf16": 1.0, "fp16": 4096.0}   # 16-bit IEEE gradients are scaled, as a mixed-precision step scales them
SEED = 20240229                   # seed of the 8-bit states' rounding


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _gen(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    ru = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] == "glr":
        B, T, D, dt = case["B"], case["T"], case["D"], DTYPES[case["dtype"]]
        # gate logits and candidates are the two halves of one projection; a bias of 1.5 on the gates keeps the state for a while
        proj = rn(B, T, 2 * D)
        proj[..., :D].add_(1.5)
        s["proj"] = proj.to(dt)
        s["state"] = rn(B, D)
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
        s["mask"] = (ru(B, T) > 0.05).float() if case["resets"] else None
        if case["mode"] == "train":
            s["dh"], s["dstate_out"] = rn(B, T, D).to(dt), rn(B, D)
        return s
    if case["op"] in ("preference", "policy"):
        n = 2 * case["n"] if case["op"] == "preference" else case["n"]
        T, V, dt = case["T"], case["V"], DTYPES[case["dtype"]]
        logits = torch.empty(n, T, V, dtype=dt, device="cuda")
        lse = torch.empty(n, T, device="cuda")
        ids = torch.randint(1, V, (n, T), generator=g, device="cuda")
        for i in range(n):                       # a sequence at a time, so that the 32-bit values never exist as a whole
            z = 2.0 * rn(T, V)
            z.scatter_add_(1, ids[i][:, None], 4.0 + rn(T, 1))     # the answers that were given are likely ones
            logits[i] = z
            lse[i] = torch.logsumexp(logits[i].float(), -1)
        logp = logits.gather(-1, ids[..., None])[..., 0].float() - lse
        lens = torch.randint(0, T + 1, (n,), generator=g, device="cuda") if case["ragged"] else torch.full((n,), T, device="cuda")
        valid = torch.arange(T, device="cuda") < lens[:, None]
        s["logits"], s["ids"] = logits, (ids * valid).to(torch.int32)
        if case["op"] == "preference":           # the reference model's sums over the same answers
            s["ref"] = ((logp + 0.3 * rn(n, T)) * valid).sum(1)
        else:                                    # the behaviour policy's and the reference's values of every step, an advantage for every sequence
            s["old"], s["ref"], s["adv"] = logp + 0.15 * rn(n, T), logp + 0.2 * rn(n, T), rn(n)
        return s
    # every kind of value is one flat arena with a tensor's part behind the other, each from a multiple of 256 on
    sizes = [int(v) for v in case["sizes"].split(",")]
    flat = lambda dt: torch.zeros(sum(k + -k % 256 for k in sizes), dtype=dt, device="cuda")  # noqa: E731
    s["arena"] = {"params": flat(torch.float32), "grads": flat(DTYPES[case["grad"]]), "m": flat(torch.float32), "v": flat(torch.float32)}
    if case["copy"] != "none":
        s["arena"]["copies"] = flat(DTYPES[case["copy"]])
    if case["bits"] == 8:
        s["arena"].update(qm=flat(torch.int8), qv=flat(torch.uint8))
    for key, buf in s["arena"].items():
        s[key], at = [], 0
        for k in sizes:
            s[key].append(buf[at:at + k])
            at += k + -k % 256
    for i, k in enumerate(sizes):
        s["params"][i].copy_(0.05 * rn(k))
        s["grads"][i].copy_(0.01 * GRAD_SCALE[case["grad"]] * rn(k) * (ru(k) > 0.2))      # (some entries get no gradient)
        if case["copy"] != "none":
            s["copies"][i].copy_(s["params"][i])
        if case["bits"] == 32:
            s["m"][i].copy_(0.003 * rn(k))
            s["v"][i].copy_((0.01 * rn(k)).square())
        else:                                    # codes and block scales, as an earlier step left them
            s["qm"][i].copy_(torch.randint(-127, 128, (k,), generator=g, device="cuda", dtype=torch.int32))
            s["qv"][i].copy_(torch.randint(1, 256, (k,), generator=g, device="cuda", dtype=torch.int32))
    s["copies"] = s.get("copies")
    if case["bits"] == 8:
        s["m_scale"], s["v_scale"] = ([f * (0.5 + ru(-(-k // 256))) for k in sizes] for f in (0.01, 0.03))
    s["t"] = 100                                 # steps taken before
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if c["op"] == "glr":
        return _own_glr(s) if own else _plain_glr(s)
    if c["op"] == "preference":
        return _own_preference(s) if own else _plain_preference(s)
    if c["op"] == "policy":
        return _own_policy(s) if own else _plain_policy(s)
    return _own_adamw(s) if own else _plain_adamw(s)


def _own_glr(s):
    from hiertcn_amd.glr import glr_scan, glr_scan_backward, glr_step
    c, proj, D = s["case"], s["proj"], s["case"]["D"]
    gate, cand = proj[..., :D], proj[..., D:]
    if c["mode"] == "step":
        h, state = glr_step(gate[:, 0], cand[:, 0], s["state"], mask=None if s["mask"] is None else s["mask"][:, 0],
                            active=s["lengths"], cand_act=c["act"])
        return {"h": h[:, None], "state": state}
    kw = dict(mask=s["mask"], lengths=s["lengths"], cand_act=c["act"])
    h, state, record = glr_scan(gate, cand, s["state"], want_record=c["mode"] == "train", **kw)
    if c["mode"] == "forward":
        return {"h": h, "state": state}
    dproj = torch.empty_like(proj)
    _, _, dstate = glr_scan_backward(gate, cand, s["dh"], record, dstate_out=s["dstate_out"], dgate=dproj[..., :D], dcand=dproj[..., D:], **kw)
    return {"h": h, "state": state, "dproj": dproj, "dstate": dstate}


def _own_preference(s):
    from hiertcn_amd.sequence_loss import preference_loss
    c = s["case"]
    out = preference_loss(s["logits"], s["ids"], s["ref"], beta=BETA, kind=c["kind"], label_smoothing=SMOOTH if c["kind"] == "sigmoid" else 0.0,
                          grad_scale=GRAD_SCALE[c["dtype"]])
    return {k: out[k] for k in ("loss", "pair_loss", "seq_logp", "dlogits")}


def _own_policy(s):
    from hiertcn_amd.sequence_loss import policy_loss
    c = s["case"]
    out = policy_loss(s["logits"], s["ids"], s["old"], s["adv"], ref_logp=s["ref"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL, mean=c["mean"],
                      grad_scale=GRAD_SCALE[c["dtype"]])
    return {k: out[k] for k in ("loss", "kl", "logp", "dlogits")}


def _own_adamw(s):
    from hiertcn_amd.adamw import AdamW
    c = s["case"]
    opt = s.get("optimizer")
    if opt is None:                              # a program builds its optimizer once
        opt = s["optimizer"] = AdamW(s["params"], s["grads"], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=DECAY, state_bits=c["bits"], copies=s["copies"], seed=SEED)
        held = {"m": s["qm"], "v": s["qv"], "m_scale": s["m_scale"], "v_scale": s["v_scale"]} if c["bits"] == 8 else {"m": s["m"], "v": s["v"]}
        opt.set_state(t=s["t"], **held)
    opt.step(grad_scale=1.0 / GRAD_SCALE[c["grad"]])
    if c["bits"] == 8:                           # the states as the values that they stand for
        opt.moments(out=(s["m"], s["v"]))
    return {k: s["arena"][k] for k in ("params", "m", "v", "copies") if k in s["arena"]}


# ---- the plain forms -----------------------------------------------------------------------------------------------------------------------
def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t from h = 0 along dim 1, by doubling: after the pass of distance k every element holds the map of its last 2 k steps.
    A coefficient of zero cuts what lies before it."""
    k, T = 1, a.shape[1]
    while k < T:
        b = torch.cat([b[:, :k], torch.where(a[:, k:] == 0, b[:, k:], a[:, k:] * b[:, :-k] + b[:, k:])], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _plain_glr(s):
    c, D = s["case"], s["case"]["D"]
    dt = s["proj"].dtype
    T = s["proj"].shape[1]
    g, x = s["proj"][..., :D].float(), s["proj"][..., D:].float()
    live = (torch.arange(T, device=g.device) < s["lengths"][:, None])[..., None] if s["lengths"] is not None else None
    keep = (s["mask"] != 0)[..., None] if s["mask"] is not None else None
    u, w = torch.sigmoid(g), torch.sigmoid(-g)
    cand = torch.tanh(x) if c["act"] == "tanh" else x
    a, b = u, w * cand
    if keep is not None:
        a = torch.where(keep, a, 0.0)
    if live is not None:                                      # a step behind the end keeps the state
        a, b = torch.where(live, a, 1.0), torch.where(live, b, 0.0)
    first = a[:, :1] * s["state"][:, None] + b[:, :1]
    full = _doubling(a, torch.cat([first, b[:, 1:]], 1))
    h = full if live is None else torch.where(live, full, 0.0)
    out = {"h": h.to(dt), "state": full[:, -1].contiguous()}
    if c["mode"] != "train":
        return out
    dh = s["dh"].float()
    if live is not None:
        dh = torch.where(live, dh, 0.0)
    dh = torch.cat([dh[:, :-1], dh[:, -1:] + s["dstate_out"][:, None]], 1)
    back = torch.cat([torch.zeros_like(a[:, :1]), a.flip(1)[:, :-1]], 1)
    lam = _doubling(back, dh.flip(1)).flip(1)                  # lambda_t = dh_t + a_{t+1} lambda_{t+1}
    prev = torch.cat([s["state"][:, None], full[:, :-1]], 1)
    if keep is not None:
        prev = torch.where(keep, prev, 0.0)
    dg, dx = lam * (prev - cand) * u * w, lam * w
    if c["act"] == "tanh":
        dx = dx * (1.0 - cand * cand)
    if live is not None:
        dg, dx = torch.where(live, dg, 0.0), torch.where(live, dx, 0.0)
    return {**out, "dproj": torch.cat([dg, dx], -1).to(dt), "dstate": a[:, 0] * lam[:, 0]}


def _plain_rows(logits, ids):
    """-> valid, logp (0 where no id), the soft-max's numerators and denominators."""
    z = logits.float()
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, keepdim=True)
    y = ids.long()
    valid = y > 0
    logp = (z.gather(-1, y[..., None]) - m)[..., 0] - torch.log(total[..., 0])
    return valid, torch.where(valid, logp, 0.0), e, total


def _plain_dlogits(e, total, ids, dlogp, dt):
    """d logits of sum dlogp * logp: dlogp (onehot - p)."""
    d = e.mul_((-dlogp / total[..., 0])[..., None])
    d.scatter_add_(-1, ids.long()[..., None], dlogp[..., None])
    return d.to(dt)


def _softplus(x):
    return torch.clamp(x, min=0.0) + torch.log1p(torch.exp(-x.abs()))


def _plain_preference(s):
    c, P = s["case"], s["case"]["n"]
    valid, logp, e, total = _plain_rows(s["logits"], s["ids"])
    seq = logp.sum(1)
    diff = (seq[:P] - s["ref"][:P]) - (seq[P:] - s["ref"][P:])
    if c["kind"] == "sigmoid":
        pair = (1 - SMOOTH) * _softplus(-BETA * diff) + SMOOTH * _softplus(BETA * diff)
        slope = BETA * (torch.sigmoid(BETA * diff) - (1 - SMOOTH))
    elif c["kind"] == "hinge":
        pair = torch.clamp(1 - BETA * diff, min=0.0)
        slope = torch.where(BETA * diff < 1, -BETA, 0.0)
    else:
        pair = (diff - 0.5 / BETA).square()
        slope = 2 * (diff - 0.5 / BETA)
    slope = slope * (GRAD_SCALE[c["dtype"]] / P)
    dlogp = torch.where(valid, torch.cat([slope, -slope])[:, None], 0.0)
    return {"loss": pair.mean(), "pair_loss": pair, "seq_logp": seq, "dlogits": _plain_dlogits(e, total, s["ids"], dlogp, s["logits"].dtype)}


def _plain_policy(s):
    c = s["case"]
    valid, logp, e, total = _plain_rows(s["logits"], s["ids"])
    ratio = torch.exp(torch.where(valid, logp - s["old"], 0.0))
    adv = s["adv"][:, None]
    clipped = torch.clamp(ratio, 1 - CLIP_LOW, 1 + CLIP_HIGH)
    gap = torch.where(valid, s["ref"] - logp, 0.0)
    kl = torch.exp(gap) - gap - 1
    loss = -torch.minimum(ratio * adv, clipped * adv) + KL * kl
    dlogp = torch.where(ratio * adv <= clipped * adv, -ratio * adv, 0.0) + KL * (1 - torch.exp(gap))
    count = valid.sum(1, keepdim=True).float()
    if c["mean"] == "sequence":
        weight = valid / count.clamp(min=1.0) / (count > 0).sum().clamp(min=1)
    else:
        weight = valid / count.sum().clamp(min=1.0)
    return {"loss": (loss * weight).sum(), "kl": (kl * weight).sum(), "logp": logp,
            "dlogits": _plain_dlogits(e, total, s["ids"], dlogp * weight * GRAD_SCALE[c["dtype"]], s["logits"].dtype)}


def _mix(numel, tensor, t, seed, device):
    """The 32 random bits of every element of a tensor at a step, from integer products and shifts modulo 2^32 (element < 2^31)."""
    wrap = lambda v: (v & 0xFFFFFFFF) - ((v & 0x80000000) << 1)  # noqa: E731
    key = (seed * 0x9E3779B1 + t * 0x6A09E667 + tensor * 0xBB67AE85) & 0xFFFFFFFF
    x = torch.arange(numel, dtype=torch.int32, device=device) * wrap(0x9E3779B1) + wrap(key)
    for shift, factor in ((16, 0x3C6EF373), (15, 0x510E527F)):
        x = (x ^ ((x >> shift) & (0xFFFFFFFF >> shift))) * wrap(factor)
    return x ^ ((x >> 16) & 0xFFFF)


def _blocks(x, k):
    return torch.nn.functional.pad(x, (0, -x.numel() % 256)).view(-1, 256) if k is None else x.reshape(-1)[:k]


def _decode(q, scale, top, squared):
    """Values of the codes: sign (q / top)^2 of the block's largest; `squared` is the second moment, whose ROOT is held that way."""
    n = q.numel()
    f = _blocks(q.float(), None) * (1.0 / top)
    x = f * f.abs() * scale[:, None]
    return _blocks(x * x if squared else x, n)


def _encode(mag, bits, top, value, keep):
    """mag [blocks][256] >= 0: codes and scales; a code is rounded up with the probability that leaves the expected value (of the magnitude, or of its
    square) what it was; `keep`: what is not zero gets no code 0."""
    scale = mag.amax(1)
    scale = torch.where(scale < 2.0 ** -100, 0.0, scale)
    inv = torch.where(scale > 0, 1.0 / scale, 0.0)
    r = mag * inv[:, None]
    q = torch.clamp(torch.floor(torch.sqrt(r) * top), max=top - 1)
    a, b = q * (1.0 / top), (q + 1) * (1.0 / top)
    a, b = a * a, b * b
    if value:
        a, b, r = a * a, b * b, r * r
    up = (r - a) > (bits * 2.0 ** -16) * (b - a)
    q = q + up
    return (torch.where((mag > 0) & (scale > 0)[:, None], q.clamp(min=1), q) if keep else q), scale


def _plain_adamw(s):
    c = s["case"]
    s["t"] += 1
    t = s["t"]
    step, root = LR / (1 - B1 ** t), 1.0 / math.sqrt(1 - B2 ** t)
    for i, (p, g) in enumerate(zip(s["params"], s["grads"])):
        g = g.float() * (1.0 / GRAD_SCALE[c["grad"]])
        if c["bits"] == 8:
            m, v = _decode(s["qm"][i], s["m_scale"][i], 127, False), _decode(s["qv"][i], s["v_scale"][i], 255, True)
        else:
            m, v = s["m"][i], s["v"][i]
        m = m * B1 + g * (1 - B1)
        v = v * B2 + (g * g) * (1 - B2)
        rt = torch.sqrt(v)
        p.copy_(p * (1 - LR * DECAY) - step * (m / (rt * root + EPS)))
        if s["copies"] is not None:
            s["copies"][i].copy_(p)
        if c["bits"] == 8:
            n = p.numel()
            bits = _blocks(_mix(n, i, t, SEED, p.device), None)
            mb = _blocks(m, None)
            q, scale = _encode(mb.abs(), (bits & 0xFFFF).float(), 127, False, False)
            s["qm"][i].copy_(_blocks(q * torch.sign(mb), n))
            s["m_scale"][i].copy_(scale)
            q, scale = _encode(_blocks(rt, None), ((bits >> 16) & 0xFFFF).float(), 255, True, True)
            s["qv"][i].copy_(_blocks(q, n))
            s["v_scale"][i].copy_(scale)
            m, v = _decode(s["qm"][i], s["m_scale"][i], 127, False), _decode(s["qv"][i], s["v_scale"][i], 255, True)
        s["m"][i].copy_(m)
        s["v"][i].copy_(v)
    return {k: s["arena"][k] for k in ("params", "m", "v", "copies") if k in s["arena"]}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "glr":
        return _exact_glr(s)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    n, V = s["logits"].shape[0], case["V"]
    valid = s["ids"] > 0
    # every sequence by itself: its values first, then, with the slopes known, its gradient
    logp = torch.zeros(valid.shape, dtype=torch.float64, device="cuda")
    for i in range(n):
        z = s["logits"][i].double()
        logp[i] = torch.log_softmax(z, -1).gather(-1, s["ids"][i].long()[:, None])[:, 0] * valid[i]
    leaf = logp.clone().requires_grad_()
    if case["op"] == "preference":
        P = case["n"]
        seq = (leaf * valid).sum(1)
        ratio = seq - s["ref"].double()
        diff = ratio[:P] - ratio[P:]
        ls = torch.nn.functional.logsigmoid
        if case["kind"] == "sigmoid":
            pair = -(1 - SMOOTH) * ls(BETA * diff) - SMOOTH * ls(-BETA * diff)
        elif case["kind"] == "hinge":
            pair = torch.relu(1 - BETA * diff)
        else:
            pair = (diff - 1 / (2 * BETA)) ** 2
        loss = pair.mean()
        out = {"loss": loss.detach(), "pair_loss": pair.detach(), "seq_logp": seq.detach()}
    else:
        lp = leaf[valid]
        old, ref, adv = s["old"].double()[valid], s["ref"].double()[valid], s["adv"].double()[:, None].expand_as(leaf)[valid]
        r = (lp - old).exp()
        kl = (ref - lp).exp() - (ref - lp) - 1
        step = -torch.min(r * adv, r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv) + KL * kl
        row = torch.arange(n, device="cuda")[:, None].expand_as(valid)[valid]
        if case["mean"] == "sequence":
            count = torch.bincount(row, minlength=n).double()
            weight = 1 / count[row] / max(1, int((count > 0).sum()))
        else:
            weight = torch.full_like(lp, 1.0 / max(1, lp.numel()))
        loss = (step * weight).sum()
        out = {"loss": loss.detach(), "kl": (kl * weight).sum().detach(), "logp": logp}
    loss.backward()
    dz = torch.empty(s["logits"].shape, dtype=torch.float64 if case["dtype"] == "fp32" else torch.float32, device="cuda")
    for i in range(n):
        z = s["logits"][i].double().requires_grad_()
        torch.log_softmax(z, -1).gather(-1, s["ids"][i].long()[:, None])[:, 0].backward(leaf.grad[i] * valid[i] * GRAD_SCALE[case["dtype"]])
        dz[i] = z.grad
    return {**out, "dlogits": dz}


def _exact_glr(s):
    c, D = s["case"], s["case"]["D"]
    proj = s["proj"].double()
    B, T = proj.shape[:2]
    state = s["state"].double()
    lens = s["lengths"].tolist() if s["lengths"] is not None else [T] * B
    n = torch.tensor(lens, device="cuda")[:, None]
    h = torch.zeros(B, T, D, dtype=torch.float64, device="cuda")
    before = torch.zeros_like(h)
    hold = torch.ones(B, T, 1, dtype=torch.float64, device="cuda") if s["mask"] is None else (s["mask"] != 0).double()[..., None]
    u = 1 / (1 + torch.exp(-proj[..., :D]))
    w = 1 / (1 + torch.exp(proj[..., :D]))
    cand = proj[..., D:].tanh() if c["act"] == "tanh" else proj[..., D:]
    for t in range(T):
        before[:, t] = hold[:, t] * state
        new = u[:, t] * before[:, t] + w[:, t] * cand[:, t]
        if c["ragged"]:
            state = torch.where(t < n, new, state)
            h[:, t] = torch.where(t < n, new, 0.0)
        else:
            state = h[:, t] = new
    out = {"h": h, "state": state}
    if c["mode"] != "train":
        return out
    carry, dh = s["dstate_out"].double(), s["dh"]
    lam = torch.zeros_like(h)
    for t in range(T - 1, -1, -1):
        total = carry + dh[:, t]
        if c["ragged"]:
            lam[:, t] = torch.where(t < n, total, 0.0)
            carry = torch.where(t < n, total * u[:, t] * hold[:, t], carry)
        else:
            lam[:, t] = total
            carry = total * u[:, t] * hold[:, t]
    dx = lam * w
    if c["act"] == "tanh":
        dx = dx * (1 - cand ** 2)
    return {**out, "dproj": torch.cat([lam * (before - cand) * u * w, dx], -1), "dstate": carry}


def _exact_adamw(s):
    """The 8-bit states' new codes are random roundings: they have no value here."""
    c, t = s["case"], s["t"] + 1
    out = {k: torch.zeros_like(s["arena"]["params"], dtype=torch.float64) for k in ("params", "m", "v")}
    at = 0
    for i, p in enumerate(s["params"]):
        k, g = p.numel(), s["grads"][i].double() / GRAD_SCALE[c["grad"]]
        if c["bits"] == 8:
            m, v, block = s["qm"][i].double(), s["qv"][i].double(), torch.arange(k, device="cuda") // 256
            m = torch.sign(m) * (m / 127) ** 2 * s["m_scale"][i].double()[block]
            v = ((v / 255) ** 2 * s["v_scale"][i].double()[block]) ** 2
        else:
            m, v = s["m"][i].double(), s["v"][i].double()
        m, v = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g ** 2
        out["params"][at:at + k] = p.double() * (1 - LR * DECAY) - LR * (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS)
        out["m"][at:at + k], out["v"][at:at + k] = m, v
        at += k + -k % 256
    if c["bits"] == 8:
        out["m"] = out["v"] = None
    if s["copies"] is not None:
        out["copies"] = out["params"]
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "glr":
        B, T, D, e = case["B"], case["T"], case["D"], SIZE[case["dtype"]]
        share = 0.5 if case["ragged"] and T > 1 else 1.0          # inputs behind a sequence's end need not be read (lengths are uniform in 0 .. T)
        read, written = (5, 3) if case["mode"] == "train" else (2, 1)
        if case["mode"] == "train":
            read = 3                                              # gates, candidates and dh once each: the two directions share them
        steps = B * T * D * e * (read * share + written) + B * D * 4 * (4 if case["mode"] == "train" else 2)
        return {"bytes": steps + (B * T * 4 * share if case["resets"] else 0), "flops": B * T * D * share * (40 if case["mode"] == "train" else 15)}
    if case["op"] in ("preference", "policy"):
        rows = case["n"] * case["T"] * (2 if case["op"] == "preference" else 1)
        share = 0.5 if case["ragged"] else 1.0                     # (lengths are uniform in 0 .. T)
        return {"bytes": rows * case["V"] * SIZE[case["dtype"]] * (share + 1.0), "flops": rows * case["V"] * share * 8}
    n = sum(int(v) for v in case["sizes"].split(","))
    state = 16 if case["bits"] == 32 else 4 + 4.0 * 4 / 256
    outputs = 4 * (2 if case["bits"] == 8 else 0)                  # the 8-bit states as values
    return {"bytes": n * (8 + SIZE[case["grad"]] + state + outputs + (0 if case["copy"] == "none" else 2)), "flops": n * 20}
