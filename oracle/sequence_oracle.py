"""64-bit restatement of the sequence operators (include/hiertcn_ops.h) in NumPy, one step after the other -- test infrastructure only.

Where a function also returns a bound, it is the error that 32-bit arithmetic may leave there, carried along with the value itself:
EPS = 2^-24 is half a step of fp32, and a sigmoid or tanh built from exp2, a reciprocal and a few products is within 16 EPS of itself: one step each for
exp2 and the reciprocal, half a step for every product and sum, and the rounding of x log2 e, which is |x| EPS where nothing is done about it (16-bit operands:
|x| <= 8 here) and |x| / 20 EPS where it is taken back (fp32 operands: up to |x| = 80)."""
from __future__ import annotations

import numpy as np

EPS = 2.0 ** -24
EPS_GATE = 16 * EPS


def _sigmoid(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1, e) / (1 + e)


def glr(gate, cand, state=None, mask=None, lengths=None, act="tanh", dh=None, dstate_out=None):
    """-> dict of float64 arrays: h, state, and with dh: dgate, dcand, dstate; every one with its bound under `<name>_err` (before the rounding to a
    16-bit output type).

    A scan joins partial sums h = A h_before + S in another order than one step after the other.  What is rounded then is S and A h_before by themselves: their
    terms are those of h, so each is at most the sum of the terms' MAGNITUDES (hm, rm below: the same recurrence on absolute values), which may exceed |h|
    where the terms cancel.  Errors are relative to that sum."""
    g, x = np.asarray(gate, np.float64), np.asarray(cand, np.float64)
    B, T, D = g.shape
    u, w = _sigmoid(g), _sigmoid(-g)
    c = np.tanh(x) if act == "tanh" else x
    ec = EPS_GATE * np.abs(c) if act == "tanh" else np.zeros_like(c)
    keep = np.ones((B, T), bool) if mask is None else np.asarray(mask) != 0
    lens = np.full(B, T) if lengths is None else np.clip(np.asarray(lengths), 0, T)
    s = np.zeros((B, D)) if state is None else np.asarray(state, np.float64).copy()
    e, hm = np.zeros((B, D)), np.abs(s)
    h, h_err, prev, prev_err = (np.zeros((B, T, D)) for _ in range(4))
    for t in range(T):
        k, on = keep[:, t, None], (t < lens)[:, None]
        hp, ep = np.where(k, s, 0.0), np.where(k, e, 0.0)
        prev[:, t], prev_err[:, t] = hp, ep
        new = u[:, t] * hp + w[:, t] * c[:, t]
        # the products of the gates and the joins of the scan: one more rounding of each
        mag = u[:, t] * np.where(k, hm, 0.0) + np.abs(w[:, t] * c[:, t])
        err = u[:, t] * ep + (EPS_GATE + 3 * EPS) * mag + w[:, t] * ec[:, t]
        s, e, hm = np.where(on, new, s), np.where(on, err, e), np.where(on, mag, hm)
        h[:, t], h_err[:, t] = np.where(on, new, 0.0), np.where(on, err, 0.0)
    out = dict(h=h, h_err=h_err, state=s, state_err=e)
    if dh is None:
        return out
    d = np.asarray(dh, np.float64)
    r = np.zeros((B, D)) if dstate_out is None else np.asarray(dstate_out, np.float64).copy()
    er, rm = np.zeros((B, D)), np.abs(r)
    # 1 - tanh^2 = 4 e / (1 + e)^2 with e = exp(-2 |x|), whose exponential is within 2 |x| + 3 half steps; the reciprocal, taken twice, 1 + e and the products: 9 more
    q = np.exp(-2 * np.abs(x))
    slope = 4 * q / (1 + q) ** 2 if act == "tanh" else np.ones_like(c)
    es = (2 * np.abs(x) + 12) * EPS if act == "tanh" else np.zeros_like(c)
    dg, dx, dg_err, dx_err = (np.zeros((B, T, D)) for _ in range(4))
    for t in range(T - 1, -1, -1):
        k, on = keep[:, t, None], (t < lens)[:, None]
        lam = d[:, t] + r
        lm = np.abs(d[:, t]) + rm
        el = er + EPS * lm
        uw, gap = u[:, t] * w[:, t], prev[:, t] - c[:, t]
        dg[:, t] = np.where(on, lam * gap * uw, 0.0)
        dx[:, t] = np.where(on, lam * w[:, t] * slope[:, t], 0.0)
        dg_err[:, t] = np.where(on, el * np.abs(gap) * uw + np.abs(lam) * uw * (prev_err[:, t] + ec[:, t] + EPS * np.abs(gap)) + (2 * EPS_GATE + 4 * EPS) * np.abs(dg[:, t]), 0.0)
        dx_err[:, t] = np.where(on, el * w[:, t] * slope[:, t] + (es[:, t] + EPS_GATE + 4 * EPS) * np.abs(dx[:, t]), 0.0)
        new = np.where(k, u[:, t] * lam, 0.0)
        err = np.where(k, u[:, t] * (el + (EPS_GATE + 2 * EPS) * lm), 0.0)
        r, er, rm = np.where(on, new, r), np.where(on, err, er), np.where(on, np.where(k, u[:, t] * lm, 0.0), rm)
    out.update(dgate=dg, dgate_err=dg_err, dcand=dx, dcand_err=dx_err, dstate=r, dstate_err=er)
    return out


# ---- losses on log-probabilities ----------------------------------------------------------------------------------------------------------------
def answered(ids, V):
    ids = np.asarray(ids)
    return (ids > 0) & (ids < V)


def rows(logits, ids):
    """-> dict: logp [n, T] with its bound, live (answered, and not all -inf), p [n, T, V] with its RELATIVE bound.  A sum of positive terms of at most
    32 elements a thread, joined over lanes, waves and at most 64 parts, is within 120 half steps of itself (a thread takes up to 128 where rows are many: 96 more, which
    the callers add); an exponential within 2 (|x| + 4)."""
    z = np.asarray(logits, np.float64)
    n, T, V = z.shape
    ok = answered(ids, V)
    logp, err = np.zeros((n, T)), np.zeros((n, T))
    p, perr, live = np.zeros_like(z), np.zeros_like(z), np.zeros((n, T), bool)
    for i, t in zip(*np.nonzero(ok)):
        row = z[i, t]
        m = row.max()
        if m == -np.inf:
            continue
        live[i, t] = True
        x = row - m
        e = np.exp(x)
        s = e.sum()
        p[i, t] = e / s
        ax = np.where(np.isfinite(x), np.abs(x), 0.0)
        serr = EPS * (120 + 2 * (p[i, t] * (ax + 4)).sum())
        perr[i, t] = serr + EPS * 2 * (ax + 8)
        logp[i, t] = x[ids[i, t]] - np.log(s)
        err[i, t] = EPS * (ax[ids[i, t]] + 2 * abs(np.log(s)) + 2) + serr
    return dict(logp=logp, logp_err=err, live=live, ok=ok, p=p, p_err=perr)


def _dlogits(r, ids, c, c_err):
    """c [n, T] = d loss / d logp, with its bound -> d logits and its bound"""
    n, T, V = r["p"].shape
    one = np.zeros((n, T, V))
    for i, t in zip(*np.nonzero(r["live"])):
        one[i, t, ids[i, t]] = 1.0
    c, c_err = np.where(r["live"], c, 0.0)[..., None], np.where(r["live"], c_err, 0.0)[..., None]
    d = c * (one - r["p"])
    return d, c_err * np.abs(one - r["p"]) + np.abs(c) * r["p"] * (r["p_err"] + 3 * EPS) + 2 * EPS * np.abs(d)


def preference(logits, ids, ref, beta, kind, smoothing=0.0, average=False, grad_scale=1.0):
    r = rows(logits, ids)
    P = len(ref) // 2
    cnt = np.maximum(r["ok"].sum(1), 1) if average else np.ones(2 * P)
    s, s_err = r["logp"].sum(1) / cnt, r["logp_err"].sum(1) / cnt
    D = (s[:P] - ref[:P]) - (s[P:] - ref[P:])
    D_err = s_err[:P] + s_err[P:]
    softplus = lambda v: np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))  # noqa: E731
    if kind == "sigmoid":
        loss = (1 - smoothing) * softplus(-beta * D) + smoothing * softplus(beta * D)
        slope = beta * (_sigmoid(beta * D) - (1 - smoothing))
        slope_err = 0.25 * beta ** 2 * D_err
    elif kind == "hinge":
        loss, slope = np.maximum(0, 1 - beta * D), np.where(beta * D < 1, -beta, 0.0)
        slope_err = np.where(np.abs(beta * D - 1) < beta * D_err, beta, 0.0)
    else:
        loss, slope, slope_err = (D - 0.5 / beta) ** 2, 2 * (D - 0.5 / beta), 2 * D_err
    loss_err = np.abs(slope) * D_err + D_err ** 2 + 2 * EPS * np.abs(loss)
    c = np.concatenate([slope, -slope]) / P * grad_scale / cnt
    c_err = np.concatenate([slope_err, slope_err]) / P * abs(grad_scale) / cnt + 2 * EPS * np.abs(c)
    d, d_err = _dlogits(r, ids, c[:, None] + 0 * r["logp"], c_err[:, None] + 0 * r["logp"])
    return dict(loss=loss.mean(), loss_err=loss_err.mean() + 2 * EPS * abs(loss.mean()), pair_loss=loss, pair_loss_err=loss_err, margin=D, margin_err=D_err + EPS * np.abs(D),
                seq_logp=s, seq_logp_err=s_err + EPS * np.abs(s), logp=r["logp"], logp_err=r["logp_err"], dlogits=d, dlogits_err=d_err)


def policy(logits, ids, old, adv, ref=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0, mean="sequence", grad_scale=1.0):
    """The inputs keep every ratio away from the clip's borders (a ratio on one would be decided by its last bit)."""
    r = rows(logits, ids)
    lp, e = r["logp"], r["logp_err"]
    adv = np.broadcast_to(adv if np.ndim(adv) == 2 else np.asarray(adv)[:, None], lp.shape)
    ok = r["ok"]
    cnt = ok.sum(1, keepdims=True)
    total = max((cnt > 0).sum() if mean == "sequence" else cnt.sum(), 1)
    w = ok / (np.maximum(cnt, 1) * total if mean == "sequence" else total)
    live = r["live"]
    with np.errstate(all="ignore"):
        gap0 = np.where(live, lp - old, 0.0)
        ratio = np.exp(gap0)
        x, y = ratio * adv, np.clip(ratio, 1 - clip_low, 1 + clip_high) * adv
        cut = x > y
        term, c = np.where(cut, -y, -x), np.where(cut, 0.0, -x)
        ratio_err = ratio * (e + EPS * (np.abs(gap0) + 6))
        term_err, c_err = np.where(cut, 4 * EPS * np.abs(y), np.abs(adv) * ratio_err), np.where(cut, 0.0, np.abs(adv) * ratio_err)
        kl, kl_err = np.zeros_like(lp), np.zeros_like(lp)
        if ref is not None:
            g = np.where(live, ref - lp, 0.0)
            kl = np.exp(g) - g - 1
            g_err = e + EPS * np.abs(g)
            kl_err = np.abs(np.expm1(g)) * g_err + g_err ** 2 + 8 * EPS * np.maximum(np.abs(kl), np.where(np.abs(g) >= 0.25, np.exp(g) + np.abs(g), 0))
            term, term_err = term + kl_coef * kl, term_err + kl_coef * kl_err
            c, c_err = c - kl_coef * np.expm1(g), c_err + kl_coef * (np.exp(g) * g_err + 6 * EPS * np.abs(np.expm1(g)))
    term, kl, cut = (np.where(live, v, 0.0) for v in (term, kl, cut))
    tot = lambda v, ve: ((v * w).sum(), (ve * w * live).sum() + 6 * EPS * (np.abs(v) * w).sum())  # noqa: E731
    out = dict(logp=lp, logp_err=e)
    out["loss"], out["loss_err"] = tot(term, term_err)
    out["kl"], out["kl_err"] = tot(kl, kl_err)
    out["clipped"], out["clipped_err"] = tot(cut, 0 * e)
    c = c * w * grad_scale
    out["dlogits"], out["dlogits_err"] = _dlogits(r, ids, c, c_err * w * abs(grad_scale) + 8 * EPS * np.abs(c))
    return out


# ---- AdamW -----------------------------------------------------------------------------------------------------------------------------------------
def adamw64(p, g, m, v, t, lr, b1, b2, eps, decay):
    """One step in 64 bits -> p, m, v"""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * decay) - lr / (1 - b1 ** t) * m / (np.sqrt(v / (1 - b2 ** t)) + eps), m, v


def mix(numel, tensor, t, seed):
    """The 32 random bits of every element of a tensor (numel < 2^32)."""
    with np.errstate(over="ignore"):
        u = np.uint32
        key = u((seed * 0x9E3779B1 + t * 0x6A09E667 + tensor * 0xBB67AE85) & 0xFFFFFFFF)
        x = np.arange(numel, dtype=u) * u(0x9E3779B1) + key
        x = (x ^ (x >> u(16))) * u(0x3C6EF373)
        x = (x ^ (x >> u(15))) * u(0x510E527F)
        return x ^ (x >> u(16))


def _block_max(x):
    return np.pad(x, (0, -x.size % 256)).reshape(-1, 256).max(1)


def decode(q, scale, squared):
    f32 = np.float32
    f = q.astype(f32) * f32(1 / (255 if squared else 127))
    x = f * np.abs(f) * np.repeat(scale, 256)[:q.size]
    return x * x if squared else x


def encode(mag, bits, squared):
    """Single fp32 operations, as the kernel's -> codes (of magnitudes), scales"""
    f32 = np.float32
    top = f32(255 if squared else 127)
    scale = _block_max(mag).astype(f32)
    scale = np.where(scale < f32(2.0 ** -100), f32(0), scale)
    inv = np.where(scale > 0, f32(1) / np.where(scale > 0, scale, f32(1)), f32(0)).astype(f32)
    r = mag * np.repeat(inv, 256)[:mag.size]
    q = np.minimum(np.floor(np.sqrt(r) * top), top - f32(1))
    a, b = q * f32(1 / float(top)), (q + f32(1)) * f32(1 / float(top))
    a, b = a * a, b * b
    if squared:
        a, b, r = a * a, b * b, r * r
    u = bits.astype(f32) * f32(2.0 ** -16)
    code = q.astype(np.int32) + (r - a > u * (b - a))
    if squared:
        code = np.where((mag > 0) & (np.repeat(scale, 256)[:mag.size] > 0), np.maximum(code, 1), code)
    return code, scale


def adamw8(p, g, qm, qv, sm, sv, t, lr, b1, b2, eps, decay, seed, index):
    """One step with 8-bit states, every fp32 operation rounded by itself -> p, qm, qv, sm, sv (codes and scales as the kernel leaves them, to the bit)"""
    f32 = np.float32
    p, g = p.astype(f32), g.astype(f32)
    m, v = decode(qm, sm, False), decode(qv, sv, True)
    m = m * f32(b1) + g * f32(1 - b1)
    v = v * f32(b2) + (g * g) * f32(1 - b2)
    s = np.sqrt(v)
    p = p * f32(1 - lr * decay) - f32(lr / (1 - b1 ** t)) * (m / (s * f32(1 / np.sqrt(1 - b2 ** t)) + f32(eps)))
    bits = mix(p.size, index, t, seed)
    cm, sm = encode(np.abs(m), bits & np.uint32(0xFFFF), False)
    cv, sv = encode(s, bits >> np.uint32(16), True)
    return p, np.where(m < 0, -cm, cm).astype(np.int8), cv.astype(np.uint8), sm, sv
