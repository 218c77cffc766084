"""CPU side of the sequence operators: the header, the binding and the library agree; bad calls are refused before anything is launched (the
C entries check shapes, strides, addresses and overlaps on the host, so made-up addresses serve); the oracle's gradients against differences."""
import ctypes as C
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from hiertcn_amd import _lib, _ops
from hiertcn_amd._lib import HierTCNError
from oracle import sequence_oracle as SO

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "hiertcn_ops.h")


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        from hiertcn_amd.build import build_lib
        build_lib()
    return _ops.lib()


def _source():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_header_and_binding_name_the_same_functions(lib):
    names = set(re.findall(r"\b(hiertcn_[a-z_0-9]+)\s*\(", _source()))
    assert names == set(_ops.SYMBOLS), names ^ set(_ops.SYMBOLS)
    for path in (_lib.LIB_PATH, _lib.LIB_PATH_F16):
        so = C.CDLL(path)
        assert all(hasattr(so, n) for n in names), path
    version = int(re.search(r"#define\s+HIERTCN_OPS_VERSION\s+(\d+)", _source()).group(1))
    assert lib.hiertcn_ops_version() == version == _ops.VERSION


def test_struct_layouts(lib, tmp_path):
    """Field names, offsets and sizes: the header as gcc compiles it, the binding, and the library."""
    fields = {}
    for body, name in re.findall(r"typedef\s+struct\s*\{(.*?)\}\s*(hiertcn_\w+_t)\s*;", _source(), flags=re.S):
        fields[name] = []
        for decl in body.split(";"):
            if decl.strip():
                first, *more = decl.strip().split(",")
                fields[name] += [re.search(r"(\w+)\s*$", v.strip()).group(1) for v in (first, *more)]
    by_name = {c.__doc__: c for c in _ops.STRUCTS}
    assert set(by_name) == set(fields)
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "hiertcn_ops.h"', "int main(void) {"]
    for st, names in fields.items():
        lines.append(f'printf("{st} %zu\\n", sizeof({st}));')
        lines += [f'printf("{st}.{f} %zu\\n", offsetof({st}, {f}));' for f in names]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"), str(tmp_path / "l.c"), "-o", str(tmp_path / "l")], check=True)
    layout = dict(ln.split() for ln in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines())
    for st, cls in by_name.items():
        assert [f for f, _ in cls._fields_] == fields[st], st
        assert C.sizeof(cls) == int(layout[st])
        for f in fields[st]:
            assert getattr(cls, f).offset == int(layout[f"{st}.{f}"]), (st, f)
    sizes = (C.c_size_t * len(_ops.STRUCTS))()
    assert lib.hiertcn_ops_struct_sizes(sizes) == 0 and list(sizes) == [C.sizeof(c) for c in _ops.STRUCTS]


# ---- gated linear recurrence ------------------------------------------------------------------------------------------------------------------
BASE = 1 << 20      # made-up addresses: never dereferenced, the calls below are refused on the host


def glr_call(B=2, T=10, D=8, **kw):
    a = _ops.Glr(B=B, T=T, D=D, dtype=0, cand_act=1)
    at = BASE
    for f in ("gate", "cand", "out", "dout", "dgate", "dcand"):
        setattr(a, f, at)
        setattr(a, f + "_sb", T * D)
        setattr(a, f + "_st", D)
        at += 1 << 20
    for f in ("state_in", "state_out", "record", "dstate_out", "dstate_in"):
        setattr(a, f, at)
        at += 1 << 20
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,word", [
    (dict(B=-1), "negative"), (dict(dtype=5), "dtype"), (dict(cand_act=2), "cand_act"), (dict(gate=None), "null"), (dict(out=None), "null"),
    (dict(gate_sb=-80), "stride"), (dict(gate=BASE + 2), "multiple"), (dict(state_in=BASE + 1), "multiple"), (dict(out_st=4), "overlap"),
    (dict(out_sb=0), "overlap"), (dict(out=BASE), "overlaps an input"), (dict(record=BASE + 64), "overlaps an input"),
    (dict(state_out=BASE + (6 << 20) + 8), "overlaps an input"), (dict(B=1 << 40), "at most"),
], ids=lambda v: str(v) if isinstance(v, dict) else "")
def test_glr_forward_refuses(lib, kw, word):
    a = glr_call(**kw)
    assert lib.hiertcn_glr_forward(C.byref(a), None) < 0
    assert word in lib.hiertcn_ops_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(dout=None), "null"), (dict(dgate=None), "null"), (dict(record=None), "null"), (dict(dgate=BASE), "overlaps an input"),
    (dict(dcand=BASE + (4 << 20) + 32), "two outputs"), (dict(dcand_st=7), "overlap"),
], ids=lambda v: str(v) if isinstance(v, dict) else "")
def test_glr_backward_refuses(lib, kw, word):
    a = glr_call(**kw)
    assert lib.hiertcn_glr_backward(C.byref(a), None) < 0
    assert word in lib.hiertcn_ops_last_error().decode()


def test_glr_a_missing_workspace_is_refused(lib):
    B, T, D = 1, 100000, 64
    need = lib.hiertcn_glr_workspace_bytes(B, T, D)
    assert need > 0 and lib.hiertcn_glr_workspace_bytes(4096, 16, 256) == 0
    at = 1 << 40
    a = _ops.Glr(B=B, T=T, D=D, dtype=1, cand_act=0)
    for f in ("gate", "cand", "out"):
        setattr(a, f, at)
        setattr(a, f + "_sb", T * D)
        setattr(a, f + "_st", D)
        at += 1 << 32
    for ws, nbytes in ((None, 0), (at, need - 1), (at + 4, need + 4)):
        a.workspace, a.workspace_bytes = ws, nbytes
        assert lib.hiertcn_glr_forward(C.byref(a), None) == -4 and b"workspace" in lib.hiertcn_ops_last_error()
    assert lib.hiertcn_glr_forward(None, None) == -1


def test_glr_python_checks():
    from hiertcn_amd.glr import glr_scan, glr_step
    g = torch.zeros(2, 3, 4)
    with pytest.raises(HierTCNError, match="GPU"):
        glr_scan(g, g)
    with pytest.raises(TypeError):
        glr_scan([1], g)
    with pytest.raises(HierTCNError, match="dtype"):
        glr_scan(g.double(), g)
    with pytest.raises(HierTCNError, match=r"\[B, D\]"):
        glr_step(g, g, g)


def test_glr_oracle_gradients_against_differences():
    rng = np.random.default_rng(0)
    B, T, D = 2, 7, 3
    g, x, dh = (rng.standard_normal((B, T, D)) for _ in range(3))
    s, ds = rng.standard_normal((B, D)), rng.standard_normal((B, D))
    mask, lens = (rng.random((B, T)) > 0.3).astype(float), np.array([7, 4])
    for act in ("tanh", "none"):
        ref = SO.glr(g, x, s, mask, lens, act, dh, ds)
        loss = lambda g, x, s: (lambda r: (r["h"] * dh).sum() + (r["state"] * ds).sum())(SO.glr(g, x, s, mask, lens, act))  # noqa: E731
        for k, (name, v) in enumerate(dict(dgate=g, dcand=x, dstate=s).items()):
            for i in np.ndindex(v.shape):
                a, b = [w.copy() for w in (g, x, s)], [w.copy() for w in (g, x, s)]
                a[k][i] += 1e-6
                b[k][i] -= 1e-6
                assert abs((loss(*a) - loss(*b)) / 2e-6 - ref[name][i]) < 1e-8


# ---- losses -------------------------------------------------------------------------------------------------------------------------------------
def rows_call(n=4, T=3, V=50, **kw):
    r = _ops.Rows(n=n, T=T, V=V, dtype=0, ld=V, dld=V, grad_scale=1.0)
    at = BASE
    for f in ("logits", "ids", "logp", "dlogits", "workspace"):
        setattr(r, f, at)
        at += 1 << 24
    r.workspace_bytes = 1 << 22
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def outputs(q, names, at=BASE + (8 << 24)):
    for f in names:
        setattr(q, f, at)
        at += 1 << 20
    return q


ROWS_BAD = [(dict(n=0), "at least 1"), (dict(T=0), "at least 1"), (dict(V=0), "at least 1"), (dict(dtype=3), "dtype"), (dict(logits=None), "null"), (dict(ids=None), "null"),
            (dict(ld=49), "stride"), (dict(dld=10), "stride"), (dict(logits=BASE + 2), "multiple"), (dict(workspace_bytes=8), "workspace"), (dict(workspace=None), "workspace"),
            (dict(dlogits=BASE + 200), "overlaps"), (dict(logp=BASE + 64), "overlaps"), (dict(workspace=BASE), "overlaps"), (dict(grad_scale=float("inf")), "grad_scale"),
            (dict(n=1 << 20, T=1 << 20), "at most")]


@pytest.mark.parametrize("kw,word", ROWS_BAD, ids=lambda v: str(v) if isinstance(v, dict) else "")
def test_losses_refuse_bad_rows(lib, kw, word):
    r = rows_call(**kw)
    q = outputs(_ops.Preference(kind=0, beta=0.1), ("ref", "loss", "pair_loss", "margin", "seq_logp"))
    o = outputs(_ops.Policy(clip_low=0.2, clip_high=0.2), ("old_logp", "advantage", "loss", "kl", "clipped"))
    calls = [lambda: lib.hiertcn_preference_loss(C.byref(r), C.byref(q), None), lambda: lib.hiertcn_policy_loss(C.byref(r), C.byref(o), None)]
    if not {"dlogits", "dld", "grad_scale"} & set(kw):
        calls.append(lambda: lib.hiertcn_sequence_logp(C.byref(r), None))
    for call in calls:
        assert call() < 0 and word in lib.hiertcn_ops_last_error().decode(), lib.hiertcn_ops_last_error()


@pytest.mark.parametrize("kw,word", [(dict(kind=3), "kind"), (dict(beta=0.0), "beta"), (dict(beta=float("nan")), "beta"), (dict(smoothing=0.5), "smoothing"),
                                     (dict(kind=1, smoothing=0.1), "smoothing"), (dict(ref=None), "ref"), (dict(loss=None), "loss"), (dict(margin=BASE), "overlaps"),
                                     (dict(seq_logp=BASE + (8 << 24)), "overlaps ref")], ids=str)
def test_preference_refuses(lib, kw, word):
    q = outputs(_ops.Preference(kind=0, beta=0.1), ("ref", "loss", "pair_loss", "margin", "seq_logp"))
    for k, v in kw.items():
        setattr(q, k, v)
    assert lib.hiertcn_preference_loss(C.byref(rows_call()), C.byref(q), None) < 0 and word in lib.hiertcn_ops_last_error().decode()
    assert lib.hiertcn_preference_loss(C.byref(rows_call(n=3)), C.byref(outputs(_ops.Preference(beta=1.0), ("ref", "loss", "pair_loss", "margin", "seq_logp"))), None) < 0
    assert b"pairs" in lib.hiertcn_ops_last_error()


@pytest.mark.parametrize("kw,word", [(dict(mean=2), "mean"), (dict(clip_low=1.5), "clip"), (dict(clip_high=-0.1), "clip"), (dict(kl_coef=0.1), "ref_logp"), (dict(kl_coef=-1.0), "kl_coef"),
                                     (dict(old_logp=None), "null"), (dict(adv_sn=-1), "stride"), (dict(kl=BASE), "overlaps"), (dict(clipped=BASE + (8 << 24)), "overlaps")], ids=str)
def test_policy_refuses(lib, kw, word):
    q = outputs(_ops.Policy(clip_low=0.2, clip_high=0.2, adv_sn=1), ("old_logp", "advantage", "loss", "kl", "clipped"))
    for k, v in kw.items():
        setattr(q, k, v)
    assert lib.hiertcn_policy_loss(C.byref(rows_call()), C.byref(q), None) < 0 and word in lib.hiertcn_ops_last_error().decode(), lib.hiertcn_ops_last_error()


def test_loss_python_checks():
    from hiertcn_amd.sequence_loss import policy_loss, preference_loss, sequence_logp
    z, ids = torch.zeros(2, 3, 4), torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: sequence_logp(z, ids), lambda: preference_loss(z, ids, torch.zeros(2)), lambda: policy_loss(z, ids, torch.zeros(2, 3), torch.zeros(2))):
        with pytest.raises(HierTCNError, match="GPU"):
            call()
    with pytest.raises(HierTCNError, match="kind"):
        preference_loss(z, ids, torch.zeros(2), kind="other")
    with pytest.raises(HierTCNError, match="mean"):
        policy_loss(z, ids, torch.zeros(2, 3), torch.zeros(2), mean="other")


def test_loss_oracle_gradients_against_differences():
    rng = np.random.default_rng(3)
    n, T, V = 4, 3, 6
    z = 2 * rng.standard_normal((n, T, V))
    ids = rng.integers(0, V, (n, T))
    lp = SO.rows(z, ids)["logp"]
    old, ref, adv, sref = lp + rng.choice([-0.5, 0.1, 0.4], (n, T)), lp + 0.3 * rng.standard_normal((n, T)), rng.standard_normal(n), rng.standard_normal(n)
    forms = [lambda x, m=m: SO.policy(x, ids, old, adv, ref, 0.2, 0.3, 0.1, m, 2.0) for m in ("sequence", "token")]
    forms += [lambda x, k=k, a=a: SO.preference(x, ids, sref, 0.4, k, 0.1 if k == "sigmoid" else 0.0, a, 2.0) for k in ("sigmoid", "hinge", "squared") for a in (False, True)]
    for form in forms:
        d = form(z)["dlogits"]
        for i in np.ndindex(z.shape):
            a, b = z.copy(), z.copy()
            a[i] += 1e-6
            b[i] -= 1e-6
            assert abs(2.0 * (form(a)["loss"] - form(b)["loss"]) / 2e-6 - d[i]) < 1e-7 * max(1, abs(d).max())


# ---- AdamW -----------------------------------------------------------------------------------------------------------------------------------------
def adamw_call(**kw):
    t = _ops.AdamwTensor(numel=1000, grad_dtype=0, copy_dtype=1, index=0)
    at = BASE
    for f in ("param", "grad", "copy", "m", "v", "m_scale", "v_scale"):
        setattr(t, f, at)
        at += 1 << 20
    a = _ops.Adamw(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, t=1, state_bits=8)
    for k, v in kw.items():
        setattr(t if hasattr(t, k) else a, k, v)
    return t, a


@pytest.mark.parametrize("kw,word", [(dict(state_bits=16), "state_bits"), (dict(t=0), "from 1"), (dict(beta1=1.0), "betas"), (dict(lr=float("nan")), "lr"), (dict(eps=-1.0), "eps"),
                                     (dict(grad_scale=float("inf")), "grad_scale"), (dict(numel=-1), "elements"), (dict(param=None), "null"), (dict(v_scale=None), "null"),
                                     (dict(grad_dtype=7), "gradient dtype"), (dict(copy_dtype=0), "copy dtype"), (dict(weight_decay=-0.1), "weight_decay"),
                                     (dict(param=BASE + 2), "multiple"), (dict(m=BASE), "overlap"), (dict(grad=BASE + 400), "overlap")], ids=str)
def test_adamw_refuses(lib, kw, word):
    t, a = adamw_call(**kw)
    assert lib.hiertcn_adamw_step(C.byref(t), 1, C.byref(a), None) < 0 and word in lib.hiertcn_ops_last_error().decode(), lib.hiertcn_ops_last_error()


def test_adamw_moments_refuses(lib):
    t, _ = adamw_call()
    for m, v, word in ((BASE + (3 << 20), None, "overlaps a state"), (BASE + (9 << 20), BASE + (9 << 20) + 64, "outputs overlap"), (BASE + 1, None, "multiple")):
        mo, vo = (C.c_void_p * 1)(m), (C.c_void_p * 1)(v)
        assert lib.hiertcn_adamw_moments(C.byref(t), 1, mo, vo, None) < 0 and word in lib.hiertcn_ops_last_error().decode()


def test_adamw_python_checks():
    from hiertcn_amd.adamw import AdamW
    with pytest.raises(HierTCNError, match="no parameters"):
        AdamW([])
    with pytest.raises(HierTCNError, match="state_bits"):
        AdamW([torch.zeros(3)], state_bits=4)
    with pytest.raises(HierTCNError, match="GPU"):
        AdamW([torch.zeros(3)])


def test_random_bits_are_even():
    """The rounding's bits: every bit of neighbouring elements, steps and tensors is one half the time (2^16 samples: 5 sigma = 0.01), and bits of one element and the
    next, of one step and the next, agree half the time."""
    n = 1 << 16
    base = SO.mix(n, 3, 10, 12345)
    bit = lambda x: (x[:, None] >> np.arange(32, dtype=np.uint32)) & 1  # noqa: E731
    for other in (SO.mix(n, 3, 11, 12345), SO.mix(n, 4, 10, 12345), SO.mix(n, 3, 10, 12346), np.roll(base, 1)):
        assert abs(bit(other).mean(0) - 0.5).max() < 0.01
        assert abs((bit(other) == bit(base)).mean(0) - 0.5).max() < 0.01


def test_codes_keep_the_expectation_and_nearest_would_not():
    """Mean of the decoded value over all 65,536 random numbers = the value (to the code width / 65,536 and fp32); and why it has to: v under a constant gradient."""
    rng = np.random.default_rng(4)
    for squared in (False, True):
        mag = np.abs(rng.standard_normal(256)).astype(np.float32) + np.float32(1e-3)
        want = mag.astype(np.float64) ** (2 if squared else 1)
        total = np.zeros(256)
        for u in range(0, 65536, 64):
            code, scale = SO.encode(mag, np.full(256, u + 31, np.uint32), squared)
            total += SO.decode(code.astype(np.uint8), scale, squared)
        got = total / 1024
        width = 4 if squared else 2
        assert (np.abs(got - want) <= want.max() * (width / 255 / 1024 + 1e-6) + 1e-5 * want).all()
    v, b2 = np.full(256, 0.25, np.float32), 0.999      # held as sqrt(v) = 0.5; the gradient's size is 1 from now on
    v[0] = 1.0
    q, s = SO.encode(np.sqrt(v), np.full(256, 1 << 15, np.uint32), True)
    q0 = q.copy()
    for _ in range(200):
        v = (SO.decode(q.astype(np.uint8), s, True) * b2 + (1 - b2)).astype(np.float32)
        q, s = SO.encode(np.sqrt(v), np.full(256, 1 << 15, np.uint32), True)
    assert (q == q0).all(), "rounding to nearest: two hundred steps do not move a code"


def test_optimizer_arguments():
    """--optimizer / --weight_decay: attributes only where given; refused where a model trains with Adam alone."""
    from hiertcn_amd.args import make_args
    from hiertcn_amd.engine import check_supported
    assert not hasattr(make_args([]), "optimizer") and not hasattr(make_args([]), "weight_decay")
    args = make_args(["--optimizer", "adamw", "--weight_decay", "0.1"])
    assert args.optimizer == "adamw" and args.weight_decay == 0.1
    check_supported(args)
    with pytest.raises(NotImplementedError, match="optimizer"):
        check_supported(args, optimizer_ok=("adam",))
    del args.optimizer
    with pytest.raises(NotImplementedError, match="weight_decay"):
        check_supported(args)
    with pytest.raises(SystemExit):
        make_args(["--optimizer", "other"])


def test_optimizer_tensors_share_no_memory():
    from hiertcn_amd.adamw import _apart
    from hiertcn_amd._lib import HierTCNError
    buf = torch.zeros(12)
    _apart((("params", [buf[:4], buf[4:8]]), ("copies", [None, buf[8:]]), ("m", None), ("v", [buf[3:3]])))     # side by side, absent and empty ones
    for lists in ([("params", [buf, buf])], [("params", [buf[:5]]), ("copies", [buf[4:]])], [("params", [buf[2:4], buf[9:], buf[:3]])]):
        with pytest.raises(HierTCNError, match="overlap"):
            _apart(lists)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("back", [1, 4096])
def test_losses_refuse_rows_that_their_indices_cannot_walk(lib, dtype, back):
    """A thread's last step goes up to 1024 vectors behind the row: V close to 2^31 would take its index over the edge (whole rows of workspaces and addresses here)."""
    V = 2 ** 31 - back
    assert lib.hiertcn_rows_workspace_bytes(2, 1, V) == 0 and lib.hiertcn_rows_workspace_bytes(2, 1, 2 ** 31 - 4097) > 0
    at = lambda k: (1 << 44) + (k << 36)  # noqa: E731
    r = _ops.Rows(n=2, T=1, V=V, dtype=dtype, ld=V, dld=V, grad_scale=1.0, logits=at(0), ids=at(1), logp=at(2), dlogits=at(3) + 4, workspace=at(4), workspace_bytes=1 << 30)
    q = outputs(_ops.Preference(kind=0, beta=0.1), ("ref", "loss", "pair_loss", "margin", "seq_logp"))
    o = outputs(_ops.Policy(clip_low=0.2, clip_high=0.2), ("old_logp", "advantage", "loss", "kl", "clipped"))
    for call in (lambda: lib.hiertcn_sequence_logp(C.byref(r), None), lambda: lib.hiertcn_preference_loss(C.byref(r), C.byref(q), None),
                 lambda: lib.hiertcn_policy_loss(C.byref(r), C.byref(o), None)):
        assert call() == -1 and b"at most 2^31 - 4097" in lib.hiertcn_ops_last_error()


@pytest.fixture
def steps(monkeypatch):
    """AdamW on host tensors: what each call of the library is given, as (function, the descriptors' fields) instead of the call."""
    seen = []

    def call(fn, device, desc, n, *rest):
        seen.append((fn, [{f: getattr(d, f) for f, _ in _ops.AdamwTensor._fields_} for d in desc]))
    monkeypatch.setattr(_ops, "on_gpu", lambda t, name: t.device)
    monkeypatch.setattr(_ops, "call", call)
    return seen


def named(opt, grads):
    lists = dict(param=opt.params, grad=grads, copy=opt.copies, m=opt.m, v=opt.v, m_scale=opt.m_scale, v_scale=opt.v_scale)
    return {f: [None if t is None else t.data_ptr() for t in ts] for f, ts in lists.items() if ts is not None}


def given(seen, lists):
    return {f: [d[f] for d in seen[-1][1]] for f in lists}


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_follows_tensors_to_other_memory(lib, steps, bits):
    from hiertcn_amd.adamw import AdamW
    k = (700, 40)
    t = lambda dt, block=1: [torch.zeros(-(-n // block), dtype=dt) for n in k]  # noqa: E731
    params, grads, copies = t(torch.float32), t(torch.float32), [torch.zeros(700, dtype=torch.bfloat16), None]
    state = (t(torch.float32), t(torch.float32)) if bits == 32 else (t(torch.int8), t(torch.uint8), t(torch.float32, 256), t(torch.float32, 256))
    opt = AdamW(params, grads, copies=copies, state_bits=bits, state=state)
    opt.step()
    assert given(steps, named(opt, grads)) == named(opt, grads)
    keep = []
    for change in (params, grads, copies[:1], *state):
        for x in change:
            before, keep = x.data_ptr(), [*keep, x.data]
            x.data = torch.ones_like(x)
            assert x.data_ptr() != before
            opt.step()
            assert given(steps, named(opt, grads)) == named(opt, grads)
    params[0].data = torch.zeros(900).resize_(700).clone()
    params[1].set_(torch.zeros(60)[7:47])
    opt.moments()
    opt.step()
    assert given(steps, named(opt, grads)) == named(opt, grads)
    taken, n = opt.t, len(steps)
    bad = [(torch.zeros(701), "701 elements"), (torch.zeros(700, dtype=torch.float64), "dtype"), (torch.zeros(1400)[::2], "contiguous")]
    for data, word in bad + [(opt.m[0].data, "overlap")] * (bits == 32):
        good, params[0].data = params[0].data, data
        for _ in range(2):
            with pytest.raises(HierTCNError, match=word):
                opt.step()
        params[0].data = good
    good, grads[1].data = grads[1].data, torch.zeros(41)
    for _ in range(2):                       # refused every time, not taken half-way
        with pytest.raises(HierTCNError, match=r"grads\[1\]"):
            opt.step()
    assert opt.t == taken and len(steps) == n
    grads[1].data = good
    opt.step()
    assert opt.t == taken + 1 and given(steps, named(opt, grads)) == named(opt, grads)


def test_adamw_holds_the_memory_that_it_names(lib, steps):
    """Until it has looked again, what the descriptors name is not handed out to anybody else."""
    from hiertcn_amd.adamw import AdamW
    p, g = torch.zeros(1 << 16), torch.zeros(1 << 16)
    opt = AdamW([p], [g])
    at = p.data_ptr()
    p.data = torch.zeros(1 << 16)
    held = [torch.zeros(1 << 16) for _ in range(20)]
    assert all(x.data_ptr() != at for x in (*held, p)) and any(x.data_ptr() == at for x in opt._held)
    opt.step()
    assert all(x.data_ptr() != at for x in opt._held) and steps[-1][1][0]["param"] == p.data_ptr()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_gradients_inside_what_it_writes(lib, steps, bits):
    """A gradient that shares memory with ANOTHER tensor's parameter, copy or state would be read while that is written; gradients may share among themselves."""
    from hiertcn_amd.adamw import AdamW
    buf = torch.zeros(1000)
    params, copies = [buf[:300], buf[300:600]], [torch.zeros(300, dtype=torch.bfloat16) for _ in range(2)]
    opt = AdamW(params, copies=copies, state_bits=bits)
    same = torch.zeros(300)
    opt.step([same, same])
    n, t = len(steps), opt.t
    bad = [([buf[299:599], None], "params"), ([None, buf[:300]], "params"), ([copies[1], None], "copies")]
    if bits == 32:
        bad.append(([None, opt.v[0]], "v"))
    for grads, name in bad:
        for call in (lambda: opt.step(grads), lambda: AdamW(params, grads, copies=copies) if name != "v" else opt.step(grads)):
            with pytest.raises(HierTCNError, match=rf"grads\[.\] and {name}\[.\] overlap"):
                call()
    assert len(steps) == n and opt.t == t
    opt.step([buf[700:], None])
    opt.step([same, same])
    assert opt.t == t + 2
    params[1].data = same                     # the parameter comes to where a gradient that was clear lies
    with pytest.raises(HierTCNError, match=r"grads\[.\] and params\[1\] overlap"):
        opt.step([same, None])


def test_adamw_moments_refuses_outputs_inside_one_another_or_what_it_writes(lib, steps):
    from hiertcn_amd.adamw import AdamW
    params = [torch.zeros(300), torch.zeros(256)]
    opt = AdamW(params, state_bits=8)
    z = lambda: [torch.zeros(300), torch.zeros(256)]  # noqa: E731
    m, v = z(), z()
    buf = torch.zeros(512)
    for out, word in (((m, [m[0], v[1]]), "overlap"), (([m[0], buf[:256]], [v[0], buf[255:511]]), "overlap"), (([params[0], m[1]], v), "params"),
                      (([None, params[1]], [None, None]), "params"), (([m[0], params[0][:256]], v), "params")):
        n = len(steps)
        with pytest.raises(HierTCNError, match=word):
            opt.moments(out=out)
        assert len(steps) == n
    for _ in range(2):
        opt.moments(out=(m, v))
        opt.moments(out=([None, buf[:256]], [v[0], buf[256:]]))
    assert len(steps) == 4


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_moments_takes_one_output_a_tensor(lib, steps, bits):
    """Lists of another length are refused in both forms of the states (entries of None are skipped)."""
    from hiertcn_amd.adamw import AdamW
    params = [torch.zeros(5), torch.zeros(5)]
    opt = AdamW(params, state_bits=bits)
    z = lambda: torch.zeros(5)  # noqa: E731
    for out in (([z()], [z(), z()]), ([z(), z(), z()], [z()])):
        with pytest.raises(HierTCNError):
            opt.moments(out=out)
    if bits == 32:
        opt.m[1].fill_(2.0)
        opt.v[0].fill_(3.0)
        out = ([None, z()], [z(), None])
        opt.moments(out=out)
        assert (out[0][1] == 2).all() and (out[1][0] == 3).all()


def test_adamw_launches_cover_every_block_within_the_limits():
    """The launches of a call (the test-hook build names them): every workgroup of every tensor once, at most 40 tensors and fewer than 2^32 threads a launch -- HIP's
    limit on the threads of a dimension -- for one tensor of 2^40 elements as for many."""
    import itertools
    from hiertcn_amd.build import LIB_TESTHOOKS
    so = C.CDLL(LIB_TESTHOOKS)
    so.hiertcn_test_adamw_walk.restype = C.c_int64
    so.hiertcn_test_adamw_walk.argtypes = [C.POINTER(C.c_int64), C.c_int64, C.c_int, C.POINTER(C.c_int64), C.c_int64]
    sizes = (C.c_int64 * 4)()
    each_moments = so.hiertcn_test_adamw_sizes(sizes)
    piece, span, most, threads = sizes
    G = 1 << 30
    cases = [[1], [0, 5, 0, 257], list(range(1, 150)), [1 << 40], [16 * G - 1], [16 * G], [16 * G + 1024, 3], [17 * G] * 5, [8 * G] * 3 + [1], [3 * G] * 41, [(1 << 40) - 1, 70, 1 << 40]]
    for numel, each in itertools.product(cases, (1, each_moments)):
        out = (C.c_int64 * 50000)()
        rows = so.hiertcn_test_adamw_walk((C.c_int64 * len(numel))(*numel), len(numel), each, out, 10000)
        assert rows > 0
        rows = np.array(out[:5 * rows]).reshape(-1, 5)
        assert (rows[:, 2] < 256).all() and (rows[:, 4] * threads < 2 ** 32).all()
        done = {i: [] for i in range(len(numel))}
        for launch in range(rows[-1, 0] + 1):
            mine = rows[rows[:, 0] == launch]
            assert 0 < len(mine) <= most and (mine[:, 4] == mine[0, 4]).all() and mine[0, 3] == 0
            ends = np.append(mine[1:, 3], mine[0, 4])
            assert (ends > mine[:, 3]).all()
            for (_, tensor, which, first, _), end in zip(mine, ends):
                done[tensor].append((which * piece, which * piece + end - first))
        for i, k in enumerate(numel):
            want, at = -(-k // (span * each)), 0
            for start, end in done[i]:              # in order, side by side
                assert start == at
                at = end
            assert at == want, (numel, i)


def big_rows(n, T, V, dtype=0):
    at = lambda k: (1 << 50) + (k << 44)  # noqa: E731
    return _ops.Rows(n=n, T=T, V=V, dtype=dtype, ld=V, dld=V, grad_scale=1.0, logits=at(0), ids=at(1), logp=at(2), dlogits=at(3), workspace=at(4), workspace_bytes=1 << 43)


@pytest.mark.parametrize("n,T,V", [(1 << 13, 1 << 13, 8), (1 << 12, 1 << 12, 9000), (1 << 11, 1 << 10, 600000), (1 << 14, 1 << 12, 20000)])
def test_losses_refuse_more_rows_than_a_launch_takes(lib, n, T, V):
    """HIP counts a launch's threads in 32 bits: 2^24 - 1 workgroups of 256.  Refused before the first launch, not by the runtime behind it."""
    r = big_rows(n, T, V)
    q = outputs(_ops.Preference(kind=0, beta=0.1), ("ref", "loss", "pair_loss", "margin", "seq_logp"))
    o = outputs(_ops.Policy(clip_low=0.2, clip_high=0.2), ("old_logp", "advantage", "loss", "kl", "clipped"))
    for call in (lambda: lib.hiertcn_sequence_logp(C.byref(r), None), lambda: lib.hiertcn_preference_loss(C.byref(r), C.byref(q), None),
                 lambda: lib.hiertcn_policy_loss(C.byref(r), C.byref(o), None)):
        assert call() == -1 and b"too many for one launch" in lib.hiertcn_ops_last_error()


def test_preference_refuses_more_pairs_than_a_launch_takes(lib):
    """A workgroup of 1024 threads a pair: 2^22 - 1 of them."""
    r = big_rows(1 << 23, 1, 4)
    q = outputs(_ops.Preference(kind=0, beta=0.1), ("ref", "loss", "pair_loss", "margin", "seq_logp"), 1 << 56)
    assert lib.hiertcn_preference_loss(C.byref(r), C.byref(q), None) == -1 and b"pairs: at most" in lib.hiertcn_ops_last_error()


@pytest.mark.parametrize("B,T,D", [(1 << 26, 1, 1), (1 << 27, 3, 64), (1 << 20, 40, 64 * 64)])
def test_glr_refuses_more_sequences_than_a_launch_takes(lib, B, T, D):
    """A wave of 64 threads a sequence and 64 channels, where they are many: fewer than 2^26 of them, by HIP's limit on the threads of a launch."""
    a = _ops.Glr(B=B, T=T, D=D, dtype=0, cand_act=1)
    for k, f in enumerate(("gate", "cand", "out", "dout", "dgate", "dcand", "state_in", "state_out", "record", "dstate_out", "dstate_in")):
        setattr(a, f, (1 << 50) + (k << 46) + 4)          # (addresses that allow one channel at a time)
        if k < 6:
            setattr(a, f + "_sb", T * D)
            setattr(a, f + "_st", D)
    for call in (lib.hiertcn_glr_forward, lib.hiertcn_glr_backward):
        assert call(C.byref(a), None) == -1 and b"too many for one launch" in lib.hiertcn_ops_last_error(), lib.hiertcn_ops_last_error()
