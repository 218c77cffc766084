"""Losses on the log-probabilities of a model's answers, with their gradients to the logits: the preference loss over pairs of sequences, the
clipped policy loss with a penalty on the distance from a reference, and the log-probabilities alone (the reference's and the behaviour policy's pass).

They stand beside loss.calc_loss (cross entropy, fused with the scoring layer) and take MATERIALISED logits [n, T, N], as Engine.score_logits or
LazyLogits.materialize give them; loss.calc_preference / loss.calc_policy call them on a model's `pred`.  ids follow the framework: int32, 0 = no answer
(model.py:59-62).  HIP kernels: csrc/seq_loss.hip; C-ABI and exact formulas: include/hiertcn_ops.h."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _ops
from ._lib import HierTCNError
from ._ops import need

_KIND = {"sigmoid": 0, "hinge": 1, "squared": 2}
_MEAN = {"sequence": 0, "token": 1}


def _stride(t, name):
    """Row stride of [n, T, V] whose rows lie at one distance."""
    n, T, V = t.shape
    sn, st, sv = t.stride()
    if V > 1 and sv != 1:
        raise HierTCNError(f"{name}: the last dimension must be contiguous (stride {sv})")
    ld = st if T > 1 else sn if n > 1 else V
    if n > 1 and T > 1 and sn != T * ld:
        raise HierTCNError(f"{name}: rows must lie at one distance (strides {t.stride()})")
    return ld


def _rows(logits, ids, grad_scale=1.0, want_grad=False, dlogits=None):
    device = _ops.on_gpu(logits, "logits")
    if logits.dim() != 3:
        raise HierTCNError(f"logits: shape {tuple(logits.shape)}, expected [n, T, N]")
    n, T, V = logits.shape
    need(ids, "ids", torch.int32, device, (n, T))
    r = _ops.Rows(n=n, T=T, V=V, dtype=_ops.DTYPE[logits.dtype], grad_scale=float(grad_scale))
    r.logits, r.ld, r.ids = logits.data_ptr(), _stride(logits, "logits"), ids.data_ptr()
    logp = torch.empty((n, T), dtype=torch.float32, device=device)
    r.logp = logp.data_ptr()
    if want_grad:
        if dlogits is None:
            dlogits = torch.empty((n, T, V), dtype=logits.dtype, device=device)
        else:
            need(dlogits, "dlogits", logits.dtype, device, logits.shape, contiguous=False)
        r.dlogits, r.dld = dlogits.data_ptr(), _stride(dlogits, "dlogits")
    elif dlogits is not None:
        raise HierTCNError("dlogits given, want_grad is False")
    ws = None
    nbytes = _ops.size("hiertcn_rows_workspace_bytes", n, T, V)
    if nbytes:
        ws = _ops.workspace(nbytes, device)
        r.workspace, r.workspace_bytes = ws.data_ptr(), nbytes
    return r, device, logp, dlogits, ws


def sequence_logp(logits: torch.Tensor, ids: torch.Tensor) -> torch.Tensor:
    """logits [n, T, N] (fp32 / bf16 / fp16; rows at one distance, e.g. a [..., :N] view of padded rows), ids [n, T] int32 -> log-probability of every
    answer [n, T] fp32, 0 where there is none."""
    r, device, logp, _, ws = _rows(logits, ids)
    _ops.call(_ops.lib().hiertcn_sequence_logp, device, C.byref(r))
    return logp


def preference_loss(logits: torch.Tensor, ids: torch.Tensor, ref_logp: torch.Tensor, beta: float = 0.1, kind: str = "sigmoid", label_smoothing: float = 0.0,
                    average: bool = False, grad_scale: float = 1.0, want_grad: bool = True, dlogits: Optional[torch.Tensor] = None) -> dict:
    """Paired log ratios: logits [2 P, T, N], ids [2 P, T] -- sequence i preferred to sequence P + i --, ref_logp [2 P] fp32: the reference model's sum over
    each sequence's answers (its mean with average=True).  With D = (logp_i - ref_i) - (logp_{P+i} - ref_{P+i}):
      kind 'sigmoid' (1 - label_smoothing) softplus(-beta D) + label_smoothing softplus(beta D); 'hinge' max(0, 1 - beta D); 'squared' (D - 1 / (2 beta))^2
    -> dict(loss: 0-d mean over the pairs, pair_loss [P], margin [P] = D, seq_logp [2 P], logp [2 P, T], dlogits: d (grad_scale * loss) in the logits'
    type, or None).  dlogits: where the gradient goes; `logits` itself is overwritten in place."""
    if kind not in _KIND:
        raise HierTCNError(f"kind {kind!r}: one of {', '.join(_KIND)}")
    r, device, logp, dlogits, ws = _rows(logits, ids, grad_scale, want_grad, dlogits)
    P = r.n // 2
    need(ref_logp, "ref_logp", torch.float32, device, (r.n,))
    loss = torch.empty((), dtype=torch.float32, device=device)
    buf = torch.empty(4 * P, dtype=torch.float32, device=device)
    pair, margin, seq = buf.split((P, P, 2 * P))
    base = buf.data_ptr()
    q = _ops.Preference(_KIND[kind], int(bool(average)), beta, label_smoothing, ref_logp.data_ptr(), loss.data_ptr(), base, base + 4 * P, base + 8 * P)
    _ops.call(_ops.lib().hiertcn_preference_loss, device, C.byref(r), C.byref(q))
    return dict(loss=loss, pair_loss=pair, margin=margin, seq_logp=seq, logp=logp, dlogits=dlogits)


def policy_loss(logits: torch.Tensor, ids: torch.Tensor, old_logp: torch.Tensor, advantage: torch.Tensor, ref_logp: Optional[torch.Tensor] = None,
                clip_low: float = 0.2, clip_high: float = 0.2, kl_coef: float = 0.0, mean: str = "sequence", grad_scale: float = 1.0,
                want_grad: bool = True, dlogits: Optional[torch.Tensor] = None) -> dict:
    """Clipped policy loss: logits [n, T, N], ids [n, T], old_logp [n, T] fp32 (the behaviour policy's, sequence_logp), advantage [n] or [n, T] fp32, ref_logp
    [n, T] fp32 (needed for kl_coef > 0).  Per answer: -min(r A, clamp(r, 1 - clip_low, 1 + clip_high) A) + kl_coef (e^g - g - 1) with
    r = exp(logp - old_logp), g = ref_logp - logp; `mean` 'sequence': over each sequence's answers, then over the sequences that have any (the lane
    mean of model.py:111-117); 'token': over all answers.  -> dict(loss, kl, clipped (share of answers the clamp decides): 0-d means; logp [n, T];
    dlogits: d (grad_scale * loss), or None).  dlogits: where the gradient goes; `logits` itself is overwritten in place."""
    if mean not in _MEAN:
        raise HierTCNError(f"mean {mean!r}: 'sequence' or 'token'")
    r, device, logp, dlogits, ws = _rows(logits, ids, grad_scale, want_grad, dlogits)
    shape = ids.shape
    need(old_logp, "old_logp", torch.float32, device, shape)
    per_sequence = isinstance(advantage, torch.Tensor) and advantage.dim() == 1
    need(advantage, "advantage", torch.float32, device, shape[:1] if per_sequence else shape, contiguous=False)
    sn, st = (*advantage.stride(), 0)[:2]
    out = torch.empty(3, dtype=torch.float32, device=device)
    base = out.data_ptr()
    ref = None if ref_logp is None else need(ref_logp, "ref_logp", torch.float32, device, shape).data_ptr()
    q = _ops.Policy(_MEAN[mean], 0, clip_low, clip_high, kl_coef, old_logp.data_ptr(), ref, advantage.data_ptr(), sn, st, base, base + 4, base + 8)
    _ops.call(_ops.lib().hiertcn_policy_loss, device, C.byref(r), C.byref(q))
    loss, kl, clipped = out.unbind()
    return dict(loss=loss, kl=kl, clipped=clipped, logp=logp, dlogits=dlogits)
