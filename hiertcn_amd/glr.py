"""Gated linear recurrence over sequences: the GRU cell's update (customed_gru_cell.py:309-337) with gates that do not read the state.

    u = sigmoid(gate),  c = tanh(cand) or cand,  h_t = u (h_{t-1} or, where mask is 0, nothing) + (1 - u) c

The state / mask / length conventions are those of the framework's GRU paths: a mask of 0 cuts the carried state (model_hier.py:93),
behind a sequence's length the output is 0 and the state is carried (dynamic_rnn, model_gru.py:47-53).  Forward, backward and single steps run as
HIP kernels (csrc/glr.hip; include/hiertcn_ops.h); gradients are explicit calls, as everywhere in this framework (no autograd graph is built).
"""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _ops
from ._lib import HierTCNError
from ._ops import need

_ACT = {"none": 0, "tanh": 1}


def _rows(t, name, dtype, device, shape):
    """[B, T, D] with a contiguous last dimension and any other strides -> (pointer, stride of b, stride of t)."""
    need(t, name, dtype, device, shape, contiguous=False)
    sb, st, sd = t.stride()
    if sd != 1 and shape[2] > 1:
        raise HierTCNError(f"{name}: the last dimension must be contiguous (stride {sd})")
    return t.data_ptr(), sb, st


def _common(gate, cand, mask, lengths, cand_act):
    device = _ops.on_gpu(gate, "gate")
    if gate.dim() != 3:
        raise HierTCNError(f"gate: shape {tuple(gate.shape)}, expected [B, T, D]")
    if cand_act not in _ACT:
        raise HierTCNError(f"cand_act {cand_act!r}: 'tanh' or 'none'")
    shape = gate.shape
    a = _ops.Glr()
    a.B, a.T, a.D = shape
    a.dtype, a.cand_act = _ops.DTYPE[gate.dtype], _ACT[cand_act]
    a.gate, a.gate_sb, a.gate_st = _rows(gate, "gate", gate.dtype, device, shape)
    a.cand, a.cand_sb, a.cand_st = _rows(cand, "cand", gate.dtype, device, shape)
    if mask is not None:
        need(mask, "mask", torch.float32, device, shape[:2], contiguous=False)
        a.mask, a.mask_sb, a.mask_st = mask.data_ptr(), mask.stride(0), mask.stride(1)
    if lengths is not None:
        a.lengths = need(lengths, "lengths", torch.int32, device, shape[:1]).data_ptr()
    ws = None
    nbytes = _ops.size("hiertcn_glr_workspace_bytes", *shape)
    if nbytes:
        ws = _ops.workspace(nbytes, device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    return a, device, ws


def glr_scan(gate: torch.Tensor, cand: torch.Tensor, state: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
             lengths: Optional[torch.Tensor] = None, cand_act: str = "tanh", want_record: bool = False, state_out: Optional[torch.Tensor] = None):
    """gate, cand [B, T, D] (fp32 / bf16 / fp16, any strides with a contiguous last dimension: the halves of one projection, say), state [B, D]
    fp32 (None: zeros), mask [B, T] fp32 (0 cuts the state in front of the step; None: never), lengths [B] int32 (None: all T)
    -> (h [B, T, D] in gate's type, 0 behind a sequence's end; state behind the last step [B, D] fp32; the record that glr_scan_backward needs, or None).
    state_out: where the state goes -- `state` itself is allowed."""
    a, device, ws = _common(gate, cand, mask, lengths, cand_act)
    B, T, D = gate.shape
    if state is not None:
        a.state_in = need(state, "state", torch.float32, device, (B, D)).data_ptr()
    if state_out is None:
        state_out = torch.empty((B, D), dtype=torch.float32, device=device) if T > 0 or state is not None else torch.zeros((B, D), dtype=torch.float32, device=device)
    else:
        need(state_out, "state_out", torch.float32, device, (B, D))
    h = torch.empty((B, T, D), dtype=gate.dtype, device=device)
    if T == 0 and state is None:
        state_out.zero_()
        return h, state_out, torch.empty(0, dtype=torch.float32, device=device) if want_record else None
    a.state_out = state_out.data_ptr()
    a.out, a.out_sb, a.out_st = h.data_ptr(), T * D, D
    record = None
    if want_record:
        record = torch.empty(_ops.size("hiertcn_glr_record_floats", B, T, D), dtype=torch.float32, device=device)
        a.record = record.data_ptr()
    _ops.call(_ops.lib().hiertcn_glr_forward, device, C.byref(a))
    return h, state_out, record


def glr_scan_backward(gate: torch.Tensor, cand: torch.Tensor, dh: torch.Tensor, record: torch.Tensor, mask: Optional[torch.Tensor] = None,
                      lengths: Optional[torch.Tensor] = None, cand_act: str = "tanh", dstate_out: Optional[torch.Tensor] = None,
                      want_dstate: bool = True, dgate: Optional[torch.Tensor] = None, dcand: Optional[torch.Tensor] = None):
    """Gradients of glr_scan (same gate, cand, mask, lengths, cand_act; its record) for dh [B, T, D] (gate's type) and dstate_out [B, D] fp32 (None:
    zeros) -> (dgate, dcand [B, T, D], 0 behind a sequence's end; dstate [B, D] fp32 or None).  dgate / dcand: where they go, any strides with a contiguous
    last dimension (the halves of one [B, T, 2 D] buffer, say)."""
    a, device, ws = _common(gate, cand, mask, lengths, cand_act)
    shape = gate.shape
    B, T, D = shape
    need(record, "record", torch.float32, device, (_ops.size("hiertcn_glr_record_floats", B, T, D),))
    a.record = record.data_ptr()
    a.dout, a.dout_sb, a.dout_st = _rows(dh, "dh", gate.dtype, device, shape)
    dgate = torch.empty(shape, dtype=gate.dtype, device=device) if dgate is None else dgate
    dcand = torch.empty(shape, dtype=gate.dtype, device=device) if dcand is None else dcand
    a.dgate, a.dgate_sb, a.dgate_st = _rows(dgate, "dgate", gate.dtype, device, shape)
    a.dcand, a.dcand_sb, a.dcand_st = _rows(dcand, "dcand", gate.dtype, device, shape)
    if dstate_out is not None:
        a.dstate_out = need(dstate_out, "dstate_out", torch.float32, device, (B, D)).data_ptr()
    dstate = None
    if want_dstate:
        if T == 0 and dstate_out is None:
            return dgate, dcand, torch.zeros((B, D), dtype=torch.float32, device=device)
        dstate = torch.empty((B, D), dtype=torch.float32, device=device)
        a.dstate_in = dstate.data_ptr()
    _ops.call(_ops.lib().hiertcn_glr_backward, device, C.byref(a))
    return dgate, dcand, dstate


def glr_step(gate: torch.Tensor, cand: torch.Tensor, state: torch.Tensor, mask: Optional[torch.Tensor] = None, active: Optional[torch.Tensor] = None,
             cand_act: str = "tanh", state_out: Optional[torch.Tensor] = None):
    """One more step of every lane (serving): gate, cand [B, D], state [B, D] fp32, mask [B] fp32, active [B] int32 (0: the lane has no step -- its output is
    0 and its state stays) -> (h [B, D], state).  state_out: where the new state goes; `state` itself updates it in place."""
    if isinstance(gate, torch.Tensor) and gate.dim() != 2:
        raise HierTCNError(f"gate: shape {tuple(gate.shape)}, expected [B, D]")
    device = _ops.on_gpu(gate, "gate")
    if cand_act not in _ACT:
        raise HierTCNError(f"cand_act {cand_act!r}: 'tanh' or 'none'")
    shape = gate.shape
    B, D = shape
    need(cand, "cand", gate.dtype, device, shape, contiguous=False)
    need(state, "state", torch.float32, device, shape)
    (gb, gd), (cb, cd) = gate.stride(), cand.stride()
    if D > 1 and (gd != 1 or cd != 1):
        raise HierTCNError("gate, cand: the last dimension must be contiguous")
    h = torch.empty(shape, dtype=gate.dtype, device=device)
    if state_out is None:
        state_out = torch.empty(shape, dtype=torch.float32, device=device)
    elif state_out is not state:
        need(state_out, "state_out", torch.float32, device, shape)
    a = _ops.Glr(B, 1, D, _ops.DTYPE[gate.dtype], _ACT[cand_act], gate.data_ptr(), gb, 0, cand.data_ptr(), cb, 0)
    if mask is not None:
        a.mask, a.mask_sb = need(mask, "mask", torch.float32, device, (B,), contiguous=False).data_ptr(), mask.stride(0)
    if active is not None:
        a.lengths = need(active, "active", torch.int32, device, (B,)).data_ptr()
    a.state_in, a.state_out, a.out, a.out_sb = state.data_ptr(), state_out.data_ptr(), h.data_ptr(), D
    _ops.call(_ops.lib().hiertcn_glr_forward, device, C.byref(a))
    return h, state_out
