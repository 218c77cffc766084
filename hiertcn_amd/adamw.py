"""AdamW (Adam with decoupled weight decay) over many tensors in one or a few launches, moments in 32 or in 8 bits.  Beside the handles' own TF-form Adam
(Engine.adam_step, model.py:139), which has neither.  Kernel: csrc/adamw.hip; exact formulas: include/hiertcn_ops.h."""
from __future__ import annotations

import bisect
import ctypes as C
from typing import List, Optional, Sequence, Union

import torch

from . import _ops
from ._lib import HierTCNError
from ._ops import need

BLOCK = 256      # elements that share a scale of the 8-bit states
_address = torch.Tensor.data_ptr


def _apart(lists):
    """Refuses two tensors of the lists that share memory: every one is written by waves of its own.  -> where they lie, in order"""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), name, i) for name, ts in lists for i, t in enumerate(ts or ()) if t is not None and t.numel())
    for (_, end, a, i), (start, _, b, j) in zip(spans, spans[1:]):
        if start < end:
            raise HierTCNError(f"{a}[{i}] and {b}[{j}] overlap")
    return spans


def _clear_of(spans, starts, name, places):
    """Refuses a place (address, bytes) that shares memory with one of `spans` (of _apart; starts: their first addresses)."""
    for i, (at, size) in enumerate(places):
        if at and size:
            k = bisect.bisect_left(starts, at + size) - 1
            if k >= 0 and spans[k][1] > at:
                raise HierTCNError(f"{name}[{i}] and {spans[k][2]}[{spans[k][3]}] overlap")


class AdamW:
    """params: fp32 masters (contiguous, on one GPU).  grads: where every step finds the gradients (fp32 / bf16 / fp16, None: no gradient) -- or give them to
    step().  copies: 16-bit tensors that receive the rounded parameters in the same pass (None entries: none).  weight_decay: one value, or one per
    tensor.  state_bits 32: m, v fp32 (8 bytes a parameter); 8: codes with a scale per 256 elements (2 bytes a parameter), rounded at random such that
    the expected state is exact -- `seed` and the step number determine the random bits, so runs repeat.  state: (m, v) or (m, v, m_scale, v_scale), taken as
    set_state takes them, in place of zeros of the optimizer's own.

    The step number is the object's (`t`), so a step cannot be captured into a graph (it would replay with the same bias corrections): it is refused
    there, as the framework's graphs leave Adam outside.

    A tensor that has other memory at the next step (`p.data = ...`, `set_`, `resize_`) is taken anew, with all the checks of the constructor: parameters, copies, bound
    gradients and states of the caller's own are looked at every time.  (The memory they had is held until then.)"""

    def __init__(self, params: Sequence[torch.Tensor], grads: Optional[Sequence[Optional[torch.Tensor]]] = None, lr: float = 1e-3, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: Union[float, Sequence[float]] = 0.0, state_bits: int = 32,
                 copies: Optional[Sequence[Optional[torch.Tensor]]] = None, seed: int = 0, state: Optional[Sequence] = None):
        if state_bits not in (8, 32):
            raise HierTCNError(f"state_bits {state_bits}: 8 or 32")
        self.params: List[torch.Tensor] = list(params)
        if not self.params:
            raise HierTCNError("no parameters")
        n = len(self.params)
        self.device = _ops.on_gpu(self.params[0], "params[0]")
        for i, p in enumerate(self.params):
            self._master(p, i)
        copies = [None] * n if copies is None else list(copies)
        if len(copies) != n:
            raise HierTCNError(f"{n} parameters, {len(copies)} copies")
        self.lr, self.betas, self.eps, self.state_bits, self.seed, self.t = float(lr), (float(betas[0]), float(betas[1])), float(eps), state_bits, int(seed), 0
        self.copies = copies
        self._desc = (_ops.AdamwTensor * n)()
        self._flat_numel = [p.numel() for p in self.params]
        self._flat = [torch.Size([k]) for k in self._flat_numel]
        for i, (d, k) in enumerate(zip(self._desc, self._flat_numel)):
            d.numel, d.index = k, i
        self.set_weight_decay(weight_decay)
        self.grads = None
        if state is not None:
            self._take(state)
        else:
            self._callers = False                  # whether the states are tensors of the caller's
            zeros = lambda dt, block=1: [torch.zeros(-(-p.numel() // block), dtype=dt, device=self.device) for p in self.params]  # noqa: E731
            self._attach(*((zeros(torch.float32), zeros(torch.float32), None, None) if state_bits == 32 else
                           (zeros(torch.int8), zeros(torch.uint8), zeros(torch.float32, BLOCK), zeros(torch.float32, BLOCK))))
        if grads is not None:
            self._bind(grads)
            self.grads = list(grads)
            self._watch()

    def _master(self, p, i):
        return need(p, f"params[{i}]", torch.float32, self.device, p.shape if isinstance(p, torch.Tensor) else ())

    def set_weight_decay(self, weight_decay: Union[float, Sequence[float]]):
        """One value, or one per tensor, from the next step on."""
        n = len(self.params)
        decay = [float(weight_decay)] * n if isinstance(weight_decay, (int, float)) else [float(w) for w in weight_decay]
        if len(decay) != n:
            raise HierTCNError(f"{n} parameters, {len(decay)} weight decays")
        for d, w in zip(self._desc, decay):
            d.weight_decay = w
        self.weight_decay = decay

    def _attach(self, m, v, m_scale, v_scale):
        """All of it, or (an exception) none."""
        dm, dv = (torch.float32, torch.float32) if self.state_bits == 32 else (torch.int8, torch.uint8)
        names = (("m", m, dm, 1), ("v", v, dv, 1)) + ((("m_scale", m_scale, torch.float32, BLOCK), ("v_scale", v_scale, torch.float32, BLOCK)) if self.state_bits == 8 else ())
        found = [[need(t, f"{name}[{i}]", dt, self.device, torch.Size([-(-k // block)])).data_ptr() for i, (t, k) in enumerate(zip(ts, self._flat_numel))]
                 for name, ts, dt, block in names]
        rows = []
        for i, (p, c, k) in enumerate(zip(self.params, self.copies, self._flat_numel)):
            if self._master(p, i).numel() != k:
                raise HierTCNError(f"params[{i}]: {p.numel()} elements, the optimizer was built on {k}")
            if c is not None and (not isinstance(c, torch.Tensor) or c.dtype not in (torch.bfloat16, torch.float16)):
                raise HierTCNError(f"copies[{i}]: a bfloat16 or float16 tensor")
            rows.append((p.data_ptr(), None, 0) if c is None else (p.data_ptr(), need(c, f"copies[{i}]", c.dtype, self.device, p.shape).data_ptr(), _ops.DTYPE[c.dtype]))
        spans = _apart((("params", self.params), ("copies", self.copies), ("m", m), ("v", v), ("m_scale", m_scale), ("v_scale", v_scale)))
        for (name, _, _, _), ptrs in zip(names, found):
            for d, ptr in zip(self._desc, ptrs):
                setattr(d, name, ptr)
        for d, row in zip(self._desc, rows):
            d.param, d.copy, d.copy_dtype = row
        self.m, self.v, self.m_scale, self.v_scale = m, v, m_scale, v_scale
        self._shapes = [p.shape for p in self.params]
        self._written, self._starts = spans, [s[0] for s in spans]        # what a step writes
        self._clear = {}                                                  # addresses of gradients / outputs that were last found clear of it
        self._watch()

    def _watch(self):
        """Notes where the tensors are whose memory a program may exchange, and holds all that the descriptors name: an address that is still the same is the same memory."""
        states = [t for ts in (self.m, self.v, self.m_scale, self.v_scale) for t in ts or ()]
        theirs = states if self._callers else []
        self._watched = theirs + [t for t in (*self.params, *self.copies, *(self.grads or ())) if t is not None]
        self._watched_states = len(theirs)
        self._at = [*map(_address, self._watched)]
        self._held = [t.untyped_storage() for t in (self._watched if self._callers else self._watched + states)]

    def _follow(self, states_only: bool = False):
        """Takes tensors that have other memory than at the last look anew."""
        watched, at = self._watched, self._at
        if states_only and at is not None:
            watched, at = watched[:self._watched_states], at[:self._watched_states]
        if [*map(_address, watched)] != at:
            self._attach(self.m, self.v, self.m_scale, self.v_scale)
            if self.grads is not None:
                at, self._at = self._at, None              # (refused gradients: not taken, and refused again)
                self._bind(self.grads)
                self._at = at

    def set_state(self, m, v, t: int, m_scale=None, v_scale=None):
        """Takes flat tensors as the states THEMSELVES (no copy): fp32 moments, or int8 / uint8 codes with their scales [ceil(numel / 256)]; t: steps taken."""
        if int(t) < 0:
            raise HierTCNError(f"t = {t}")
        self._take((m, v, m_scale, v_scale))
        self.t = int(t)

    def _take(self, state):
        lists = [list(x) if x is not None else None for x in (*state, None, None)[:4]]
        if any(x is not None and len(x) != len(self.params) for x in lists) or None in lists[:2] or (self.state_bits == 8) != (None not in lists[2:]):
            raise HierTCNError("one m and one v per parameter, and a scale of each with 8-bit states only")
        before, self._callers = getattr(self, "_callers", True), True
        try:
            self._attach(*lists)
        except Exception:
            self._callers = before
            raise

    def state_dict(self) -> dict:
        """t, seed and the states on the host (checkpoints)."""
        out = dict(t=self.t, seed=self.seed, state_bits=self.state_bits, m=[x.cpu() for x in self.m], v=[x.cpu() for x in self.v])
        if self.state_bits == 8:
            out.update(m_scale=[x.cpu() for x in self.m_scale], v_scale=[x.cpu() for x in self.v_scale])
        return out

    def load_state_dict(self, state: dict):
        """Copies a state_dict() into the states."""
        names = ("m", "v") + (("m_scale", "v_scale") if self.state_bits == 8 else ())
        if int(state["state_bits"]) != self.state_bits or any(len(state[k]) != len(self.params) for k in names):
            raise HierTCNError("the state belongs to another optimizer (state_bits or number of tensors)")
        pairs = [(a, b) for k in names for a, b in zip(getattr(self, k), state[k])]
        if any(a.shape != b.shape or a.dtype != b.dtype for a, b in pairs):
            raise HierTCNError("the state belongs to other tensors")
        for a, b in pairs:
            a.copy_(b)
        self.t, self.seed = int(state["t"]), int(state["seed"])

    def _bind(self, grads):
        """All of them, or (an exception) none."""
        if len(grads) != len(self.params):
            raise HierTCNError(f"{len(self.params)} parameters, {len(grads)} gradients")
        found = []
        for i, (shape, g) in enumerate(zip(self._shapes, grads)):
            if g is not None and (not isinstance(g, torch.Tensor) or g.dtype not in _ops.DTYPE):
                raise HierTCNError(f"grads[{i}]: a float32, bfloat16 or float16 tensor")
            found.append((None, 0) if g is None else (need(g, f"grads[{i}]", g.dtype, self.device, shape).data_ptr(), _ops.DTYPE[g.dtype]))
        if self._clear.get("grads") != found:         # (sizes are the parameters')
            _clear_of(self._written, self._starts, "grads", [(ptr, k * (2 if dtype else 4)) for (ptr, dtype), k in zip(found, self._flat_numel)])
            self._clear["grads"] = found
        for d, (ptr, dtype) in zip(self._desc, found):
            d.grad, d.grad_dtype = ptr, dtype

    def step(self, grads: Optional[Sequence[Optional[torch.Tensor]]] = None, lr: Optional[float] = None, grad_scale: Union[float, torch.Tensor] = 1.0):
        """One step.  grads: this step's (default: the buffers given to the constructor); a parameter without one is left as it is.  grad_scale multiplies
        every gradient: a number, or a device float32 tensor of one element (clipping by the global norm)."""
        self._follow()
        if grads is not None:
            self._bind(grads)
        elif self.grads is None:
            raise HierTCNError("no gradients: give them to step() or to the constructor")
        a = _ops.Adamw(lr=self.lr if lr is None else float(lr), beta1=self.betas[0], beta2=self.betas[1], eps=self.eps, grad_scale=1.0, t=self.t + 1,
                       seed=self.seed, state_bits=self.state_bits)
        if isinstance(grad_scale, torch.Tensor):
            if grad_scale.numel() != 1:
                raise HierTCNError(f"grad_scale: {grad_scale.numel()} elements, expected one")
            a.grad_scale_dev = need(grad_scale, "grad_scale", torch.float32, self.device, grad_scale.shape).data_ptr()
        else:
            a.grad_scale = float(grad_scale)
        try:
            _ops.call(_ops.lib().hiertcn_adamw_step, self.device, self._desc, len(self._desc), C.byref(a))
        finally:
            if grads is not None and self.grads is not None:
                self._bind(self.grads)
        self.t += 1

    def moments(self, out=None):
        """-> (m, v): lists of flat fp32 tensors -- the states themselves (32 bits), or the values that the codes stand for, written to `out` = (list, list)
        where that is given (entries of None are skipped)."""
        n = len(self.params)
        if out is not None and (len(out[0]) != n or len(out[1]) != n):
            raise HierTCNError(f"{n} parameters, outputs for {len(out[0])} and {len(out[1])}")
        if self.state_bits == 32:
            if out is not None:
                for dst, src in zip((*out[0], *out[1]), (*self.m, *self.v)):
                    if dst is not None:
                        dst.copy_(src)
                return out
            return self.m, self.v
        self._follow(states_only=True)
        fresh = out is None
        if fresh:
            out = tuple([torch.empty(p.numel(), dtype=torch.float32, device=self.device) for p in self.params] for _ in range(2))
        found = [[None if o is None else need(o, "out", torch.float32, self.device, k).data_ptr() for o, k in zip(lst, self._flat)] for lst in out]
        if not fresh and self._clear.get("out") != found:
            _apart((("m out", out[0]), ("v out", out[1])))
            for name, ptrs in zip(("m out", "v out"), found):
                _clear_of(self._written, self._starts, name, [(ptr, 4 * k) for ptr, k in zip(ptrs, self._flat_numel)])
            self._clear["out"] = found
        _ops.call(_ops.lib().hiertcn_adamw_moments, self.device, self._desc, n, *((C.c_void_p * n)(*ptrs) for ptrs in found))
        return out
