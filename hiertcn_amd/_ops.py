"""ctypes binding of include/hiertcn_ops.h (the sequence operators; exported by the same libhiertcn_gfx950.so as the model handles)."""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib
from ._lib import HierTCNError

VERSION = 1
DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

_p, _i32, _i64, _f, _d, _sz = C.c_void_p, C.c_int32, C.c_int64, C.c_float, C.c_double, C.c_size_t


class Glr(C.Structure):
    """hiertcn_glr_t"""
    _fields_ = [("B", _i64), ("T", _i64), ("D", _i64), ("dtype", _i32), ("cand_act", _i32),
                ("gate", _p), ("gate_sb", _i64), ("gate_st", _i64), ("cand", _p), ("cand_sb", _i64), ("cand_st", _i64),
                ("mask", _p), ("mask_sb", _i64), ("mask_st", _i64), ("lengths", _p),
                ("state_in", _p), ("state_out", _p), ("record", _p), ("out", _p), ("out_sb", _i64), ("out_st", _i64),
                ("dout", _p), ("dout_sb", _i64), ("dout_st", _i64), ("dstate_out", _p),
                ("dgate", _p), ("dgate_sb", _i64), ("dgate_st", _i64), ("dcand", _p), ("dcand_sb", _i64), ("dcand_st", _i64),
                ("dstate_in", _p), ("workspace", _p), ("workspace_bytes", _sz)]


class Rows(C.Structure):
    """hiertcn_rows_t"""
    _fields_ = [("n", _i64), ("T", _i64), ("V", _i64), ("dtype", _i32), ("reserved", _i32), ("logits", _p), ("ld", _i64), ("ids", _p), ("logp", _p),
                ("dlogits", _p), ("dld", _i64), ("grad_scale", _f), ("workspace", _p), ("workspace_bytes", _sz)]


class Preference(C.Structure):
    """hiertcn_preference_t"""
    _fields_ = [("kind", _i32), ("average", _i32), ("beta", _f), ("smoothing", _f), ("ref", _p), ("loss", _p), ("pair_loss", _p), ("margin", _p), ("seq_logp", _p)]


class Policy(C.Structure):
    """hiertcn_policy_t"""
    _fields_ = [("mean", _i32), ("reserved", _i32), ("clip_low", _f), ("clip_high", _f), ("kl_coef", _f), ("old_logp", _p), ("ref_logp", _p),
                ("advantage", _p), ("adv_sn", _i64), ("adv_st", _i64), ("loss", _p), ("kl", _p), ("clipped", _p)]


class AdamwTensor(C.Structure):
    """hiertcn_adamw_tensor_t"""
    _fields_ = [("numel", _i64), ("param", _p), ("grad", _p), ("grad_dtype", _i32), ("copy_dtype", _i32), ("copy", _p), ("m", _p), ("v", _p),
                ("m_scale", _p), ("v_scale", _p), ("weight_decay", _f), ("index", _i32)]


class Adamw(C.Structure):
    """hiertcn_adamw_t"""
    _fields_ = [("lr", _d), ("beta1", _d), ("beta2", _d), ("eps", _d), ("grad_scale", _d), ("grad_scale_dev", _p), ("t", _i64), ("seed", _i64),
                ("state_bits", _i32), ("reserved", _i32)]


STRUCTS = (Glr, Rows, Preference, Policy, AdamwTensor, Adamw)

# every symbol include/hiertcn_ops.h declares: (restype, argtypes)
SYMBOLS = {
    "hiertcn_ops_version": (C.c_int, []),
    "hiertcn_ops_last_error": (C.c_char_p, []),
    "hiertcn_ops_struct_sizes": (C.c_int, [C.POINTER(_sz)]),
    "hiertcn_glr_record_floats": (_sz, [_i64, _i64, _i64]),
    "hiertcn_glr_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "hiertcn_glr_forward": (C.c_int, [C.POINTER(Glr), _p]),
    "hiertcn_glr_backward": (C.c_int, [C.POINTER(Glr), _p]),
    "hiertcn_rows_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "hiertcn_sequence_logp": (C.c_int, [C.POINTER(Rows), _p]),
    "hiertcn_preference_loss": (C.c_int, [C.POINTER(Rows), C.POINTER(Preference), _p]),
    "hiertcn_policy_loss": (C.c_int, [C.POINTER(Rows), C.POINTER(Policy), _p]),
    "hiertcn_adamw_step": (C.c_int, [C.POINTER(AdamwTensor), _i64, C.POINTER(Adamw), _p]),
    "hiertcn_adamw_moments": (C.c_int, [C.POINTER(AdamwTensor), _i64, C.POINTER(_p), C.POINTER(_p), _p]),
    "hiertcn_train_masters_changed": (C.c_int, [_p, _p]),
}

_bound = None


def lib():
    """The loaded library with the operators' prototypes set (raises where it is missing or of another version: there is no fallback)."""
    global _bound
    if _bound is None:
        _bound = bind(_lib.load())
    return _bound


def bind(so):
    for name, (res, args) in SYMBOLS.items():
        fn = getattr(so, name)
        fn.restype = res
        fn.argtypes = args
    if so.hiertcn_ops_version() != VERSION:
        raise HierTCNError(f"operator ABI mismatch: library {so.hiertcn_ops_version()} vs binding {VERSION}")
    return so


def check(rc: int):
    if rc != 0:
        msg = lib().hiertcn_ops_last_error()
        raise HierTCNError(f"hiertcn call failed ({rc}): {msg.decode() if msg else '?'}")


def need(t, name, dtype, device, shape, contiguous=True):
    """The argument check of the operators: type, place, element type, shape and layout of a tensor."""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device and t.shape == shape and (not contiguous or t.is_contiguous()):
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype != dtype:
        raise HierTCNError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if t.device != device:
        raise HierTCNError(f"{name}: on {t.device}, expected {device}")
    if t.shape != shape:
        raise HierTCNError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    raise HierTCNError(f"{name}: must be contiguous")


def on_gpu(t, name):
    """The device of the call: that of its first tensor, which has to be a GPU."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor")
    if t.dtype not in DTYPE:
        raise HierTCNError(f"{name}: dtype {t.dtype}: float32, bfloat16 or float16")
    if not t.is_cuda:
        raise HierTCNError(f"{name}: must live on the GPU (got {t.device})")
    return t.device


def call(fn, device, *args):
    """fn(*args, stream) on `device` and its current stream, whatever the current device is."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))     # (torch.cuda.current_stream(device).cuda_stream without building the Stream object)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc != 0:
        check(rc)


@functools.lru_cache(maxsize=4096)
def size(name, *dims):
    """A workspace or record size of the library: a function of the dimensions alone."""
    return getattr(lib(), name)(*dims)


def workspace(nbytes, device):
    """Scratch of ONE call: taken from torch's allocator each time (a graph that captures the call owns its own), None where none is needed."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
