"""ctypes view of include/lobpolicy.h: struct layouts and function prototypes (rl4mm_amd/policy_ops.py is what a caller uses)."""
from __future__ import annotations

import ctypes as C

from ._capi import LobsimError

ABI_VERSION = 1  # LOBPOLICY_ABI_VERSION of the header this file mirrors
MAX_HEAD, MAX_WIDTH = 128, 8192
MAX_HEADS, MAX_UNITS, MAX_TENSORS = 1 << 16, 1 << 22, 1_000_000  # heads, environments x heads, tensors of one clip: what the entries check
F32, BF16 = 0, 1


class Operand(C.Structure):
    _fields_ = [("data", C.c_void_p), ("stride_t", C.c_int64), ("stride_n", C.c_int64), ("stride_h", C.c_int64)]


class Attention(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32), ("heads", C.c_int32), ("dk", C.c_int32), ("dv", C.c_int32),
        ("steps", C.c_int64), ("envs", C.c_int64),
        ("q", Operand), ("k", Operand), ("v", Operand), ("out", Operand),
        ("grad_q", Operand), ("grad_k", Operand), ("grad_v", Operand),
        ("log_decay", C.c_void_p), ("reset", C.c_void_p), ("reset_stride_t", C.c_int64), ("reset_stride_n", C.c_int64),
        ("lengths", C.c_void_p), ("skip", C.c_void_p),
        ("state_in", C.c_void_p), ("state_out", C.c_void_p), ("grad_state_out", C.c_void_p), ("grad_state_in", C.c_void_p),
        ("scale", C.c_float), ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64), ("forward_workspace", C.c_void_p),
    ]  # fmt: skip


class Block(C.Structure):
    _fields_ = [
        ("stream_dtype", C.c_int32), ("dtype", C.c_int32), ("rows", C.c_int64), ("width", C.c_int64),
        ("x", C.c_void_p), ("block", C.c_void_p), ("gate", C.c_void_p),
        ("x_stride", C.c_int64), ("block_stride", C.c_int64), ("gate_stride", C.c_int64),
        ("post", C.c_void_p), ("res", C.c_void_p), ("pre", C.c_void_p), ("eps", C.c_float),
        ("y", C.c_void_p), ("z", C.c_void_p), ("grad_y", C.c_void_p), ("grad_z", C.c_void_p), ("grad_y_stride", C.c_int64), ("grad_z_stride", C.c_int64),
        ("grad_x", C.c_void_p), ("grad_block", C.c_void_p), ("grad_gate", C.c_void_p),
        ("grad_post", C.c_void_p), ("grad_res", C.c_void_p), ("grad_pre", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64),
    ]  # fmt: skip


_PA, _PB = C.POINTER(Attention), C.POINTER(Block)
# name -> (restype, argtypes); the names without their lobpolicy_ prefix
PROTOTYPES = {
    "abi_version": (C.c_int, []),
    "last_error": (C.c_char_p, []),
    "attention_workspace": (C.c_int64, [_PA]),
    "attention_forward": (C.c_int, [_PA, C.c_void_p]),
    "attention_backward": (C.c_int, [_PA, C.c_void_p]),
    "attention_step": (C.c_int, [_PA, C.c_void_p]),
    "block_workspace": (C.c_int64, [_PB]),
    "block_forward": (C.c_int, [_PB, C.c_void_p]),
    "block_backward": (C.c_int, [_PB, C.c_void_p]),
    "clip_workspace": (C.c_int64, [C.c_void_p, C.c_void_p, C.c_int64]),
    "clip": (C.c_int, [C.c_void_p, C.c_void_p, C.c_void_p, C.c_int64, C.c_int32, C.c_double, C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]),
}


class Binding:
    """The entry points of one library, each with its prototype; raises if a declared symbol is missing."""

    def __init__(self, path):
        self.lib = C.CDLL(str(path))
        self.fn = {}
        for name, (res, args) in PROTOTYPES.items():
            f = getattr(self.lib, "lobpolicy_" + name)
            f.restype, f.argtypes = res, args
            self.fn[name] = f
        got = self.fn["abi_version"]()
        if got != ABI_VERSION:
            raise LobsimError(f"{path}: lobpolicy_abi_version() = {got}, this binding mirrors include/lobpolicy.h at version {ABI_VERSION}: rebuild the library")

    def check(self, code, what):
        """`code`, or LobsimError with the library's message where it is negative."""
        if code < 0:
            raise LobsimError(f"lobpolicy_{what} failed ({code}): {(self.fn['last_error']() or b'').decode()}")
        return code
