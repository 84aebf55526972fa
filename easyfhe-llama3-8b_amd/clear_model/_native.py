"""ctypes binding of libclear_mi355x.so (include/clear_mi355x.h).

The library is the only compute path of rotary positions, attention and the
vocabulary loss: if it is missing this module raises at import, and none of
them falls back to torch's own operators.  (``ClearDecoder`` does its norms,
projections and SiLU with torch.)  The operators take torch tensors, and torch
is imported first: the library binds to the HIP runtime that torch has loaded.
"""

from __future__ import annotations

import ctypes
import struct
from pathlib import Path

import torch

_LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libclear_mi355x.so"

CLEAR_OK = 0
CLEAR_EINVAL = 1
CLEAR_ERUNTIME = 2

TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}

# The argument structs of the header, every field 8 bytes: pointers and
# integers q / Q, floating point d.
ROPE_ARGS = struct.Struct("<6Q10q8q")
ATTENTION_ARGS = struct.Struct("<12Qq8qd12q")
LOSS_ARGS = struct.Struct("<9Qq5q2q")

VP = ctypes.c_void_p
I = ctypes.c_int
I64 = ctypes.c_int64
I64P = ctypes.POINTER(ctypes.c_int64)
ARGS = ctypes.c_char_p

# name -> (restype, argtypes); every function declared in include/clear_mi355x.h
SIGNATURES = {
    "clear_last_error": (ctypes.c_char_p, []),
    "clear_rope": (I, [ARGS, VP]),
    "clear_attention_workspace": (I, [ARGS, I64, I64P]),
    "clear_attention_forward": (I, [ARGS, VP]),
    "clear_attention_backward": (I, [ARGS, VP]),
    "clear_loss_workspace": (I, [ARGS, I64, I64P]),
    "clear_loss_forward": (I, [ARGS, VP]),
    "clear_loss_backward": (I, [ARGS, VP]),
}


def library_path() -> Path:
    return _LIB_PATH


def _load():
    if not _LIB_PATH.exists():
        raise ImportError(
            f"{_LIB_PATH} is missing: build the gfx950 libraries first "
            "(python __graft_entry__.py build, or python easyfhe-llama3-8b_amd/build.py)"
        )
    lib = ctypes.CDLL(str(_LIB_PATH))
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    return lib


lib = _load()


class OperatorError(RuntimeError):
    """Runtime failure reported by the library."""


def check(rc: int) -> None:
    if rc == CLEAR_OK:
        return
    msg = (lib.clear_last_error() or b"").decode()
    if rc == CLEAR_EINVAL:
        raise ValueError(msg)
    raise OperatorError(msg)


_grad_enabled = torch.is_grad_enabled


def without_graph(name: str, x, y=None, z=None) -> None:
    """The plain entry points leave no graph: refused where one would be missed.
    (Written out: a generator over the tensors would cost a small call 1 us.)"""
    if _grad_enabled() and (x.requires_grad or y is not None and y.requires_grad
                            or z is not None and z.requires_grad):
        raise ValueError(f"a tensor requires gradients: use {name} for them, or torch.no_grad().")


# torch's own compiled code asks for the current stream's handle this way; the
# public route through a Stream object costs 2 us, a tenth of a small call.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)

_current_device = torch.cuda.current_device


def call(fn, args: bytes, index: int) -> None:
    """Enqueue on the current stream of device `index`."""
    if _current_device() == index:
        rc = fn(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(args, _raw_stream(index))
    if rc:
        check(rc)


def query(fn, args: bytes, backward: bool) -> int:
    n = ctypes.c_int64()
    check(fn(args, int(backward), ctypes.byref(n)))
    return n.value
