"""Checks and layouts shared by the row lookup and the gated recurrence."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from .. import _lib
from .._lib import LightGBMError

_core = None
_TYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2, torch.float64: 3}


def core():
    """The HIP core; raises where there is none."""
    global _core
    if _core is None:
        lib, hip = _lib.load()
        if not hip:
            raise LightGBMError("lightgbm_amd.ops needs the HIP build and a visible GPU")
        _core = lib
    return _core


def type_code(dtype) -> int:
    """0..3 for bf16, fp16, fp32, fp64; -1 for every other type."""
    return _TYPE_CODES.get(dtype, -1)


def fail(what: str):
    raise LightGBMError(what)


def need_tensor(op: str, name: str, t):
    """``t`` as its memory has to be read: a lazily negated view (``z.conj().imag``) is written out."""
    if not isinstance(t, torch.Tensor):
        fail(f"{op}: {name} has to be a torch tensor, got {type(t).__name__}")
    if t.requires_grad and torch.is_grad_enabled():
        fail(f"{op}: {name} requires grad, and nothing is recorded here: call it under torch.no_grad() and take the gradient from {op}_grad")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        fail(f"{op}: {name} is a dual tensor, and its tangent would be lost here: pass its primal value")
    if not t.data_ptr() and t.numel():
        fail(f"{op}: {name} has no memory (its storage was released)")
    return t.resolve_neg() if t.is_neg() else t


def need_type(op: str, name: str, t) -> int:
    code = _TYPE_CODES.get(t.dtype, -1)
    if code < 0:
        fail(f"{op}: {name} has to be bfloat16, float16, float32 or float64, got {t.dtype}")
    return code


def need_device(op: str, first, *others) -> int:
    """All tensors on one GPU; returns its index."""
    device = first.get_device()            # -1 on the CPU; the device object's words are only looked at for a message
    for t in others:
        if t is not None and t.get_device() != device:
            fail(f"{op}: tensors on {first.device} and {t.device}")
    if not first.is_cuda:
        fail(f"{op}: needs tensors on the GPU, got {first.device}")
    return device


# The current stream's handle without a Python Stream object around it (2 us less a call), where torch offers that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device: int) -> int:
    return _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream


def run(fn, pack, device) -> None:
    """Calls the core with the words that ``pack(address of the workspace)`` gives.  Without a workspace the core launches
    only what needs none and says how much is missing."""
    need = ctypes.c_int64()
    if fn(pack(0), need):
        _lib.check(-1)
    if need.value:
        work = torch.empty(need.value, dtype=torch.uint8, device=device)
        if fn(pack(work.data_ptr()), need):
            _lib.check(-1)


def two_dims(shape, *strides):
    """Merges neighbouring dimensions that every stride tuple walks evenly.  Returns (sizes, [strides, ...]) of two
    dimensions, or None if more are left."""
    if len(shape) == 1:
        return (1, shape[0]), [(0, s[0]) for s in strides]
    sizes, kept = [], [[] for _ in strides]
    for d, n in enumerate(shape):
        if n == 1:
            continue
        if sizes and all(k[-1] == n * s[d] for k, s in zip(kept, strides)):
            sizes[-1] *= n
            for k, s in zip(kept, strides):
                k[-1] = s[d]
        else:
            sizes.append(n)
            for k, s in zip(kept, strides):
                k.append(s[d])
    if len(sizes) > 2:
        return None
    while len(sizes) < 2:
        sizes.insert(0, 1)
        for k in kept:
            k.insert(0, 0)
    return sizes, kept
