"""Gated linear recurrence over the steps of a batch of sequences, and its gradients (``csrc/hip/recurrence.hip``).

    states[:, t] = gate[:, t] * states[:, t - 1] + w * x[:, t]        w = 1, or 1 - gate (``mix=True``)

Staged scores of a boosted ensemble are the recurrence over its trees without a gate (a running sum), those of a random
forest its mixed form with gates ``(k - 1) / k`` (a running mean); recurrent layers of sequence models have a gate per
channel or head.  Everything runs on torch's current stream of the tensors' device, can be captured into a HIP graph,
and gives the same bits every time.
"""
from __future__ import annotations

import struct

import torch

from ._args import core, fail, need_device, need_tensor, need_type, run, stream_of

_SCAN = struct.Struct("20q")
_SCAN_GRAD = struct.Struct("29q")


def _wide(t):
    return torch.float64 if t.dtype == torch.float64 else torch.float32


def _rows(t):
    """``t`` with a sequence step's channels next to each other."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check(op: str, x, code: int, gate, lengths, ends):
    """Checks what forward and backward share; returns (gate, gate type code, groups, the states at the ends, lengths)."""
    b, t, d = x.shape
    gate_code = groups = 0
    if gate is not None:
        gate = need_tensor(op, "gate", gate)
        gate_code = need_type(op, "gate", gate)
        if gate_code != code and not (gate_code == 2 and code < 2):
            fail(f"{op}: a gate of {gate.dtype} for values of {x.dtype}; it has to be of that type or, for 16-bit values, float32")
        if gate.dim() != 3 or gate.shape[0] not in (1, b) or gate.shape[1] != t:
            fail(f"{op}: the gate has to be [{b} or 1, {t}, groups], got {tuple(gate.shape)}")
        groups = gate.shape[2]
        if d and (groups < 1 or d % groups):
            fail(f"{op}: the width {d} is not a multiple of the gate's {groups} groups")
        gate = _rows(gate)
    checked = []
    for name, end in ends:
        if end is not None:
            end = need_tensor(op, name, end)
            if end.dtype != _wide(x) or end.shape != (b, d):
                fail(f"{op}: {name} has to be {_wide(x)} [{b}, {d}], got {end.dtype} {tuple(end.shape)}")
            end = end.contiguous()
        checked.append(end)
    if lengths is not None:
        lengths = need_tensor(op, "lengths", lengths)
        if lengths.dtype != torch.int32 or lengths.shape != (b,):
            fail(f"{op}: lengths have to be int32 [{b}], got {lengths.dtype} {tuple(lengths.shape)}")
        lengths = lengths.contiguous()
    return gate, gate_code, groups, checked, lengths


def _address(t) -> int:
    return 0 if t is None else t.data_ptr()


def _gate_steps(gate, batch: int):
    """Elements between the gates of neighbouring sequences and steps."""
    if gate is None:
        return 0, 0
    gate_b, gate_t, _ = gate.stride()
    return (gate_b if gate.shape[0] == batch else 0), gate_t


def gated_scan(x, gate=None, state=None, *, mix: bool = False, lengths=None):
    """All states of the recurrence: ``(states [batch, steps, width], last [batch, width])``.

    ``x``: [batch, steps, width] of bf16, fp16, fp32 or fp64.  ``gate``: [batch or 1, steps, groups] of ``x``'s type or
    float32, where channel ``d`` takes the gate of group ``d // (width / groups)``; ``None`` is a gate of one.  ``state``:
    the state before the first step (zeros if not given).  ``lengths``: int32 [batch]; behind a sequence's length (clamped to
    0 .. steps) the states are zero, ``last`` is the state after its last step, and what stands in ``x`` and ``gate`` there
    is not used.  States are carried in float32 (float64 for fp64), which is also the type of ``state`` and ``last``: feeding
    ``last`` back in continues a sequence, step by step or in pieces.  The product of a run of gates may
    leave the type's range either way; results are finite wherever the recurrence over absolute values is.
    """
    x = need_tensor("gated_scan", "x", x)
    code = need_type("gated_scan", "x", x)
    if x.dim() != 3:
        fail(f"gated_scan: x has to be [batch, steps, width], got {tuple(x.shape)}")
    gate, gate_code, groups, (state,), lengths = _check("gated_scan", x, code, gate, lengths, (("state", state),))
    if mix and gate is None:
        fail("gated_scan: the mixed form needs a gate")
    device = need_device("gated_scan", x, gate, state, lengths)
    lib = core()
    x = _rows(x)
    b, t, d = x.shape
    where = x.device
    states = torch.empty((b, t, d), dtype=x.dtype, device=where)
    last = torch.empty((b, d), dtype=_wide(x), device=where)
    if b and d:
        gate_b, gate_t = _gate_steps(gate, b)
        x_b, x_t, _ = x.stride()
        stream = stream_of(device)
        run(lib.lga_hip_gated_scan,
            lambda work: _SCAN.pack(x.data_ptr(), _address(gate) if t else 0, _address(state), _address(lengths), states.data_ptr(), last.data_ptr(),
                                    work, stream, device, b, t, d, x_b, x_t, gate_b, gate_t, groups, code, gate_code, bool(mix)), where)
    return states, last


def gated_scan_grad(grad_states, states, gate=None, state=None, *, x=None, grad_last=None, mix: bool = False, lengths=None):
    """Gradients of :func:`gated_scan`: ``(grad_x, grad_state, grad_gate)``.

    ``states`` is what the forward pass gave back; ``gate``, ``state``, ``mix`` and ``lengths`` are what it got, and ``x``
    too if it was the mixed form.  ``grad_states`` and ``grad_last`` are the gradients of its two results (``grad_last`` may
    be left out).  ``grad_x`` has the type of ``states``, ``grad_state`` is float32 (float64), ``grad_gate`` has the gate's
    type and shape - summed over the channels and sequences that shared a gate - and is ``None`` without one.  Behind a
    sequence's length all of them are zero.
    """
    grad_states = need_tensor("gated_scan_grad", "grad_states", grad_states)
    states = need_tensor("gated_scan_grad", "states", states)
    x = None if x is None else need_tensor("gated_scan_grad", "x", x)
    code = need_type("gated_scan_grad", "states", states)
    if states.dim() != 3:
        fail(f"gated_scan_grad: states have to be [batch, steps, width], got {tuple(states.shape)}")
    for name, like in (("grad_states", grad_states), ("x", x)):
        if like is not None and (like.dtype != states.dtype or like.shape != states.shape):
            fail(f"gated_scan_grad: {name} has to be {states.dtype} {tuple(states.shape)} as the states, got {like.dtype} {tuple(like.shape)}")
    gate, gate_code, groups, (state, grad_last), lengths = _check("gated_scan_grad", states, code, gate, lengths, (("state", state), ("grad_last", grad_last)))
    if mix and (gate is None or x is None):
        fail("gated_scan_grad: the mixed form needs the gate and x")
    device = need_device("gated_scan_grad", states, grad_states, x, gate, state, grad_last, lengths)
    lib = core()
    grad_states, states, x = _rows(grad_states), _rows(states), _rows(x) if mix else None
    b, t, d = states.shape
    where = states.device
    grad_x = torch.empty((b, t, d), dtype=states.dtype, device=where)
    grad_state = torch.empty((b, d), dtype=_wide(states), device=where)
    grad_gate = None if gate is None else torch.empty(gate.shape, dtype=gate.dtype, device=where)
    if b and d:
        gate_b, gate_t = _gate_steps(gate, b)
        (g_b, g_t, _), (h_b, h_t, _), (x_b, x_t, _) = grad_states.stride(), states.stride(), x.stride() if mix else (0, 0, 0)
        stream = stream_of(device)
        gates = 0 if gate is None else gate.shape[0]
        run(lib.lga_hip_gated_scan_grad,
            lambda work: _SCAN_GRAD.pack(grad_states.data_ptr(), states.data_ptr(), _address(gate) if t else 0, _address(state), _address(x),
                                         _address(grad_last), _address(lengths), grad_x.data_ptr(), grad_state.data_ptr(), _address(grad_gate), work,
                                         stream, device, b, t, d, g_b, g_t, h_b, h_t, x_b, x_t, gate_b, gate_t, groups, gates, code, gate_code,
                                         bool(mix)), where)
    elif grad_gate is not None:
        grad_gate.zero_()
    return grad_x, grad_state, grad_gate
