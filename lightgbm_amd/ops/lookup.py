"""Row lookup by token and its gradient (``csrc/hip/lookup.hip``).

A tree ensemble's raw score is a sum of looked-up leaf values (tokens: leaf indices, table: one row per leaf), and the
gradient of a leaf value is the sum of the gradients of the rows in the leaf; an embedding layer does the same with
words.  Both run on torch's current stream of the tensors' device, can be captured into a HIP graph, and give the same
bits every time for the same sizes, strides and values.
"""
from __future__ import annotations

import struct

import torch

from ._args import core, fail, need_device, need_tensor, need_type, run, stream_of, two_dims, type_code

_LOOKUP = struct.Struct("14qd")
_LOOKUP_GRAD = struct.Struct("17qd")
_MAX_TOKENS = 2**31 - 1


def _check_ids(op: str, ids):
    ids = need_tensor(op, "ids", ids)
    if ids.dtype not in (torch.int32, torch.int64):
        fail(f"{op}: ids have to be int32 or int64, got {ids.dtype}")
    if ids.numel() > _MAX_TOKENS:
        fail(f"{op}: {ids.numel()} ids; at most 2^31 - 1 in one call")
    return ids, int(ids.dtype == torch.int64)


def embedding(table, ids, scale: float = 1.0):
    """``scale * table[ids]``: ``table`` [rows, width], ``ids`` int32 / int64 of any shape -> ``[*ids.shape, width]`` of
    the table's type (bf16, fp16, fp32, fp64).

    An id outside ``0 .. rows - 1`` (a padding token) gives a row of zeros.  The product is taken in 32 bits (64 for
    fp64) and rounded once.  Strided tables and ids are read in place as long as a row's values are neighbours and the
    ids' dimensions merge to two; otherwise they are copied first.
    """
    table = need_tensor("embedding", "table", table)
    code = need_type("embedding", "table", table)
    if table.dim() != 2:
        fail(f"embedding: the table has to be [rows, width], got {tuple(table.shape)}")
    ids, wide_ids = _check_ids("embedding", ids)
    device = need_device("embedding", table, ids)
    lib = core()
    rows, width = table.shape
    if width > 1 and table.stride(1) != 1:
        table = table.contiguous()
    out = torch.empty((*ids.shape, width), dtype=table.dtype, device=table.device)
    if out.numel():
        view = two_dims(ids.shape, ids.stride())
        if view is None:
            ids = ids.contiguous()
            view = two_dims(ids.shape, ids.stride())
        (n0, n1), ((s0, s1),) = view
        run(lib.lga_hip_embedding,
            lambda work: _LOOKUP.pack(table.data_ptr(), ids.data_ptr(), out.data_ptr(), stream_of(device), device, rows, width, table.stride(0),
                                      n0, n1, s0, s1, code, wide_ids, float(scale)), table.device)
    return out


def embedding_grad(grad, ids, num_rows: int, scale: float = 1.0, dtype=None):
    """Gradient of :func:`embedding` for its table: ``out[v] = scale * sum of grad[i] over all i with ids[i] = v``,
    ``[num_rows, width]``; rows that no id names are zero, ids outside the table are left out.

    ``grad``: ``[*ids.shape, width]`` (an expanded tensor is read in place).  ``dtype``: the result's type, ``grad``'s own
    or float32; the sums are held in 32 bits (64 for fp64); ``scale`` has to be finite.  A row's gradients are added up in
    an order that the sizes, strides and ids determine, never the timing: sorted and strip by strip, or in partial sums of
    waves where the tokens are few or outnumber the rows.
    """
    grad = need_tensor("embedding_grad", "grad", grad)
    code = need_type("embedding_grad", "grad", grad)
    ids, wide_ids = _check_ids("embedding_grad", ids)
    if grad.dim() != ids.dim() + 1 or grad.shape[:-1] != ids.shape:
        fail(f"embedding_grad: grad has to be [*ids.shape, width], got {tuple(grad.shape)} for ids {tuple(ids.shape)}")
    if isinstance(num_rows, bool) or int(num_rows) != num_rows or not 0 <= num_rows < 2**31 - 1:
        fail(f"embedding_grad: num_rows has to be a whole number from 0 to 2^31 - 2, got {num_rows!r}")
    num_rows = int(num_rows)
    out_type = grad.dtype if dtype is None else dtype
    out_code = type_code(out_type)
    if out_code < 0 or out_code != code and not (out_code == 2 and code < 2):
        fail(f"embedding_grad: a gradient of {grad.dtype} can be given back as that type or float32, not as {out_type}")
    device = need_device("embedding_grad", grad, ids)
    lib = core()
    width = grad.shape[-1]
    if width > 1 and grad.stride(-1) != 1:
        grad = grad.contiguous()
    if not ids.numel():
        ids, grad = ids.reshape(0), grad.reshape(0, width)
    view = two_dims(ids.shape, ids.stride(), grad.stride()[:-1])
    if view is None:
        ids, grad = ids.contiguous(), grad.contiguous()
        view = two_dims(ids.shape, ids.stride(), grad.stride()[:-1])
    (n0, n1), ((s0, s1), (g0, g1)) = view
    out = torch.empty((num_rows, width), dtype=out_type, device=grad.device)
    if out.numel():
        run(lib.lga_hip_embedding_grad,
            lambda work: _LOOKUP_GRAD.pack(grad.data_ptr(), ids.data_ptr(), out.data_ptr(), work, stream_of(device), device, num_rows, width,
                                           n0, n1, s0, s1, g0, g1, code, out_code, wide_ids, float(scale)), grad.device)
    return out
