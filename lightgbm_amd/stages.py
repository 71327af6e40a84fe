"""All stages of an ensemble at once: the scores after 1, 2, ..., n iterations, and refitting leaf values through them.

The raw score after iteration k is a linear recurrence over the iterations whose inputs are looked-up leaf values,

    score_k = a_k * score_(k-1) + b_k * leaf_value[leaf_k(row)]

with a = b = 1 for boosting and the running mean a_k = (k - 1) / k, b_k = 1 / k for random forests.  On the GPU that is
``ops.embedding`` (tokens: the leaves of all trees, numbered one after the other) followed by ``ops.gated_scan``, and the
gradient of a loss on the stages reaches the leaf values through ``ops.gated_scan_grad`` and ``ops.embedding_grad``; on
the CPU the same sums run in NumPy.  Everything is fp64.

The reference draws staged predictions of boosting and bagging side by side (bagging_boosting.ipynb:136, 194-212).
"""
from __future__ import annotations

from typing import Iterator, List, Optional, Tuple

import numpy as np

from . import _lib
from ._lib import LightGBMError, check

_BLOCK_VALUES = 1 << 28        # values of one staged array that are worked on at a time (2 GiB of fp64)


class _Forest:
    """Leaf values and leaf indices of the iterations [first, first + count) of a booster."""

    def __init__(self, booster, start_iteration: int, num_iteration: Optional[int]):
        from .models.ensemble import TreeEnsemble
        trees = TreeEnsemble.from_booster(booster).trees
        self.classes = booster.num_model_per_iteration()
        total = len(trees) // self.classes
        self.first = max(0, min(int(start_iteration), total))
        if num_iteration is None:
            num_iteration = booster.best_iteration if booster.best_iteration > 0 else -1
        self.count = total - self.first if num_iteration <= 0 else min(total - self.first, int(num_iteration))
        used = trees[self.first * self.classes:(self.first + self.count) * self.classes]
        sizes = [len(t.leaf_value) for t in used]
        self.offsets = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int64)
        self.values = np.concatenate([t.leaf_value for t in used]) if used else np.zeros(0)
        if len(self.values) >= 2**31 - 1:
            raise LightGBMError("the model has too many leaves to number them in 32 bits")
        info = booster.objective_info()
        self.objective, self.sigmoid, self.average = info["objective"], info["sigmoid"], info["average_output"]
        self.booster = booster

    def tokens(self, mat) -> np.ndarray:
        """Leaf tokens, int32 [rows, iterations * classes]."""
        leaf = self.booster.predict(mat, start_iteration=self.first, num_iteration=self.count, pred_leaf=True)
        return leaf + self.offsets[:-1].astype(np.int32)

    def blocks(self, mat, arrays: int) -> Iterator[Tuple[int, int]]:
        rows = mat.shape[0]
        step = max(1, _BLOCK_VALUES // max(1, self.count * self.classes * arrays))
        for at in range(0, rows, step):
            yield at, min(rows, at + step)

    def gates(self) -> Optional[np.ndarray]:
        """One gate per iteration, or None where the scores just add up."""
        if not self.average:
            return None
        k = np.arange(1, self.count + 1, dtype=np.float64)
        return (k - 1) / k


def _matrix(booster, data):
    from .basic import _encode_pandas_categories, _is_torch, _to_matrix
    from .basic import Dataset
    if isinstance(data, Dataset):
        raise TypeError("Cannot predict a Dataset; pass the raw matrix")
    raw, _, _ = _encode_pandas_categories(data, booster.pandas_categorical)
    mat, _ = _to_matrix(raw)
    return mat.cpu().numpy() if _is_torch(mat) else mat


def _on_gpu(device: Optional[str], work: int) -> bool:
    _, hip = _lib.load()
    if device not in (None, "cpu", "gpu"):
        raise LightGBMError(f"device has to be 'cpu' or 'gpu', got {device!r}")
    if device == "gpu" and not hip:
        raise LightGBMError("device='gpu' needs the HIP build and a visible GPU")
    return hip and (device == "gpu" or device is None and work >= 2_000_000)


def _link(raw, objective: str, sigmoid: float, lib):
    """Raw scores [..., classes] -> predictions; ``lib`` is numpy or torch."""
    words = objective.split()
    kind = words[0]
    if kind == "multiclass":
        top = raw.max(axis=-1, keepdims=True) if lib is np else raw.amax(dim=-1, keepdim=True)
        e = lib.exp(raw - top)
        return e / (e.sum(axis=-1, keepdims=True) if lib is np else e.sum(dim=-1, keepdim=True))
    if kind in ("binary", "multiclassova"):
        return 1.0 / (1.0 + lib.exp(-sigmoid * raw))
    if kind in ("cross_entropy", "xentropy"):
        return 1.0 / (1.0 + lib.exp(-raw))
    if kind in ("poisson", "gamma", "tweedie"):
        return lib.exp(raw)
    if kind == "regression" and "sqrt" in words:
        return lib.sign(raw) * raw * raw
    return raw


def _stages_cpu(forest: _Forest, tokens: np.ndarray, values: np.ndarray) -> np.ndarray:
    """Raw scores [iterations, rows, classes]."""
    x = values[tokens].reshape(len(tokens), forest.count, forest.classes).transpose(1, 0, 2)
    out = np.cumsum(x, axis=0)
    if forest.average:
        out /= np.arange(1, forest.count + 1, dtype=np.float64).reshape(-1, 1, 1)
    return out


def _by_stage(forest: _Forest, tokens):
    """Token tensor [rows, iterations * classes] seen as [iterations, rows, classes]."""
    return tokens.view(tokens.shape[0], forest.count, forest.classes).transpose(0, 1)


def _stages_gpu(forest: _Forest, tokens, values, gate):
    """Raw scores [iterations, rows, classes]; ``values`` fp64 [leaves, 1] on the GPU."""
    from . import ops
    x = ops.embedding(values, _by_stage(forest, tokens))
    states, _ = ops.gated_scan(x.view(1, forest.count, -1), gate, mix=gate is not None)
    return states.view(forest.count, tokens.shape[0], forest.classes)


def staged_predict(booster, data, start_iteration: int = 0, num_iteration: Optional[int] = None, raw_score: bool = False,
                   device: Optional[str] = None) -> np.ndarray:
    mat = _matrix(booster, data)
    forest = _Forest(booster, start_iteration, num_iteration)
    rows = mat.shape[0]
    out = np.empty((forest.count, rows, forest.classes), dtype=np.float64)
    if out.size:
        gpu = _on_gpu(device, out.size)
        if gpu:
            import torch
            values = torch.from_numpy(forest.values).cuda().view(-1, 1)
            gates = forest.gates()
            gate = None if gates is None else torch.from_numpy(gates).cuda().view(1, -1, 1)
        for lo, hi in forest.blocks(mat, 1):
            tokens = forest.tokens(mat[lo:hi])
            if gpu:
                raw = _stages_gpu(forest, torch.from_numpy(tokens).cuda(), values, gate)
                out[:, lo:hi] = (raw if raw_score else _link(raw, forest.objective, forest.sigmoid, torch)).cpu().numpy()
            else:
                raw = _stages_cpu(forest, tokens, forest.values)
                out[:, lo:hi] = raw if raw_score else _link(raw, forest.objective, forest.sigmoid, np)
    return out[:, :, 0] if forest.classes == 1 else out


# -- refitting --------------------------------------------------------------------------------------------------------

# Largest curvature of the loss in a raw score: with it in place of the true one a step never overshoots.
_CURVATURE = {"regression": lambda sigmoid: 1.0, "binary": lambda sigmoid: sigmoid * sigmoid / 4.0, "multiclass": lambda sigmoid: 0.5}


def _slopes(raw, target, forest: _Forest, lib):
    """d loss / d raw score, [iterations, rows, classes]; target [rows, classes] (multiclass: one-hot)."""
    kind = forest.objective.split()[0]
    if kind == "regression":
        return raw - target
    if kind == "binary":
        return forest.sigmoid * (_link(raw, forest.objective, forest.sigmoid, lib) - target)
    return _link(raw, forest.objective, forest.sigmoid, lib) - target


def refit_stages(booster, data, label, weight=None, num_steps: int = 20, learning_rate: float = 1.0, lambda_l2: float = 0.0, stages: str = "all",
                 device: Optional[str] = None):
    from .basic import Booster, _to_1d
    mat = _matrix(booster, data)
    rows = mat.shape[0]
    forest = _Forest(booster, 0, -1)
    kind = forest.objective.split()[0]
    if kind not in _CURVATURE or "sqrt" in forest.objective.split():
        raise LightGBMError(f"refit_stages supports the objectives regression, binary and multiclass, not {forest.objective!r}")
    if forest.average:
        raise LightGBMError("refit_stages is not defined for averaged (boosting=rf) models")
    if stages not in ("all", "last"):
        raise LightGBMError(f"refit_stages: stages has to be 'all' or 'last', got {stages!r}")
    if int(num_steps) != num_steps or num_steps < 0:
        raise LightGBMError(f"refit_stages: num_steps has to be a whole number >= 0, got {num_steps!r}")
    if not 0.0 < learning_rate <= 2.0:
        raise LightGBMError(f"refit_stages: learning_rate has to be in (0, 2], got {learning_rate!r}")
    if not 0.0 <= lambda_l2 < np.inf:
        raise LightGBMError(f"refit_stages: lambda_l2 has to be a number >= 0, got {lambda_l2!r}")
    y = _to_1d(label, np.float64)
    w = np.ones(rows) if weight is None else _to_1d(weight, np.float64)
    if len(y) != rows or len(w) != rows:
        raise LightGBMError("refit_stages: the label's or the weights' length differs from the number of rows")
    if not np.isfinite(y).all():          # one NaN would reach every leaf that shares a row with its own
        raise LightGBMError("refit_stages: the labels have to be finite")
    if kind == "binary":
        y = (y > 0).astype(np.float64)
    target = y.reshape(-1, 1)
    if kind == "multiclass":
        if rows and (y.min() < 0 or y.max() >= forest.classes or (y != np.floor(y)).any()):
            raise LightGBMError("refit_stages: multiclass labels have to be whole numbers from 0 to num_class - 1")
        target = np.eye(forest.classes)[y.astype(np.int64)]
    out = Booster(model_str=booster.model_to_string(num_iteration=-1))
    if rows == 0 or forest.count == 0 or num_steps == 0:
        return out
    total = float(w.sum())
    if not (w >= 0).all() or not 0 < total < np.inf:
        raise LightGBMError("refit_stages: weights have to be finite, with a finite sum, >= 0 and not all zero")
    run = _RefitGpu if _on_gpu(device, rows * len(forest.offsets[:-1])) else _RefitCpu
    values = run(forest, mat, target, w / total, stages).descend(int(num_steps), float(learning_rate), float(lambda_l2))
    lib, _ = _lib.load()
    for tree, (lo, hi) in enumerate(zip(forest.offsets[:-1], forest.offsets[1:])):
        for leaf in range(hi - lo):
            if values[lo + leaf] != forest.values[lo + leaf]:
                check(lib.lga_booster_set_leaf_value(out._handle, tree, leaf, float(values[lo + leaf])))
    return out


class _Refit:
    """Descent on the weighted mean loss of the stages, as a function of all leaf values.

    The loss has curvature of at most q in a raw score, and a row's score of stage k is a sum of k leaf values, so the
    Hessian is bounded by the diagonal  P_v = sum over the rows in leaf v of  w * sum over the stages k at or behind v's
    tree of  s_k * q * k  (s_k: the stage's share).  A step  -learning_rate * gradient / P  never raises the loss for
    learning rates up to 2.  Leaves that no row reaches keep their values."""

    def __init__(self, forest: _Forest, mat, target, weight, stages: str):
        self.forest = forest
        n = forest.count
        self.share = np.full(n, 1.0 / n) if stages == "all" else np.eye(n)[n - 1]
        curvature = _CURVATURE[forest.objective.split()[0]](forest.sigmoid)
        self.bound_by_stage = curvature * self.share * np.arange(1, n + 1)
        self.parts: List[tuple] = [self.part(forest.tokens(mat[lo:hi]), target[lo:hi], weight[lo:hi]) for lo, hi in forest.blocks(mat, 6)]

    def descend(self, steps: int, rate: float, lambda_l2: float) -> np.ndarray:
        start = values = self.start()
        bound = sum(self.bound(*p) for p in self.parts) + lambda_l2
        reached = bound > 0
        for _ in range(steps):
            grad = sum(self.gradient(values, *p) for p in self.parts) + lambda_l2 * (values - start)
            values = self.where(reached, values - rate * grad / self.where(reached, bound, 1.0), values)
        return self.finish(values)


class _RefitCpu(_Refit):
    def start(self):
        return self.forest.values.copy()

    def part(self, tokens, target, weight):
        return tokens, target, weight

    def _by_leaf(self, by_stage, tokens):
        """Sums over the tokens of a leaf of the sums over the stages behind its tree."""
        behind = np.cumsum(by_stage[::-1], axis=0)[::-1]                           # [iterations, rows, classes]
        flat = np.ascontiguousarray(behind.transpose(1, 0, 2)).reshape(-1)
        return np.bincount(tokens.reshape(-1), weights=flat, minlength=len(self.forest.values))

    def bound(self, tokens, target, weight):
        q = self.bound_by_stage.reshape(-1, 1, 1) * weight.reshape(1, -1, 1)
        return self._by_leaf(np.broadcast_to(q, (self.forest.count, len(tokens), self.forest.classes)), tokens)

    def gradient(self, values, tokens, target, weight):
        slopes = _slopes(_stages_cpu(self.forest, tokens, values), target, self.forest, np)
        return self._by_leaf(slopes * self.share.reshape(-1, 1, 1) * weight.reshape(1, -1, 1), tokens)

    where = staticmethod(np.where)

    def finish(self, values):
        return values


class _RefitGpu(_Refit):
    def start(self):
        import torch
        return torch.from_numpy(self.forest.values).cuda()

    def part(self, tokens, target, weight):
        import torch
        return tuple(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (tokens, target, weight))

    def _by_leaf(self, by_stage, states, tokens):
        from . import ops
        n = self.forest.count
        grad_x, _, _ = ops.gated_scan_grad(by_stage.reshape(1, n, -1), states.reshape(1, n, -1))
        return ops.embedding_grad(grad_x.view(n, tokens.shape[0], self.forest.classes, 1), _by_stage(self.forest, tokens), len(self.forest.values)).view(-1)

    def _weights(self, by_stage: np.ndarray, weight):
        import torch
        return torch.from_numpy(by_stage).cuda().view(-1, 1, 1) * weight.view(1, -1, 1)

    def bound(self, tokens, target, weight):
        q = self._weights(self.bound_by_stage, weight).expand(-1, -1, self.forest.classes).contiguous()
        return self._by_leaf(q, q, tokens)

    def gradient(self, values, tokens, target, weight):
        import torch
        raw = _stages_gpu(self.forest, tokens, values.view(-1, 1), None)
        return self._by_leaf(_slopes(raw, target, self.forest, torch) * self._weights(self.share, weight), raw, tokens)

    def where(self, condition, a, b):
        import torch
        return torch.where(condition, a, b)

    def finish(self, values):
        return values.cpu().numpy()
