"""Operators of a training or serving step around the relational layers, for fp32, bf16 and fp16
tensors on the GPU (C ABI calls on torch's current stream of the tensors' device).

``layer_norm``           torch.nn.functional.layer_norm over the last dimension, with its gradients
``grouped_linear``       x[i] @ weight[g] (+ bias[g]) for the rows i of group g: row ranges of ragged sizes,
                         each with a weight of its own (node types, relations, experts)
``clip_by_global_norm``  the global norm over a list of tensors and the tensors scaled to at most
                         ``max_norm``; ``clip_grad_norm_`` does it in place on parameters' gradients
                         (between ``loss.backward()`` and ``optimizer.step()``)

Statistics, sums and matrix accumulators are held in fp32 or wider and a 16-bit result is rounded
once. Results do not change from run to run. No call synchronises the device or keeps anything
from one call to the next, so all of them can be captured into a HIP graph. A forward-mode tangent
(torch.autograd.forward_ad) on an argument and a recording torch.jit.trace or make_fx raise NotImplementedError.
"""
from __future__ import annotations

import math

import torch

__all__ = ["layer_norm", "grouped_linear", "clip_by_global_norm", "clip_grad_norm_"]

_native = None  # the module over the C ABI (csrc/operators_torch.cpp)


def _ops():
    """Checks, outputs, autograd nodes and launches are compiled: a step's small calls are bound by the host."""
    global _native
    if _native is None:
        try:
            from . import _operators
        except ImportError as exc:
            raise ImportError("mpgnn_amd/_operators.so is missing or does not fit the installed torch: build it with "
                              "`make -C csrc` or __graft_entry__.build()") from exc
        _native = _operators
    return _native


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x`` (any leading
    dimensions; the variance is the mean squared difference, as torch.nn.LayerNorm's).

    ``weight`` / ``bias``: [x.shape[-1]], of x's type or both fp32, or None. A column slice of a
    matrix is read in place. Differentiable once in x, weight and bias."""
    return _ops().layer_norm(x, weight, bias, eps)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, group_ptr: torch.Tensor,
                   bias: torch.Tensor = None) -> torch.Tensor:
    """``out[i] = x[i] @ weight[g] + bias[g]`` for the rows i of group g, rows ``group_ptr[g]`` to
    ``group_ptr[g + 1]`` of ``x`` [rows, K]; ``weight`` [groups, K, N] as in RGCNConv, ``bias`` [groups, N]
    or None, all of one type (fp32, bf16 or fp16).

    ``group_ptr``: [groups + 1] int32 or int64, non-decreasing, on x's device (it is never read by the host:
    the sizes may come from a kernel just launched, and may differ between replays of a captured graph).
    Groups may be empty. Rows before ``group_ptr[0]`` or from ``group_ptr[-1]`` on belong to no group: their
    output and gradient rows are zero. Differentiable once in x, weight and bias."""
    return _ops().grouped_linear(x, weight, group_ptr, bias)


def _largest(norm_type) -> bool:
    if norm_type == 2.0:
        return False
    if norm_type == math.inf:
        return True
    raise ValueError(f"norm_type must be 2 or inf, got {norm_type!r}")


def _check_max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number of at least 0, got {max_norm}")
    return max_norm


def clip_by_global_norm(tensors, max_norm: float, norm_type: float = 2.0, out=None):
    """``(norm, clipped)``: the global norm over ``tensors`` (the 2-norm of all elements, or the largest
    magnitude with ``norm_type=inf``) as an fp32 scalar tensor, and ``t * min(1, max_norm / (norm + 1e-6))``
    of each, in new tensors or in those of ``out`` (same sizes, types and device, contiguous; ``out`` may
    be ``tensors`` itself; one that overlaps another tensor otherwise is refused). Not differentiable; no host
    synchronisation.

    The factor is computed and applied in fp32 and each product rounded once to its tensor's type. An
    infinite or NaN gradient makes the norm so, and the products what the formula gives."""
    max_norm = _check_max_norm(max_norm)
    tensors = list(tensors)
    if not tensors:
        raise ValueError("clip_by_global_norm needs at least one tensor")
    largest = _largest(norm_type)
    if out is not None:
        out = list(out)
        if len(out) != len(tensors):
            raise ValueError(f"out has {len(out)} tensors for {len(tensors)}")
    norm, clipped = _ops().clip(tensors, out, 1, max_norm, largest)
    return norm, clipped if out is None else out


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False,
                    foreach=None) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` over GPU gradients of fp32, bf16 and fp16, mixed at will: scales
    the gradients in place to a global norm of at most ``max_norm`` and returns the norm before that (fp32
    scalar tensor). Parameters without a gradient are skipped; without any, the norm is 0.

    ``error_if_nonfinite`` raises before anything is scaled if the norm is infinite or NaN (this reads the
    norm on the host: the only synchronisation, and not possible in a graph capture). ``foreach`` is
    accepted for torch's signature; there is one implementation."""
    max_norm = _check_max_norm(max_norm)
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in (p.grad for p in parameters) if g is not None]
    if not grads:
        return torch.tensor(0.0)
    largest = _largest(norm_type)
    if error_if_nonfinite:
        norm, _ = _ops().clip(grads, None, 0, max_norm, largest)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so "
                               "it cannot be clipped. To disable this error and scale the gradients by the non-finite "
                               "norm anyway, set `error_if_nonfinite=False`")
    return _ops().clip(grads, None, 2, max_norm, largest)[0]
