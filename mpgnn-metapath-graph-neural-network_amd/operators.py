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
from one call to the next, so all of them can be captured into a HIP graph.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from ._lib import BF16, F16, F32, NORM_2, NORM_INF, check, lib
from .functional import _ptr, _stream_of

__all__ = ["layer_norm", "grouped_linear", "clip_by_global_norm", "clip_grad_norm_"]

_DTYPE = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}


def _require(t: torch.Tensor, name: str) -> int:
    """The mpgnn_dtype of a GPU tensor that the operators take."""
    if not t.is_cuda:
        raise RuntimeError(f"mpgnn_amd: `{name}` is on {t.device}; the operators run only as HIP kernels on a ROCm "
                           "GPU (there is no CPU fallback). Move the model and data to 'cuda'.")
    code = _DTYPE.get(t.dtype)
    if code is None:
        raise TypeError(f"mpgnn_amd: `{name}` must be float32, bfloat16 or float16, got {t.dtype}")
    return code


class _on:
    """The tensor's device made current for the call (a launch goes to the current device)."""
    __slots__ = ("device", "guard")

    def __init__(self, device):
        self.device = device
        self.guard = None

    def __enter__(self):
        if self.device.index != torch.cuda.current_device():
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()
        return _stream_of(self.device)

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


# ---------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------
def _rows_view(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(tensor, rows, row pitch) of t as rows of its last dimension: t itself where its rows lie a
    constant pitch apart (contiguous, or a column slice of a matrix), else a contiguous copy."""
    width = t.shape[-1]
    rows = t.numel() // width
    if t.is_contiguous():
        return t, rows, width
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= width:
        return t, rows, t.stride(0)
    return t.contiguous(), rows, width


def _norm_forward(x, weight, bias, eps, code, wcode, keep):
    xr, rows, pitch = _rows_view(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device) if keep else None
    mean = rstd = None
    if keep:
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    with _on(x.device) as stream:
        st = lib.mpgnn_layer_norm_fwd(xr.data_ptr(), rows, x.shape[-1], pitch, code, _ptr(weight), _ptr(bias), wcode,
                                      eps, y.data_ptr(), mean, rstd, stream)
    if st:
        check(st, "mpgnn_layer_norm_fwd")
    return y, xr, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, code, wcode):
        y, xr, stats = _norm_forward(x, weight, bias, eps, code, wcode, True)
        ctx.codes = code, wcode
        ctx.save_for_backward(xr, weight, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        code, wcode = ctx.codes
        nx, nw, nb = ctx.needs_input_grad[:3]
        width = x.shape[-1]
        rows = x.numel() // width
        pitch = width if x.is_contiguous() else x.stride(0)
        dyr, _, dy_pitch = _rows_view(dy)
        pdt = x.dtype if wcode == code else torch.float32
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if nx else None
        dw = torch.empty(width, dtype=pdt, device=x.device) if nw else None
        db = torch.empty(width, dtype=pdt, device=x.device) if nb else None
        ws = None
        if nw or nb:
            nbytes = ctypes.c_int64()
            check(lib.mpgnn_layer_norm_bwd_workspace_bytes(rows, width, ctypes.byref(nbytes)),
                  "mpgnn_layer_norm_bwd_workspace_bytes")
            # a buffer of its own per call: a captured backward keeps it in its graph's pool
            ws = torch.empty(max(nbytes.value, 16), dtype=torch.uint8, device=x.device)
        mean = stats.data_ptr()
        with _on(x.device) as stream:
            st = lib.mpgnn_layer_norm_bwd(dyr.data_ptr(), dy_pitch, x.data_ptr(), pitch, rows, width, code,
                                          _ptr(weight), wcode, mean, mean + 4 * rows, _ptr(dx), _ptr(dw), _ptr(db),
                                          _ptr(ws), stream)
        if st:
            check(st, "mpgnn_layer_norm_bwd")
        return dx, dw, db, None, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x`` (any leading
    dimensions; the variance is the mean squared difference, as torch.nn.LayerNorm's).

    ``weight`` / ``bias``: [x.shape[-1]], of x's type or both fp32, or None. A column slice of a
    matrix is read in place. Differentiable once in x, weight and bias."""
    code = _require(x, "x")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm normalises a last dimension of at least one element, got shape {tuple(x.shape)}")
    wcode = code
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        c = _require(p, name)
        if p.dim() != 1 or p.shape[0] != x.shape[-1]:
            raise ValueError(f"`{name}` has shape {tuple(p.shape)}, expected ({x.shape[-1]},)")
        if p.device != x.device:
            raise RuntimeError(f"`{name}` is on {p.device}, x on {x.device}")
        if c != code and c != F32:
            raise TypeError(f"`{name}` must be {x.dtype} or float32, got {p.dtype}")
        wcode = c
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, float(eps), code, wcode)
    return _norm_forward(x, weight, bias, float(eps), code, wcode, False)[0]


# ---------------------------------------------------------------------------------------
# grouped linear
# ---------------------------------------------------------------------------------------
def _grouped_forward(x, pitch, weight, bias, ptr, bits, code):
    groups, k, n = weight.shape
    y = torch.empty((x.shape[0], n), dtype=x.dtype, device=x.device)
    with _on(x.device) as stream:
        st = lib.mpgnn_grouped_linear_fwd(x.data_ptr(), x.shape[0], pitch, code, weight.data_ptr(), groups, k, n,
                                          _ptr(bias), ptr.data_ptr(), bits, y.data_ptr(), stream)
    if st:
        check(st, "mpgnn_grouped_linear_fwd")
    return y


class _GroupedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, ptr, bits, code):
        xr, _, pitch = _rows_view(x)
        wc = weight if weight.is_contiguous() else weight.contiguous()
        bc = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        ctx.meta = pitch, bits, code
        ctx.save_for_backward(xr, wc, ptr)
        return _grouped_forward(xr, pitch, wc, bc, ptr, bits, code)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, ptr = ctx.saved_tensors
        pitch, bits, code = ctx.meta
        nx, nw, nb = ctx.needs_input_grad[:3]
        groups, k, n = weight.shape
        rows = x.shape[0]
        dyr, _, dy_pitch = _rows_view(dy)
        dx = torch.empty((rows, k), dtype=x.dtype, device=x.device) if nx else None
        dw = torch.empty((groups, k, n), dtype=x.dtype, device=x.device) if nw or nb else None
        db = torch.empty((groups, n), dtype=x.dtype, device=x.device) if nb else None
        with _on(x.device) as stream:
            if nx:
                st = lib.mpgnn_grouped_linear_dgrad(dyr.data_ptr(), rows, dy_pitch, code, weight.data_ptr(), groups, k,
                                                    n, ptr.data_ptr(), bits, dx.data_ptr(), stream)
                if st:
                    check(st, "mpgnn_grouped_linear_dgrad")
            if nw or nb:
                nbytes = ctypes.c_int64()
                check(lib.mpgnn_grouped_linear_wgrad_workspace_bytes(rows, groups, k, n, ctypes.byref(nbytes)),
                      "mpgnn_grouped_linear_wgrad_workspace_bytes")
                ws = torch.empty(nbytes.value, dtype=torch.uint8, device=x.device) if nbytes.value else None
                st = lib.mpgnn_grouped_linear_wgrad(x.data_ptr(), pitch, dyr.data_ptr(), dy_pitch, rows, code, groups,
                                                    k, n, ptr.data_ptr(), bits, dw.data_ptr(), _ptr(db), _ptr(ws),
                                                    stream)
                if st:
                    check(st, "mpgnn_grouped_linear_wgrad")
        return dx, dw if nw else None, db, None, None, None


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, group_ptr: torch.Tensor,
                   bias: torch.Tensor = None) -> torch.Tensor:
    """``out[i] = x[i] @ weight[g] + bias[g]`` for the rows i of group g, rows ``group_ptr[g]`` to
    ``group_ptr[g + 1]`` of ``x`` [rows, K]; ``weight`` [groups, K, N] as in RGCNConv, ``bias`` [groups, N]
    or None, all of one type (fp32, bf16 or fp16).

    ``group_ptr``: [groups + 1] int32 or int64, non-decreasing, on x's device (it is never read by the host:
    the sizes may come from a kernel just launched, and may differ between replays of a captured graph).
    Groups may be empty. Rows before ``group_ptr[0]`` or from ``group_ptr[-1]`` on belong to no group: their
    output and gradient rows are zero. Differentiable once in x, weight and bias."""
    code = _require(x, "x")
    if x.dim() != 2 or weight.dim() != 3 or group_ptr.dim() != 1:
        raise ValueError("grouped_linear takes x [rows, K], weight [groups, K, N] and group_ptr [groups + 1], got "
                         f"{tuple(x.shape)}, {tuple(weight.shape)} and {tuple(group_ptr.shape)}")
    groups, k, n = weight.shape
    if groups < 1 or k < 1 or n < 1:
        raise ValueError(f"grouped_linear needs at least one group, input and output column, got weight {tuple(weight.shape)}")
    if x.shape[1] != k:
        raise RuntimeError(f"mat1 and mat2 shapes cannot be multiplied ({x.shape[0]}x{x.shape[1]} and {k}x{n})")
    if group_ptr.shape[0] != groups + 1:
        raise ValueError(f"group_ptr has {group_ptr.shape[0]} entries, expected groups + 1 = {groups + 1}")
    if group_ptr.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"group_ptr must be int32 or int64, got {group_ptr.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if _require(t, name) != code:
            raise TypeError(f"`{name}` must be {x.dtype} as x is, got {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"`{name}` is on {t.device}, x on {x.device}")
    if group_ptr.device != x.device:
        raise RuntimeError(f"`group_ptr` is on {group_ptr.device}, x on {x.device}")
    if bias is not None and tuple(bias.shape) != (groups, n):
        raise ValueError(f"bias has shape {tuple(bias.shape)}, expected {(groups, n)}")
    ptr = group_ptr if group_ptr.is_contiguous() else group_ptr.contiguous()
    bits = 64 if ptr.dtype == torch.int64 else 32
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _GroupedLinearFn.apply(x, weight, bias, ptr, bits, code)
    xr, _, pitch = _rows_view(x)
    return _grouped_forward(xr, pitch, weight if weight.is_contiguous() else weight.contiguous(),
                            bias if bias is None or bias.is_contiguous() else bias.contiguous(), ptr, bits, code)


# ---------------------------------------------------------------------------------------
# global norm and clipping
# ---------------------------------------------------------------------------------------
_CLIP_RECORD = struct.Struct("=QQqii")  # mpgnn_clip_tensor


def _clip(grads, outs, max_norm, norm_type) -> torch.Tensor:
    """The norm of ``grads`` (one device, contiguous); ``outs``: where the scaled tensors go, or None."""
    if norm_type == 2.0:
        kind = NORM_2
    elif norm_type == math.inf:
        kind = NORM_INF
    else:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type!r}")
    n = len(grads)
    device = grads[0].device
    # the records packed at once: hundreds of tensors a step make this loop the call's host time
    pack = _CLIP_RECORD.pack
    if outs is None:
        table = b"".join([pack(g.data_ptr(), 0, g.numel(), _DTYPE[g.dtype], 0) for g in grads])
    elif outs is grads:
        table = b"".join([pack(p, p, g.numel(), _DTYPE[g.dtype], 0) for g in grads for p in (g.data_ptr(),)])
    else:
        table = b"".join([pack(g.data_ptr(), o.data_ptr(), g.numel(), _DTYPE[g.dtype], 0)
                          for g, o in zip(grads, outs)])
    nbytes = ctypes.c_int64()
    st = lib.mpgnn_clip_workspace_bytes(n, ctypes.byref(nbytes))
    if st:
        check(st, "mpgnn_clip_workspace_bytes")
    ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    with _on(device) as stream:
        st = lib.mpgnn_clip_by_global_norm(table, n, kind, max_norm, norm.data_ptr(), ws.data_ptr(), stream)
    if st:
        check(st, "mpgnn_clip_by_global_norm")
    if outs is not None:
        increment_version(outs)  # written behind autograd's back, as any in-place operator counts
    return norm


def _check_list(tensors, what):
    device = tensors[0].device
    for t in tensors:
        if not (t.is_cuda and t.dtype in _DTYPE and t.layout is torch.strided and t.device == device):
            if t.layout is not torch.strided:
                raise TypeError(f"mpgnn_amd: {what} must be dense, got {t.layout}")
            _require(t, what)
            raise RuntimeError(f"{what} are on several devices: {device} and {t.device}")


def _check_max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number of at least 0, got {max_norm}")
    return max_norm


def _distinct(tensors, what):
    """Each tensor with elements starts at an address of its own: scaled in place twice, one would
    be scaled by the factor's square."""
    ptrs = [t.data_ptr() for t in tensors]
    if len(set(ptrs)) != len(ptrs):  # empty tensors may share one
        ptrs = [t.data_ptr() for t in tensors if t.numel()]
        if len(set(ptrs)) != len(ptrs):
            raise ValueError(f"{what} holds one tensor twice")


def clip_by_global_norm(tensors, max_norm: float, norm_type: float = 2.0, out=None):
    """``(norm, clipped)``: the global norm over ``tensors`` (the 2-norm of all elements, or the largest
    magnitude with ``norm_type=inf``) as an fp32 scalar tensor, and ``t * min(1, max_norm / (norm + 1e-6))``
    of each, in new tensors or in those of ``out`` (same shapes, types and device, contiguous; ``out`` may
    be ``tensors`` itself, otherwise the two must not overlap). Not differentiable; no host synchronisation.

    The factor is computed and applied in fp32 and each product rounded once to its tensor's type. An
    infinite or NaN gradient makes the norm so, and the products what the formula gives."""
    max_norm = _check_max_norm(max_norm)
    tensors = list(tensors)
    if not tensors:
        raise ValueError("clip_by_global_norm needs at least one tensor")
    _check_list(tensors, "tensors")
    if out is None:
        outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in tensors]
    else:
        outs = list(out)
        if len(outs) != len(tensors):
            raise ValueError(f"out has {len(outs)} tensors for {len(tensors)}")
        for o, t in zip(outs, tensors):
            if not (o.dtype == t.dtype and o.shape == t.shape and o.device == t.device and o.is_contiguous()):
                raise ValueError("out must hold contiguous tensors of the inputs' shapes, types and device")
        _distinct(outs, "out")
    grads = [t if t.is_contiguous() else t.detach().contiguous() for t in tensors]
    return _clip(grads, outs, max_norm, norm_type), outs


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
    _check_list(grads, "gradients")
    _distinct(grads, "the parameters' gradients")
    flat = grads
    strided = [k for k, g in enumerate(grads) if not g.is_contiguous()]
    if strided:
        flat = list(grads)
        for k in strided:
            g = grads[k]
            if any(st == 0 and n > 1 for n, st in zip(g.shape, g.stride())):
                raise ValueError("a gradient is an expanded tensor, whose elements share memory: it cannot be scaled "
                                 "in place")
            flat[k] = g.detach().contiguous()
    if error_if_nonfinite:
        norm = _clip(flat, None, max_norm, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so "
                               "it cannot be clipped. To disable this error and scale the gradients by the non-finite "
                               "norm anyway, set `error_if_nonfinite=False`")
    norm = _clip(flat, flat, max_norm, norm_type)
    if strided:
        with torch.no_grad():
            for k in strided:
                grads[k].copy_(flat[k])
    return norm
