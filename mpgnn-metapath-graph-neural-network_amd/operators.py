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
from array import array

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from ._lib import BF16, F16, F32, NORM_2, NORM_INF, check, lib
from .functional import _ptr, _stream_of

__all__ = ["layer_norm", "grouped_linear", "clip_by_global_norm", "clip_grad_norm_"]

_DTYPE = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_PTR_BITS = {torch.int64: 64, torch.int32: 32}


def _require(t: torch.Tensor, name: str) -> int:
    """The mpgnn_dtype of a GPU tensor that the operators take."""
    code = _DTYPE.get(t.dtype)
    if code is not None and t.is_cuda:
        return code
    if not t.is_cuda:
        raise RuntimeError(f"mpgnn_amd: `{name}` is on {t.device}; the operators run only as HIP kernels on a ROCm "
                           "GPU (there is no CPU fallback). Move the model and data to 'cuda'.")
    raise TypeError(f"mpgnn_amd: `{name}` must be float32, bfloat16 or float16, got {t.dtype}")


def _call(device: torch.device, entry, *args) -> None:
    """A C entry point on torch's current stream of ``device``, made the current device for the call (a
    launch goes to the current device)."""
    if device.index == torch.cuda.current_device():
        st = entry(*args, _stream_of(device))
    else:
        with torch.cuda.device(device):
            st = entry(*args, _stream_of(device))
    if st:
        check(st, entry.__name__)


_WS_BYTES: dict = {}  # (entry, sizes) -> bytes: they depend on the sizes only, asked once for each


def _workspace_bytes(entry, *sizes) -> int:
    n = _WS_BYTES.get((entry.__name__, sizes))
    if n is None:
        out = ctypes.c_int64()
        check(entry(*sizes, ctypes.byref(out)), entry.__name__)
        if len(_WS_BYTES) >= 4096:  # ragged batches: every step may bring new sizes
            _WS_BYTES.clear()
        n = _WS_BYTES[(entry.__name__, sizes)] = out.value
    return n


def _once(backward):
    """``once_differentiable`` where a graph of the backward is wanted; it costs a few us a call otherwise."""
    guarded = once_differentiable(backward)

    def run(ctx, dy):
        return guarded(ctx, dy) if torch.is_grad_enabled() else backward(ctx, dy)
    return run


# ---------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------
def _rows_view(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(tensor, rows, row pitch) of t as rows of its last dimension: t itself where its rows lie a
    constant pitch apart (contiguous, or a column slice of a matrix), else a contiguous copy."""
    shape = t.shape
    width = shape[-1]
    rows = shape[0] if len(shape) == 2 else t.numel() // width
    if not t.is_contiguous():
        if len(shape) == 2:
            pitch, inner = t.stride()
            if inner == 1 and pitch >= width:
                return t, rows, pitch
        t = t.contiguous()
    return t, rows, width


def _norm_forward(x, weight, bias, eps, code, wcode, keep):
    xr, rows, pitch = _rows_view(x)
    device = x.device
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    stats = mean = rstd = None
    if keep:
        stats = torch.empty((2, rows), dtype=torch.float32, device=device)
        mean = stats.data_ptr()
        rstd = mean + 4 * rows
    _call(device, lib.mpgnn_layer_norm_fwd, xr.data_ptr(), rows, x.shape[-1], pitch, code,
          None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(), wcode, eps,
          y.data_ptr(), mean, rstd)
    return y, xr, stats


class _LayerNormFn(torch.autograd.Function):
    # what the backward needs of sizes is worked out in the forward: autograd runs backwards of GPU tensors on
    # a thread of its own, where Python is about three times as slow
    @staticmethod
    def forward(ctx, x, weight, bias, eps, code, wcode):
        y, xr, stats = _norm_forward(x, weight, bias, eps, code, wcode, True)
        width = x.shape[-1]
        rows = stats.shape[1]
        params = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        nbytes = max(16, _workspace_bytes(lib.mpgnn_layer_norm_bwd_workspace_bytes, rows, width)) if params else 0
        ctx.stats = stats  # neither an input nor an output
        ctx.meta = (rows, width, width if xr.is_contiguous() else xr.stride(0), code, wcode, nbytes, stats.data_ptr(),
                    x.dtype if wcode == code else torch.float32)
        ctx.save_for_backward(xr, weight)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        rows, width, pitch, code, wcode, nbytes, mean, pdt = ctx.meta
        nx, nw, nb = ctx.needs_input_grad[:3]
        device = x.device
        dyr, _, dy_pitch = _rows_view(dy)
        dx = torch.empty_like(x, memory_format=torch.contiguous_format) if nx else None
        dw = torch.empty(width, dtype=pdt, device=device) if nw else None
        db = torch.empty(width, dtype=pdt, device=device) if nb else None
        # a buffer of its own per call: a captured backward keeps it in its graph's pool
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _call(device, lib.mpgnn_layer_norm_bwd, dyr.data_ptr(), dy_pitch, x.data_ptr(), pitch, rows, width, code,
              _ptr(weight), wcode, mean, mean + 4 * rows, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws))
        return dx, dw, db, None, None, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension of ``x`` (any leading
    dimensions; the variance is the mean squared difference, as torch.nn.LayerNorm's).

    ``weight`` / ``bias``: [x.shape[-1]], of x's type or both fp32, or None. A column slice of a
    matrix is read in place. Differentiable once in x, weight and bias."""
    code = wcode = _require(x, "x")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"layer_norm normalises a last dimension of at least one element, got shape {tuple(shape)}")
    grad = x.requires_grad
    if weight is not None:
        wcode = _check_param(weight, "weight", x, shape[-1], code)
        grad = grad or weight.requires_grad
        if not weight.is_contiguous():
            weight = weight.contiguous()
    if bias is not None:
        c = _check_param(bias, "bias", x, shape[-1], code)
        if weight is not None and c != wcode:
            raise TypeError(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
        wcode = c
        grad = grad or bias.requires_grad
        if not bias.is_contiguous():
            bias = bias.contiguous()
    if grad and torch.is_grad_enabled():
        return _LayerNormFn.apply(x, weight, bias, float(eps), code, wcode)
    return _norm_forward(x, weight, bias, float(eps), code, wcode, False)[0]


def _check_param(p, name, x, width, code) -> int:
    c = _require(p, name)
    if p.shape != (width,):
        raise ValueError(f"`{name}` has shape {tuple(p.shape)}, expected ({width},)")
    if p.get_device() != x.get_device():
        raise RuntimeError(f"`{name}` is on {p.device}, x on {x.device}")
    if c != code and c != F32:
        raise TypeError(f"`{name}` must be {x.dtype} or float32, got {p.dtype}")
    return c


# ---------------------------------------------------------------------------------------
# grouped linear
# ---------------------------------------------------------------------------------------
def _grouped_forward(x, pitch, weight, bias, ptr, bits, code):
    groups, k, n = weight.shape
    y = torch.empty((x.shape[0], n), dtype=x.dtype, device=x.device)
    _call(x.device, lib.mpgnn_grouped_linear_fwd, x.data_ptr(), x.shape[0], pitch, code, weight.data_ptr(), groups, k, n,
          _ptr(bias), ptr.data_ptr(), bits, y.data_ptr())
    return y


class _GroupedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, ptr, bits, code):
        xr, rows, pitch = _rows_view(x)
        wc = weight if weight.is_contiguous() else weight.contiguous()
        bc = bias if bias is None or bias.is_contiguous() else bias.contiguous()
        sizes = tuple(wc.shape)
        params = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        nbytes = _workspace_bytes(lib.mpgnn_grouped_linear_wgrad_workspace_bytes, rows, *sizes) if params else 0
        ctx.meta = rows, pitch, bits, code, sizes, nbytes
        ctx.save_for_backward(xr, wc, ptr)
        return _grouped_forward(xr, pitch, wc, bc, ptr, bits, code)

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, ptr = ctx.saved_tensors
        rows, pitch, bits, code, sizes, nbytes = ctx.meta
        nx, nw, nb = ctx.needs_input_grad[:3]
        device, p = x.device, ptr.data_ptr()
        dyr, _, dy_pitch = _rows_view(dy)
        dx = dw = db = None
        if nx:
            dx = torch.empty_like(x, memory_format=torch.contiguous_format)
            _call(device, lib.mpgnn_grouped_linear_dgrad, dyr.data_ptr(), rows, dy_pitch, code, weight.data_ptr(), *sizes,
                  p, bits, dx.data_ptr())
        if nw or nb:
            dw = torch.empty_like(weight)
            if nb:
                db = torch.empty((sizes[0], sizes[2]), dtype=x.dtype, device=device)
            ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
            _call(device, lib.mpgnn_grouped_linear_wgrad, x.data_ptr(), pitch, dyr.data_ptr(), dy_pitch, rows, code,
                  *sizes, p, bits, dw.data_ptr(), _ptr(db), _ptr(ws))
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
    sx, sw, sp = x.shape, weight.shape, group_ptr.shape
    if len(sx) != 2 or len(sw) != 3 or len(sp) != 1:
        raise ValueError("grouped_linear takes x [rows, K], weight [groups, K, N] and group_ptr [groups + 1], got "
                         f"{tuple(sx)}, {tuple(sw)} and {tuple(sp)}")
    groups, k, n = sw
    if groups < 1 or k < 1 or n < 1:
        raise ValueError(f"grouped_linear needs at least one group, input and output column, got weight {tuple(sw)}")
    if sx[1] != k:
        raise RuntimeError(f"mat1 and mat2 shapes cannot be multiplied ({sx[0]}x{sx[1]} and {k}x{n})")
    if sp[0] != groups + 1:
        raise ValueError(f"group_ptr has {sp[0]} entries, expected groups + 1 = {groups + 1}")
    bits = _PTR_BITS.get(group_ptr.dtype)
    if bits is None:
        raise TypeError(f"group_ptr must be int32 or int64, got {group_ptr.dtype}")
    where = x.get_device()
    if _require(weight, "weight") != code:
        raise TypeError(f"`weight` must be {x.dtype} as x is, got {weight.dtype}")
    if weight.get_device() != where:
        raise RuntimeError(f"`weight` is on {weight.device}, x on {x.device}")
    if group_ptr.get_device() != where:
        raise RuntimeError(f"`group_ptr` is on {group_ptr.device}, x on {x.device}")
    grad = x.requires_grad or weight.requires_grad
    if bias is not None:
        if _require(bias, "bias") != code:
            raise TypeError(f"`bias` must be {x.dtype} as x is, got {bias.dtype}")
        if bias.get_device() != where:
            raise RuntimeError(f"`bias` is on {bias.device}, x on {x.device}")
        if bias.shape != (groups, n):
            raise ValueError(f"bias has shape {tuple(bias.shape)}, expected {(groups, n)}")
        grad = grad or bias.requires_grad
    if not group_ptr.is_contiguous():
        group_ptr = group_ptr.contiguous()
    if grad and torch.is_grad_enabled():
        return _GroupedLinearFn.apply(x, weight, bias, group_ptr, bits, code)
    xr, _, pitch = _rows_view(x)
    return _grouped_forward(xr, pitch, weight if weight.is_contiguous() else weight.contiguous(),
                            bias if bias is None or bias.is_contiguous() else bias.contiguous(), group_ptr, bits, code)


# ---------------------------------------------------------------------------------------
# global norm and clipping
# ---------------------------------------------------------------------------------------
def _describe(tensors, what) -> tuple[list, list]:
    """(mpgnn_dtype codes, element counts) of tensors that lie dense on one GPU; a column of the list at
    a time, as with hundreds of tensors a step these checks are the calls' host time."""
    codes = [_DTYPE.get(d) for d in [t.dtype for t in tensors]]
    if None in codes or not tensors[0].is_cuda or len({t.get_device() for t in tensors}) != 1:
        device = tensors[0].device
        for t in tensors:
            _require(t, what)
            if t.device != device:
                raise RuntimeError(f"{what} are on several devices: {device} and {t.device}")
    return codes, [t.numel() for t in tensors]


def _contiguous(tensors, what) -> list:
    """Indices of the tensors that are not contiguous."""
    try:
        flags = [t.is_contiguous() for t in tensors]
    except RuntimeError as exc:  # a sparse layout
        raise TypeError(f"mpgnn_amd: {what} must be dense") from exc
    if False not in flags:
        return []
    strided = [k for k, c in enumerate(flags) if not c]
    for k in strided:
        if tensors[k].layout is not torch.strided:
            raise TypeError(f"mpgnn_amd: {what} must be dense, got {tensors[k].layout}")
    return strided


def _clip(grads, codes, numels, outs, max_norm, norm_type) -> torch.Tensor:
    """The norm of ``grads`` (checked and contiguous); ``outs``: where the scaled tensors go, or None."""
    if norm_type == 2.0:
        kind = NORM_2
    elif norm_type == math.inf:
        kind = NORM_INF
    else:
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type!r}")
    n = len(grads)
    device = grads[0].device
    # mpgnn_clip_tensor records: four 64-bit words (grad, out, numel, dtype)
    words = array("q", bytes(32 * n))
    words[0::4] = array("q", [g.data_ptr() for g in grads])
    if outs is grads:
        words[1::4] = words[0::4]
    elif outs is not None:
        words[1::4] = array("q", [o.data_ptr() for o in outs])
    if outs is not None and len(set(words[1::4])) != n:
        # each tensor with elements at an address of its own: scaled in place twice, one would be scaled by
        # the factor's square
        used = [p for p, m in zip(words[1::4], numels) if m]
        if len(set(used)) != len(used):
            raise ValueError("one tensor is to be scaled twice")
    words[2::4] = array("q", numels)
    words[3::4] = array("q", codes)
    ws = torch.empty(_workspace_bytes(lib.mpgnn_clip_workspace_bytes, n), dtype=torch.uint8, device=device)
    norm = torch.empty((), dtype=torch.float32, device=device)
    _call(device, lib.mpgnn_clip_by_global_norm, words.buffer_info()[0], n, kind, max_norm, norm.data_ptr(),
          ws.data_ptr())
    if outs is not None:
        increment_version(outs)  # written behind autograd's back, as any in-place operator counts
    return norm


def _check_max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be a number of at least 0, got {max_norm}")
    return max_norm


def clip_by_global_norm(tensors, max_norm: float, norm_type: float = 2.0, out=None):
    """``(norm, clipped)``: the global norm over ``tensors`` (the 2-norm of all elements, or the largest
    magnitude with ``norm_type=inf``) as an fp32 scalar tensor, and ``t * min(1, max_norm / (norm + 1e-6))``
    of each, in new tensors or in those of ``out`` (same sizes, types and device, contiguous; ``out`` may
    be ``tensors`` itself, otherwise the two must not overlap). Not differentiable; no host synchronisation.

    The factor is computed and applied in fp32 and each product rounded once to its tensor's type. An
    infinite or NaN gradient makes the norm so, and the products what the formula gives."""
    max_norm = _check_max_norm(max_norm)
    tensors = list(tensors)
    if not tensors:
        raise ValueError("clip_by_global_norm needs at least one tensor")
    codes, numels = _describe(tensors, "tensors")
    strided = _contiguous(tensors, "tensors")
    if out is None:
        outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in tensors]
    else:
        outs = list(out)
        if len(outs) != len(tensors):
            raise ValueError(f"out has {len(outs)} tensors for {len(tensors)}")
        if _describe(outs, "out") != (codes, numels) or outs[0].device != tensors[0].device or \
                _contiguous(outs, "out"):
            raise ValueError("out must hold contiguous tensors of the inputs' sizes, types and device")
    for k in strided:
        tensors[k] = tensors[k].detach().contiguous()
    return _clip(tensors, codes, numels, outs, max_norm, norm_type), outs


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
    codes, numels = _describe(grads, "gradients")
    strided = _contiguous(grads, "gradients")
    flat = grads
    if strided:
        flat = list(grads)
        if len({id(g) for g in grads}) != len(grads):
            raise ValueError("one tensor is to be scaled twice")
        for k in strided:
            g = grads[k]
            if any(st == 0 and n > 1 for n, st in zip(g.shape, g.stride())):
                raise ValueError("a gradient is an expanded tensor, whose elements share memory: it cannot be scaled "
                                 "in place")
            flat[k] = g.detach().contiguous()
    if error_if_nonfinite:
        norm = _clip(flat, codes, numels, None, max_norm, norm_type)
        if not math.isfinite(float(norm)):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so "
                               "it cannot be clipped. To disable this error and scale the gradients by the non-finite "
                               "norm anyway, set `error_if_nonfinite=False`")
    norm = _clip(flat, codes, numels, flat, max_norm, norm_type)
    if strided:
        with torch.no_grad():
            for k in strided:
                grads[k].copy_(flat[k])
    return norm
