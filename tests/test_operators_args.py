"""CPU: layer_norm, grouped_linear and the clipping refuse CPU tensors and bad arguments before any
launch, and size their workspaces on the host."""
import ctypes

import pytest
import torch

import mpgnn_amd
from mpgnn_amd import _lib
from mpgnn_amd._lib import lib

P = ctypes.c_void_p(4096)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(2, 8, 5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mpgnn_amd.layer_norm(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mpgnn_amd.grouped_linear(x, w, torch.tensor([0, 2, 4]))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mpgnn_amd.clip_by_global_norm([x], 1.0)
    p = torch.nn.Parameter(x)
    p.grad = torch.ones_like(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mpgnn_amd.clip_grad_norm_([p], 1.0)
    assert torch.equal(p.grad, torch.ones_like(x))
    assert float(mpgnn_amd.clip_grad_norm_([torch.nn.Parameter(x)], 1.0)) == 0.0


def test_layer_norm_entry_points_check_their_arguments():
    def fwd(x=P, rows=4, width=8, pitch=8, dt=0, wdt=0, y=P, mean=None, rstd=None):
        return lib.mpgnn_layer_norm_fwd(x, rows, width, pitch, dt, None, None, wdt, 1e-5, y, mean, rstd, None)

    assert fwd(rows=0, x=None, y=None) == _lib.MPGNN_OK
    for kw in (dict(rows=-1), dict(width=0), dict(pitch=7), dict(dt=3), dict(dt=0, wdt=1), dict(x=None), dict(y=None),
               dict(mean=P)):
        assert fwd(**kw) == _lib.MPGNN_ERR_ARG, kw
    assert fwd(width=1 << 25, pitch=1 << 25) == _lib.MPGNN_ERR_UNSUPPORTED

    def bwd(dy=P, dpitch=8, rows=4, stats=P, dx=P, dw=None, ws=None):
        return lib.mpgnn_layer_norm_bwd(dy, dpitch, P, 8, rows, 8, 0, None, 0, stats, stats, dx, dw, None, ws, None)

    assert bwd(dx=None) == _lib.MPGNN_OK  # nothing wanted
    for kw in (dict(dy=None), dict(dpitch=5), dict(rows=-2), dict(stats=None), dict(dw=P)):
        assert bwd(**kw) == _lib.MPGNN_ERR_ARG, kw
    nb = ctypes.c_int64()
    assert lib.mpgnn_layer_norm_bwd_workspace_bytes(10, 16, ctypes.byref(nb)) == 0 and nb.value == 10 * 2 * 16 * 4
    assert lib.mpgnn_layer_norm_bwd_workspace_bytes(10, 0, ctypes.byref(nb)) == _lib.MPGNN_ERR_ARG


def test_grouped_linear_entry_points_check_their_arguments():
    def fwd(x=P, rows=4, pitch=8, dt=0, w=P, groups=2, k=8, n=5, ptr=P, bits=64, out=P):
        return lib.mpgnn_grouped_linear_fwd(x, rows, pitch, dt, w, groups, k, n, None, ptr, bits, out, None)

    def dgrad(dy=P, rows=4, pitch=5, dt=0, w=P, groups=2, k=8, n=5, ptr=P, bits=64, out=P):
        return lib.mpgnn_grouped_linear_dgrad(dy, rows, pitch, dt, w, groups, k, n, ptr, bits, out, None)

    for f in (fwd, dgrad):
        assert f(rows=0) == _lib.MPGNN_OK
        for kw in (dict(rows=-1), dict(pitch=4), dict(dt=9), dict(w=None), dict(groups=0), dict(k=0), dict(n=0),
                   dict(ptr=None), dict(bits=16), dict(out=None)):
            assert f(**kw) == _lib.MPGNN_ERR_ARG, kw
        assert f(k=1 << 25, n=1 << 25, pitch=1 << 26) == _lib.MPGNN_ERR_UNSUPPORTED
    assert fwd(x=None) == _lib.MPGNN_ERR_ARG

    def wgrad(rows=4, xp=8, dp=5, dw=P, ws=None, groups=2, k=8, n=5):
        return lib.mpgnn_grouped_linear_wgrad(P, xp, P, dp, rows, 0, groups, k, n, P, 64, dw, None, ws, None)

    for kw in (dict(rows=-1), dict(xp=7), dict(dp=4), dict(dw=None), dict(rows=1 << 20)):  # the last: no workspace
        assert wgrad(**kw) == _lib.MPGNN_ERR_ARG, kw
    nb = ctypes.c_int64()
    # a weight with tiles enough to fill the chip needs none; one tile over many rows does
    assert lib.mpgnn_grouped_linear_wgrad_workspace_bytes(1 << 15, 32, 2048, 4096, ctypes.byref(nb)) == 0
    assert nb.value == 0
    assert lib.mpgnn_grouped_linear_wgrad_workspace_bytes(1 << 20, 2, 128, 128, ctypes.byref(nb)) == 0
    assert nb.value >= 2 * 128 * 128 * 4
    assert lib.mpgnn_grouped_linear_wgrad_workspace_bytes(4, 2, 8, 5, None) == _lib.MPGNN_ERR_ARG


def test_clip_entry_point_checks_its_arguments():
    arr = (_lib.ClipTensor * 2)()
    for t in arr:
        t.grad, t.out, t.numel, t.dtype = 4096, 8192, 16, _lib.F32

    def clip(n=2, kind=_lib.NORM_2, norm=P, ws=P):
        return lib.mpgnn_clip_by_global_norm(ctypes.addressof(arr), n, kind, 1.0, norm, ws, None)

    assert clip(n=0) == clip(n=-1) == clip(kind=1) == clip(norm=None) == clip(ws=None) == _lib.MPGNN_ERR_ARG
    assert lib.mpgnn_clip_by_global_norm(None, 1, 2, 1.0, P, P, None) == _lib.MPGNN_ERR_ARG
    for k in range(2):  # out for one tensor only
        arr[k].out = None
        assert clip() == _lib.MPGNN_ERR_ARG
        arr[k].out = 8192
    for field, v, back in (("dtype", 7, 0), ("numel", -1, 16), ("grad", None, 4096), ("grad", 4098, 4096),
                           ("out", 8193, 8192)):
        setattr(arr[1], field, v)
        assert clip() == _lib.MPGNN_ERR_ARG, field
        setattr(arr[1], field, back)
    arr[0].numel = 1 << 41
    assert clip() == _lib.MPGNN_ERR_UNSUPPORTED
    nb = ctypes.c_int64()
    assert lib.mpgnn_clip_workspace_bytes(3, ctypes.byref(nb)) == 0 and nb.value == 2048 * 8  # a partial per workgroup
    assert lib.mpgnn_clip_workspace_bytes(-3, ctypes.byref(nb)) == _lib.MPGNN_ERR_ARG


def test_modules_match_torch_parameters():
    a, b = mpgnn_amd.LayerNorm(12), torch.nn.LayerNorm(12)
    assert a.state_dict().keys() == b.state_dict().keys()
    assert all(torch.equal(x, y) for x, y in zip(a.state_dict().values(), b.state_dict().values()))
    assert mpgnn_amd.LayerNorm(12, elementwise_affine=False).weight is None
    assert mpgnn_amd.LayerNorm(12, bias=False).bias is None
    with pytest.raises(NotImplementedError):
        mpgnn_amd.LayerNorm((3, 4))
    g = mpgnn_amd.GroupedLinear(6, 4, 3)
    assert tuple(g.weight.shape) == (3, 6, 4) and tuple(g.bias.shape) == (3, 4) and float(g.bias.abs().max()) == 0.0
    assert float(g.weight.abs().max()) <= (6.0 / (6 + 4)) ** 0.5


def test_tangents_and_traces_are_refused():
    """A forward-mode tangent would be lost and a trace would hold no kernel: refused before anything else."""
    from torch.autograd import forward_ad
    x, w, ptr = torch.ones(4, 8), torch.ones(2, 8, 5), torch.tensor([0, 2, 4])
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        for f in (lambda: mpgnn_amd.layer_norm(dual(x)), lambda: mpgnn_amd.layer_norm(x, dual(x[0])),
                  lambda: mpgnn_amd.layer_norm(x, None, dual(x[0])), lambda: mpgnn_amd.layer_norm(dual(x).requires_grad_()),
                  lambda: mpgnn_amd.grouped_linear(dual(x), w, ptr), lambda: mpgnn_amd.grouped_linear(x, dual(w), ptr),
                  lambda: mpgnn_amd.grouped_linear(x, w, ptr, dual(w[:, 0])),
                  lambda: mpgnn_amd.clip_by_global_norm([dual(x)], 1.0)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
    for f in (lambda t: mpgnn_amd.layer_norm(t), lambda t: mpgnn_amd.grouped_linear(t, w, ptr),
              lambda t: mpgnn_amd.clip_by_global_norm([t], 1.0)[0]):
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(f, (x,))


def test_clip_refuses_overlapping_tensors():
    """An out that shares memory with another tensor of the list, written or read, would depend on which workgroup
    comes first: refused on the host (the addresses here are never read)."""
    def clip(*tensors):
        arr = (_lib.ClipTensor * len(tensors))()
        for t, (grad, out, numel, dtype) in zip(arr, tensors):
            t.grad, t.out, t.numel, t.dtype = grad, out, numel, dtype
        return lib.mpgnn_clip_by_global_norm(ctypes.addressof(arr), len(tensors), _lib.NORM_2, 1.0, P, P, None)

    a, b, c, f32, bf16 = 1 << 16, 1 << 17, 1 << 18, _lib.F32, _lib.BF16
    for bad in ([(a, a, 64, f32), (a + 128, a + 128, 8, f32)],            # a bucket and a view into it, in place
                [(a + 128, a + 128, 8, f32), (a, a, 64, f32)],            # in either order
                [(a, a, 64, f32), (a, a, 64, f32)],                       # one tensor twice
                [(a, a, 64, f32), (a, a, 32, f32)],
                [(a, b, 64, f32), (b, a, 64, f32)],                       # swapped
                [(a, b, 64, f32), (b + 64, c, 64, f32)],                  # an out over the end of another's input
                [(a, b, 64, f32), (c, b + 252, 64, f32)],                 # two outs by one element
                [(a, a + 4, 64, f32)],                                    # its own input, moved by an element
                [(c, c, 64, bf16), (c + 124, b, 4, bf16)]):               # read while it is scaled
        assert clip(*bad) == _lib.MPGNN_ERR_ARG, bad
        assert "overlaps" in lib.mpgnn_last_error().decode()


def test_grouped_linear_refuses_more_tiles_than_a_launch_has():
    """A launch has 2^32 - 1 threads at most: group counts that need more workgroups are refused as unsupported before
    anything is launched, not by a failed launch (no address here is read)."""
    for dt in (_lib.F32, _lib.BF16):
        for rows, groups, n in ((4, 1 << 24, 5), (4, 1 << 24, 1 << 20), (1 << 33, 1, 5), (1 << 30, 1 << 23, 1 << 20)):
            assert lib.mpgnn_grouped_linear_fwd(P, rows, 8, dt, P, groups, 8, n, None, P, 64, P,
                                                None) == _lib.MPGNN_ERR_UNSUPPORTED, (rows, groups, n)
            assert "tiles" in lib.mpgnn_last_error().decode()
            assert lib.mpgnn_grouped_linear_dgrad(P, rows, 8, dt, P, groups, n, 8, P, 64, P,
                                                  None) == _lib.MPGNN_ERR_UNSUPPORTED, (rows, groups, n)
        assert lib.mpgnn_grouped_linear_wgrad(P, 8, P, 5, 4, dt, 1 << 24, 8, 5, P, 64, P, None, P,
                                              None) == _lib.MPGNN_ERR_UNSUPPORTED
        assert lib.mpgnn_grouped_linear_wgrad(P, 1 << 22, P, 1 << 22, 4, dt, 1 << 14, 1 << 22, 1 << 22, P, 64, P, None, P,
                                              None) == _lib.MPGNN_ERR_UNSUPPORTED


def test_inline_assembly_writes_no_register_behind_the_compiler():
    """m0 cannot be named as clobbered (the compiler holds it reserved), so no assembly text may write it: it is an
    operand, "{m0}"."""
    import os
    import re
    src = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
    texts = [open(os.path.join(src, f)).read() for f in sorted(os.listdir(src)) if f.endswith((".hip", ".h"))]
    assert any('"{m0}"' in t for t in texts)
    assert not any(re.search(r"s_\w+ m0\s*,", t) for t in texts)


def test_the_c_library_builds_without_torch():
    """A host without torch's headers gets the C library and its stamp from the default target, and no module of
    other sources stays beside it; with them both are built. (What make would run, nothing is built here.)"""
    import os
    import shutil
    import subprocess
    src = os.path.join(os.path.dirname(_lib.LIB_PATH), "csrc")
    if shutil.which("make") is None:
        pytest.skip("no make")

    def commands(*args):
        out = subprocess.run(["make", "-n", "-B", "-C", src, *args], capture_output=True, text=True, timeout=60)
        assert out.returncode == 0, out.stderr
        return out.stdout

    alone = commands("TORCH=")
    assert "operators_torch" not in alone and "grouped_kernels.hip" in alone and "_srchash.py" in alone
    assert "rm -f ../_operators.so" in alone
    both = commands()
    assert "operators_torch.cpp" in both and "_srchash.py" in both


def test_net_pickled_before_it_had_norms():
    """A whole Net saved without the attributes of layer_norm=True loads and runs as one without norms; one with norms
    keeps them."""
    import copy
    import pickle
    net = mpgnn_amd.Net(4, 8, 2, 8, 3, 2)
    for name in ("norm1", "norm2"):
        del net.__dict__[name]
    old = pickle.loads(pickle.dumps(net))
    assert old.norm1 is None and old.norm2 is None
    assert old.state_dict().keys() == mpgnn_amd.Net(4, 8, 2, 8, 3, 2).state_dict().keys()
    normed = mpgnn_amd.Net(4, 8, 2, 8, 3, 2, layer_norm=True)
    for again in (pickle.loads(pickle.dumps(normed)), copy.deepcopy(normed)):
        assert isinstance(again.norm1, mpgnn_amd.LayerNorm) and isinstance(again.norm2, mpgnn_amd.LayerNorm)
        assert again.state_dict().keys() == normed.state_dict().keys()


def test_make_fx_is_refused():
    """As torch.jit.trace: the graph would hold the outputs' allocation and no kernel."""
    from torch.fx.experimental.proxy_tensor import make_fx
    x, w, ptr = torch.ones(4, 8), torch.ones(2, 8, 5), torch.tensor([0, 2, 4])
    for f in (lambda t: mpgnn_amd.layer_norm(t), lambda t: mpgnn_amd.grouped_linear(t, w, ptr),
              lambda t: mpgnn_amd.clip_by_global_norm([t], 1.0)[0]):
        with pytest.raises(NotImplementedError, match="make_fx"):
            make_fx(f)(x)
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # and nothing is left behind
        mpgnn_amd.layer_norm(x)


def test_tangents_pass_where_forward_mode_is_off():
    """Inside the forward of a torch.autograd.Function with a jvp of its own the inputs still carry their tangents:
    the calls there are not refused for them (here they go on to the next check)."""
    from torch.autograd import forward_ad
    w, ptr = torch.ones(2, 8, 5), torch.tensor([0, 2, 4])

    class Own(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, call):
            return call(x)

        @staticmethod
        def jvp(ctx, t, _):
            return t

    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.ones(4, 8), torch.ones(4, 8))
        for call in (lambda t: mpgnn_amd.layer_norm(t), lambda t: mpgnn_amd.grouped_linear(t, w, ptr),
                     lambda t: mpgnn_amd.clip_by_global_norm([t], 1.0)[0]):
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                Own.apply(x, call)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(x)
