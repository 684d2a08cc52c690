"""layer_norm, grouped_linear and the global-norm clipping on the GPU against their definitions in
64 bits, computed here on the CPU.

Tolerances. u = 2^-24 bounds fp32's rounding, ``half(T)`` = finfo(T).eps / 2 that of a result
rounded to type T. A sum of n fp32 terms in any order is off by at most (depth) * u * sum |terms|,
where depth counts the additions that a term passes through."""
import math

import pytest
import torch

import mpgnn_amd

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0") if torch.cuda.is_available() else None
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half the step of the type's subnormal numbers: what rounding a value near zero may cost."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, scale=1.0, shift=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def within(got, ref, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    bad = ~((got - ref).abs() <= tol)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {ref.numel()} off, worst "
                                 f"{float(((got - ref).abs() - tol)[bad].max()):.3e} over its tolerance")


# ---------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------
def ln_reference(x, w, b, dy, eps):
    x, dy = x.double(), None if dy is None else dy.double()
    f = x.shape[-1]
    w64 = torch.ones(f, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros(f, dtype=torch.float64) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1.0 / (((x - mean) ** 2).mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    y = xh * w64 + b64
    if dy is None:
        return y, xh, rstd, mean, w64, b64
    h = dy * w64
    dx = rstd * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True))
    return (y, xh, rstd, mean, w64, b64), dx, (dy * xh).flatten(0, -2).sum(0), dy.flatten(0, -2).sum(0)


def ln_depth(f):
    """Additions on the way of one term into a row's sum: at most 32 elements of a thread, six steps
    of a wave and sixteen waves; a row too wide for that is summed by 1,024 threads."""
    return 32 + 6 + 16 if f <= 16384 else f // 1024 + 1 + 22


def ln_tolerances(x, ref, dt, depth):
    y, xh, rstd, mean, w, b = ref
    a = x.double().abs().mean(-1, keepdim=True)
    # xhat: the mean is off by depth * u * mean|x|; the difference, the two products and rstd round,
    # and the variance (depth + 3 roundings, halved by the root) is off by twice the mean's part at most
    exh = rstd * (depth + 2) * U * a + (depth / 2 + 8) * U * xh.abs() + (rstd * (depth + 2) * U * a) * xh.abs()
    ty = exh * w.abs() + 3 * U * (xh * w).abs() + 2 * U * b.abs()
    return exh, ty + half(dt) * y.abs() + tiny(dt)


LN_SHAPES = [(1, 1), (1, 64), (7, 771), (5, 128), (300, 16), (33, 100), (1000, 256), (64, 1000), (3, 2047),
             (9, 4096), (130, 1024), (2, 8192), (2, 8200), (2, 16384), (3, 20001), (2049, 48), (1200, 2)]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("shape", LN_SHAPES, ids=str)
def test_layer_norm_against_64_bits(shape, dt):
    rows, f = shape
    g = gen(rows * 31 + f)
    x = rnd(g, rows, f, scale=2.0, shift=0.5, dtype=dt)
    w, b, dy = rnd(g, f, scale=0.3, shift=1.0, dtype=dt), rnd(g, f, dtype=dt), rnd(g, rows, f, dtype=dt)
    ref, dx, dw, db = ln_reference(x, w, b, dy, 1e-5)
    xg, wg, bg = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = mpgnn_amd.layer_norm(xg, wg, bg)
    assert y.dtype == dt and y.is_contiguous()
    y.backward(dy.to(DEV))
    depth = ln_depth(f)
    exh, ty = ln_tolerances(x, ref, dt, depth)
    within(y, ref[0], ty, "y")
    _, xh, rstd, _, w64, _ = ref
    h = dy.double() * w64
    m1, m2 = h.mean(-1, keepdim=True), (h * xh).mean(-1, keepdim=True)
    em1 = (depth + 2) * U * h.abs().mean(-1, keepdim=True)
    em2 = (depth + 3) * U * (h * xh).abs().mean(-1, keepdim=True) + (h.abs() * exh).mean(-1, keepdim=True)
    tdx = rstd * (4 * U * (h.abs() + m1.abs() + (xh * m2).abs()) + em1 + xh.abs() * em2 + exh * (m2.abs() + em2))
    relr = (depth / 2 + 8) * U + 2 * (rstd * (depth + 2) * U * x.double().abs().mean(-1, keepdim=True))
    tdx = tdx * (1 + relr) + relr * dx.abs()
    within(xg.grad, dx, tdx + half(dt) * dx.abs() + tiny(dt), "dx")
    # a term passes the additions of its thread's rows (a 512th of them, 16 row slots), the slots' and
    # the partial rows' sum (in 64 bits)
    n = rows // 512 + 1 + 20
    tdw = (dy.double().abs() * exh).sum(0) + n * U * (dy.double() * xh).abs().sum(0)
    within(wg.grad, dw, tdw + half(dt) * dw.abs() + tiny(dt), "dw")
    within(bg.grad, db, n * U * dy.double().abs().sum(0) + half(dt) * db.abs() + tiny(dt), "db")
    with torch.no_grad():
        assert torch.equal(mpgnn_amd.layer_norm(xg, wg, bg), y), "without gradients: the same values"


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("affine", ["both32", "weight", "bias", "none"])
def test_layer_norm_parameters(dt, affine):
    g = gen(5)
    rows, f = 37, 264
    x, dy = rnd(g, rows, f, dtype=dt), rnd(g, rows, f, dtype=dt)
    pdt = torch.float32 if affine == "both32" else dt
    w = rnd(g, f, dtype=pdt) if affine in ("both32", "weight") else None
    b = rnd(g, f, dtype=pdt) if affine in ("both32", "bias") else None
    ref, dx, dw, db = ln_reference(x, w, b, dy, 1e-3)
    xg = x.to(DEV).requires_grad_(True)
    wg, bg = (None if t is None else t.to(DEV).requires_grad_(True) for t in (w, b))
    y = mpgnn_amd.layer_norm(xg, wg, bg, 1e-3)
    y.backward(dy.to(DEV))
    exh, ty = ln_tolerances(x, ref, dt, ln_depth(f))
    within(y, ref[0], ty, "y")
    n = 21
    if w is not None:
        assert wg.grad.dtype == pdt
        t = (dy.double().abs() * exh).sum(0) + n * U * (dy.double() * ref[1]).abs().sum(0)
        within(wg.grad, dw, t + half(pdt) * dw.abs(), "dw")
    if b is not None:
        within(bg.grad, db, n * U * dy.double().abs().sum(0) + half(pdt) * db.abs(), "db")


def test_layer_norm_slices_leading_dimensions_and_broadcast_gradients():
    g = gen(9)
    wide = rnd(g, 50, 200).to(DEV)
    w, b = rnd(g, 64).to(DEV), rnd(g, 64).to(DEV)
    for off in (0, 3, 64):  # a column slice, aligned or not, is read in place
        sl = wide[:, off:off + 64]
        assert torch.equal(mpgnn_amd.layer_norm(sl, w, b)[:, :].cpu(),
                           mpgnn_amd.layer_norm(sl.contiguous(), w, b).cpu()) or off % 4, off
        ref = ln_reference(sl.cpu(), w.cpu(), b.cpu(), None, 1e-5)
        within(mpgnn_amd.layer_norm(sl, w, b), ref[0], ln_tolerances(sl.cpu(), ref, torch.float32, 54)[1], off)
    x3 = rnd(g, 3, 5, 64).to(DEV)
    assert torch.equal(mpgnn_amd.layer_norm(x3, w, b), mpgnn_amd.layer_norm(x3.view(15, 64), w, b).view(3, 5, 64))
    xt = rnd(g, 64, 15).to(DEV).t()  # strided along the row: copied
    assert torch.equal(mpgnn_amd.layer_norm(xt, w, b), mpgnn_amd.layer_norm(xt.contiguous(), w, b))
    # a broadcast output gradient (of a sum) and a sliced input's gradient
    base = wide.clone().requires_grad_(True)
    mpgnn_amd.layer_norm(base[:, 8:72], w, b).sum().backward()
    ref = ln_reference(base.detach().cpu()[:, 8:72], w.cpu(), b.cpu(), torch.ones(50, 64), 1e-5)[1]
    got = base.grad.cpu()
    assert float(got[:, :8].abs().max()) == 0.0 and float(got[:, 72:].abs().max()) == 0.0
    # sums of 64 terms |h| <= 4 cancel: 54 additions and a few products on values up to rstd * 16
    within(got[:, 8:72], ref, torch.full_like(ref, 200 * U * 16), "dx of a sum")


def test_layer_norm_empty_constant_and_non_finite_rows():
    w, b = torch.ones(8, device=DEV, requires_grad=True), torch.zeros(8, device=DEV, requires_grad=True)
    x = torch.empty(0, 8, device=DEV, requires_grad=True)
    y = mpgnn_amd.layer_norm(x, w, b)
    y.sum().backward()
    assert y.shape == (0, 8) and x.grad.shape == (0, 8)
    assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))
    x = torch.full((4, 8), 3.25, device=DEV)  # no variance: the bias
    x[1, 2] = math.inf
    x[2, 3] = math.nan
    y = mpgnn_amd.layer_norm(x, None, torch.full((8,), 0.5, device=DEV)).cpu()
    assert torch.equal(y[0], torch.full((8,), 0.5)) and torch.equal(y[3], torch.full((8,), 0.5))
    assert bool(torch.isnan(y[1]).any()) and bool(torch.isnan(y[2]).all())


def test_layer_norm_gradient_against_differences():
    """sum(c * layer_norm(x)) along a direction: central differences of step s of the kernel's own
    forward. The third derivative of y along a unit-variance direction is below 30 at these inputs'
    rstd (about 1), so the truncation is below 30 s^2 / 6 per output; each output is off by 60 u."""
    g = gen(3)
    rows, f, s = 6, 96, 2.0 ** -7
    x, w, b, c, v = (rnd(g, *sh).to(DEV) for sh in ((rows, f), (f,), (f,), (rows, f), (rows, f)))
    xg = x.clone().requires_grad_(True)
    mpgnn_amd.layer_norm(xg, w, b).backward(c)
    with torch.no_grad():
        up = (mpgnn_amd.layer_norm(x + s * v, w, b).double() * c).sum()
        dn = (mpgnn_amd.layer_norm(x - s * v, w, b).double() * c).sum()
    got, want = float((xg.grad.double() * v).sum()), float((up - dn) / (2 * s))
    cw = float((c * w).abs().sum())
    assert abs(got - want) <= cw * (5 * s * s + 60 * U * 4 / s), (got, want)


# ---------------------------------------------------------------------------------------
# grouped linear
# ---------------------------------------------------------------------------------------
def offsets(sizes, before=0):
    out = [before]
    for s in sizes:
        out.append(out[-1] + s)
    return out


def gl_reference(x, w, b, off, dy=None):
    x, w = x.double(), w.double()
    y = torch.zeros(x.shape[0], w.shape[2], dtype=torch.float64)
    mag = torch.zeros_like(y)
    for g in range(w.shape[0]):
        lo, hi = off[g], off[g + 1]
        y[lo:hi] = x[lo:hi] @ w[g] + (0 if b is None else b[g].double())
        mag[lo:hi] = x[lo:hi].abs() @ w[g].abs() + (0 if b is None else b[g].double().abs())
    if dy is None:
        return y, mag
    dy = dy.double()
    dx, dxm = torch.zeros_like(x), torch.zeros_like(x)
    dw, dwm = torch.zeros_like(w), torch.zeros_like(w)
    db = torch.zeros(w.shape[0], w.shape[2], dtype=torch.float64)
    dbm = torch.zeros_like(db)
    for g in range(w.shape[0]):
        lo, hi = off[g], off[g + 1]
        dx[lo:hi], dxm[lo:hi] = dy[lo:hi] @ w[g].t(), dy[lo:hi].abs() @ w[g].abs().t()
        dw[g], dwm[g] = x[lo:hi].t() @ dy[lo:hi], x[lo:hi].abs().t() @ dy[lo:hi].abs()
        db[g], dbm[g] = dy[lo:hi].sum(0), dy[lo:hi].abs().sum(0)
    return (y, mag), (dx, dxm), (dw, dwm), (db, dbm)


def gl_tol(ref, mag, length, dt):
    """A product of two 16-bit values is exact in fp32; the six piece products of two fp32 values miss
    at most 2^-25 of them. An output passes ceil(length / 32) accumulations (six times that from fp32)
    of matrix instructions that add 32 products: at most 33 roundings each, u * sum |products| each;
    one more for the bias. Roundings are independent of each other: four standard deviations of a
    random walk instead of their sum."""
    n = 33 * (6 if dt == torch.float32 else 1) * (-(-max(length, 1) // 32)) + 2
    return (4 * math.sqrt(n) + 2) * U * mag + half(dt) * ref.abs() + tiny(dt)


GL_CASES = [  # sizes, rows before the first group, rows behind the last, K, N
    ([1], 0, 0, 1, 1),
    ([0, 3, 0], 0, 0, 5, 7),
    ([0, 0], 0, 4, 16, 16),
    ([2, 0, 1, 130], 3, 5, 64, 128),
    ([128, 256, 1, 127], 0, 0, 128, 128),
    ([129, 0, 77], 0, 0, 193, 301),
    ([40, 300], 2, 1, 72, 136),
    ([1000, 17, 0, 3, 700], 0, 9, 256, 64),
    ([64] * 5, 0, 0, 32, 40),
    ([5000, 1, 0, 900], 0, 0, 128, 128),
    ([3, 1, 2], 0, 0, 515, 1030),
]


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("case", range(len(GL_CASES)))
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "bias"])
def test_grouped_linear_against_64_bits(case, dt, biased):
    sizes, before, behind, k, n = GL_CASES[case]
    g = gen(case)
    off = offsets(sizes, before)
    rows, groups = off[-1] + behind, len(sizes)
    x, w = rnd(g, rows, k, dtype=dt), rnd(g, groups, k, n, scale=k ** -0.5, dtype=dt)
    b = rnd(g, groups, n, dtype=dt) if biased else None
    dy = rnd(g, rows, n, dtype=dt)
    ry, rx, rw, rb = gl_reference(x, w, b, off, dy)
    xg, wg = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    bg = b.to(DEV).requires_grad_(True) if biased else None
    ptr = torch.tensor(off, dtype=torch.int32 if case % 2 else torch.int64, device=DEV)
    y = mpgnn_amd.grouped_linear(xg, wg, ptr, bg)
    assert y.dtype == dt
    y.backward(dy.to(DEV))
    within(y, *[ry[0], gl_tol(*ry, k, dt)], "y")
    within(xg.grad, rx[0], gl_tol(*rx, n, dt), "dx")
    longest = max(sizes)
    within(wg.grad, rw[0], gl_tol(*rw, longest, dt), "dw")
    if biased:
        # a column's rows: a sixteenth of a chunk in a row, then 16 partials, then the chunks
        within(bg.grad, rb[0], (longest / 16 + 40) * U * rb[1] + half(dt) * rb[0].abs() + tiny(dt), "db")
    out = [i for i in range(rows) if i < off[0] or i >= off[-1]]
    assert not out or float(y.detach()[out].abs().max()) == 0.0
    assert not out or float(xg.grad[out].abs().max()) == 0.0
    with torch.no_grad():
        assert torch.equal(mpgnn_amd.grouped_linear(xg, wg, ptr, bg), y)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("biased", [False, True], ids=["plain", "bias"])
@pytest.mark.parametrize("shape", [([5000, 1, 3100, 255], 3, 64, 4096), ([300] * 5 + [0, 900, 130], 0, 1024, 4096)],
                         ids=["rows", "weights"])
def test_grouped_linear_large(shape, dt, biased):
    """Sizes that fill the chip with the largest tiles (whole, halved and cut ones): rows over many
    columns, and many weights. The 64-bit products run on the GPU."""
    sizes, behind, k, n = shape
    g = gen(13)
    off = offsets(sizes)
    rows, groups = off[-1] + behind, len(sizes)
    x, w = rnd(g, rows, k, dtype=dt).to(DEV), rnd(g, groups, k, n, scale=k ** -0.5, dtype=dt).to(DEV)
    b = rnd(g, groups, n, dtype=dt).to(DEV) if biased else None
    dy = rnd(g, rows, n, dtype=dt).to(DEV)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b) if t is not None]
    y = mpgnn_amd.grouped_linear(leaves[0], leaves[1], torch.tensor(off, device=DEV), leaves[2] if biased else None)
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    for q in range(groups):
        lo, hi = off[q], off[q + 1]
        xg, wg, dg = x[lo:hi].double(), w[q].double(), dy[lo:hi].double()
        bg = b[q].double() if biased else torch.zeros(n, dtype=torch.float64, device=DEV)
        pairs = [(got[0][lo:hi], xg @ wg + bg, xg.abs() @ wg.abs() + bg.abs(), k),
                 (got[1][lo:hi], dg @ wg.t(), dg.abs() @ wg.abs().t(), n),
                 (got[2][q], xg.t() @ dg, xg.abs().t() @ dg.abs(), hi - lo)]
        for a, ref, mag, length in pairs:
            assert bool(((a.double() - ref).abs() <= gl_tol(ref, mag, length, dt)).all()), (q, length)
        if biased:
            ref = dg.sum(0)
            tol = ((hi - lo) / 16 + 40) * U * dg.abs().sum(0) + half(dt) * ref.abs() + tiny(dt)
            assert bool(((got[3][q].double() - ref).abs() <= tol).all()), q
    if behind:
        assert float(got[0][off[-1]:].abs().max()) == 0.0 and float(got[1][off[-1]:].abs().max()) == 0.0


def test_grouped_linear_fp32_is_as_near_as_fp32_products():
    """The split products against 64 bits, normwise: 24 accumulations of K = 128, rounding to 2^-24
    of partial sums of about the result's size each, and 2^-25 a product: below 2 sqrt(24) u."""
    g = gen(77)
    x, w = rnd(g, 900, 128), rnd(g, 2, 128, 128)
    off = [0, 400, 900]
    y = mpgnn_amd.grouped_linear(x.to(DEV), w.to(DEV), torch.tensor(off, device=DEV))
    ref, _ = gl_reference(x, w, None, off)
    assert float((y.cpu().double() - ref).norm() / ref.norm()) <= 2 * math.sqrt(24) * U


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_grouped_linear_strides_and_many_groups(dt):
    g = gen(21)
    sizes = [(i * 7) % 5 for i in range(700)]
    off = offsets(sizes, 1)
    rows, k, n = off[-1] + 2, 24, 33
    wide, dyw = rnd(g, rows, k + 9, dtype=dt).to(DEV), rnd(g, rows, n + 5, dtype=dt).to(DEV)
    w = rnd(g, 700, n, k, dtype=dt).to(DEV).transpose(1, 2)  # a strided weight is copied
    ptr = torch.tensor(off, device=DEV)
    ptr2 = torch.stack([ptr, ptr], 1)[:, 0]                   # so is a strided ptr
    for sl in (slice(0, k), slice(5, 5 + k)):
        base = wide.clone().requires_grad_(True)
        wl = w.clone().requires_grad_(True)
        y = mpgnn_amd.grouped_linear(base[:, sl], wl, ptr2)
        y.backward(dyw[:, 2:2 + n])
        ry, rx, rw, _ = gl_reference(wide[:, sl].cpu(), w.cpu(), None, off, dyw[:, 2:2 + n].cpu())
        within(y, ry[0], gl_tol(*ry, k, dt), "y")
        within(base.grad[:, sl], rx[0], gl_tol(*rx, n, dt), "dx")
        within(wl.grad, rw[0], gl_tol(*rw, 4, dt), "dw")


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_grouped_linear_non_finite_values_stay_in_their_group(dt):
    """A NaN or infinity in a row, a weight or a row of no group reaches what a sum of products hands it
    to and nothing else; a finite fp32 value near the largest gives finite products."""
    g = gen(4)
    off, k, n = [1, 70, 70, 140], 48, 40
    x, w, dy = rnd(g, 145, k, dtype=dt), rnd(g, 3, k, n, dtype=dt), rnd(g, 145, n, dtype=dt)
    x[0], dy[0], x[142], dy[142] = math.nan, math.inf, math.inf, math.nan  # no group's rows
    w[1] = math.nan                                                          # an empty group's weight
    x[10, 5] = math.inf
    x[80, 7] = math.nan
    w[2, 3, 9] = -math.inf
    dy[30, 2] = math.inf
    xg, wg = x.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    y = mpgnn_amd.grouped_linear(xg, wg, torch.tensor(off, device=DEV))
    y.backward(dy.to(DEV))

    def same(got, ref, what):
        got = got.detach().double().cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
        assert torch.equal(torch.where(got.isinf(), got, 0.0), torch.where(ref.isinf(), ref, 0.0)), what
        ok = torch.isfinite(ref)
        # sums of at most 140 products of values below 6
        assert float((got - ref)[ok].abs().max()) <= 140 * 36 * (140 * U + half(dt)), what

    def mm(a, b):  # products in 64 bits, one sum after the other: infinities as IEEE has them
        return (a.double().unsqueeze(2) * b.double().unsqueeze(0)).sum(1)

    ry, rx = torch.zeros(145, n, dtype=torch.float64), torch.zeros(145, k, dtype=torch.float64)
    for q in range(3):
        lo, hi = off[q], off[q + 1]
        ry[lo:hi], rx[lo:hi] = mm(x[lo:hi], w[q]), mm(dy[lo:hi], w[q].t())
    rw = torch.stack([mm(x[off[q]:off[q + 1]].t(), dy[off[q]:off[q + 1]]) for q in range(3)])
    same(y, ry, "y")
    same(xg.grad, rx, "dx")
    same(wg.grad, rw, "dw")
    big = torch.full((2, 8), 3.4e38)
    out = mpgnn_amd.grouped_linear(big.to(DEV), torch.eye(8, device=DEV)[None], torch.tensor([0, 2], device=DEV))
    assert torch.equal(out.cpu(), big)


def test_grouped_linear_gradient_against_differences():
    """The product is linear in each argument: differences of the kernel's own forward, of step 1, are
    exact up to the two forwards' roundings."""
    g = gen(6)
    off, k, n = [0, 50, 50, 131], 40, 56
    x, w, b, c = (rnd(g, *s).to(DEV) for s in ((131, k), (3, k, n), (3, n), (131, n)))
    ptr = torch.tensor(off, device=DEV)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    mpgnn_amd.grouped_linear(leaves[0], leaves[1], ptr, leaves[2]).backward(c)
    for k_, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=gen(k_)).to(DEV)
        args = [x, w, b]
        args[k_] = args[k_] + v
        with torch.no_grad():
            up = mpgnn_amd.grouped_linear(args[0], args[1], ptr, args[2]).double()
            at = mpgnn_amd.grouped_linear(x, w, ptr, b).double()
        want, got = float(((up - at) * c).sum()), float((leaf.grad.double() * v).sum())
        size = float(((up.abs() + at.abs()) * c.abs()).sum())
        assert abs(got - want) <= 200 * U * size, (k_, got, want)


# ---------------------------------------------------------------------------------------
# global norm and clipping
# ---------------------------------------------------------------------------------------
def clip_reference(ts, max_norm, kind):
    if kind == 2.0:
        norm = math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in ts))
    else:
        norm = max([float(t.double().abs().max()) for t in ts if t.numel()], default=0.0)
    return norm, min(1.0, max_norm / (norm + 1e-6))


CLIP_LISTS = {
    "one": [5], "empty_among": [0, 3, 0, 4097], "units": [4096, 8192, 4095, 8193], "small": [7, 1000, 33, 20000],
    "many": [17 + 13 * i for i in range(333)], "large": [3_000_001, 64, 1_500_000],
}


@pytest.mark.parametrize("kinds", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("name", list(CLIP_LISTS))
@pytest.mark.parametrize("norm_type", [2.0, math.inf])
def test_clip_by_global_norm(name, kinds, norm_type):
    g = gen(len(name))
    dts = {"fp32": [torch.float32], "bf16": [torch.bfloat16], "fp16": [torch.float16], "mixed": TYPES}[kinds]
    ts = [rnd(g, n, scale=0.5, dtype=dts[i % len(dts)]) for i, n in enumerate(CLIP_LISTS[name])]
    gpu = [t.to(DEV) for t in ts]
    full = clip_reference(ts, 1.0, norm_type)[0]
    for max_norm in (full / 3, full * 2):
        ref, factor = clip_reference(ts, max_norm, norm_type)
        norm, out = mpgnn_amd.clip_by_global_norm(gpu, max_norm, norm_type)
        # squares and their sum in 64 bits (over 5 M terms: below u), the root rounded once
        assert norm.dtype == torch.float32 and norm.dim() == 0
        assert abs(float(norm) - ref) <= 2 * U * ref
        for t, o, gt in zip(ts, out, gpu):
            want = t.double() * factor
            # norm, sum, quotient and max_norm rounded, then the product: at most 6 u before the last rounding
            within(o, want, (6 * U + half(t.dtype)) * want.abs() + tiny(t.dtype), name)
            if factor == 1.0:
                assert torch.equal(o, gt)
        again = [t.clone() for t in gpu]
        n2, o2 = mpgnn_amd.clip_by_global_norm(again, max_norm, norm_type, out=again)
        assert all(a is not b and torch.equal(a, c) for a, b, c in zip(o2, gpu, out)) and torch.equal(n2, norm)
        assert all(torch.equal(a, c) for a, c in zip(again, out)), "in place: the same values"


def test_clip_grad_norm_parameters_views_and_strides():
    g = gen(8)
    flat = rnd(g, 5003).to(DEV)
    p = [torch.nn.Parameter(torch.zeros(*s, device=DEV)) for s in ((10, 7), (33,), (40, 50), (4, 5), (3,))]
    p[0].grad = flat[1:71].view(10, 7)                       # not aligned to 16 bytes
    p[1].grad = flat[103:136]
    p[2].grad = rnd(g, 50, 40).to(DEV).t()                   # strided
    p[3].grad = flat[1000:1040].view(4, 10)[:, ::2]          # strided view: its gaps stay
    before = flat.clone()
    want = [q.grad.clone() for q in p[:4]]
    ref, factor = clip_reference([t.cpu() for t in want], 0.25, 2.0)
    norm = mpgnn_amd.clip_grad_norm_(iter(p), 0.25)          # p[4] has no gradient
    assert abs(float(norm) - ref) <= 2 * U * ref
    for q, t in zip(p, want):
        w64 = t.double().cpu() * factor
        within(q.grad, w64, 8 * U * w64.abs(), "grad")
    touched = torch.zeros_like(flat, dtype=torch.bool)
    touched[1:71] = touched[103:136] = True
    touched[1000:1040] = (torch.arange(40, device=DEV) % 2 == 0)
    assert torch.equal(flat[~touched], before[~touched]), "elements that belong to no gradient stay"
    assert p[4].grad is None
    assert float(mpgnn_amd.clip_grad_norm_([p[4]], 1.0)) == 0.0
    one = torch.nn.Parameter(torch.zeros(3, device=DEV))
    one.grad = torch.tensor([3.0, 4.0, 0.0], device=DEV)
    assert float(mpgnn_amd.clip_grad_norm_(one, 1.0)) == 5.0


def test_clip_extremes():
    """Gradients whose squares leave fp32's range, zeros, and values that are not finite."""
    for v, n in ((1e30, 4), (1e-30, 9)):
        t = torch.full((n,), v, device=DEV)
        norm, (out,) = mpgnn_amd.clip_by_global_norm([t], 1.0)
        assert abs(float(norm) - v * math.sqrt(n)) <= 4 * U * v * math.sqrt(n)
        want = min(1.0, 1.0 / (v * math.sqrt(n) + 1e-6)) * v
        assert abs(float(out[0]) - want) <= 8 * U * want
    z = torch.zeros(100, device=DEV)
    norm, (out,) = mpgnn_amd.clip_by_global_norm([z], 0.0)
    assert float(norm) == 0.0 and torch.equal(out, z)
    for bad, kind in ((math.inf, 2.0), (math.nan, 2.0), (math.nan, math.inf), (math.inf, math.inf)):
        a, b = torch.ones(70000, device=DEV), torch.ones(5, device=DEV)
        a[40000] = bad
        norm, (oa, ob) = mpgnn_amd.clip_by_global_norm([a, b], 1.0, kind)
        if math.isnan(bad):
            assert math.isnan(float(norm)) and bool(torch.isnan(oa).all()) and bool(torch.isnan(ob).all())
        else:
            assert float(norm) == math.inf and math.isnan(float(oa[40000]))
            assert float(oa[0]) == 0.0 and float(ob.abs().max()) == 0.0
        q = torch.nn.Parameter(torch.zeros_like(a))
        q.grad = a.clone()
        with pytest.raises(RuntimeError, match="non-finite"):
            mpgnn_amd.clip_grad_norm_([q], 1.0, kind, error_if_nonfinite=True)
        assert torch.equal(q.grad.nan_to_num(7.0), a.nan_to_num(7.0)), "nothing was scaled"


# ---------------------------------------------------------------------------------------
# together, streams, graphs, refusals
# ---------------------------------------------------------------------------------------
def _step_model(dt):
    g = gen(50)
    norm = mpgnn_amd.LayerNorm(48, device=DEV, dtype=dt)
    lin = mpgnn_amd.GroupedLinear(48, 40, 4, device=DEV, dtype=dt)
    with torch.no_grad():
        for p in (*norm.parameters(), *lin.parameters()):
            p.copy_(rnd(g, *p.shape, scale=0.3).to(DEV))
    off = offsets([30, 0, 100, 7])
    x, t = rnd(g, 140, 48, dtype=dt).to(DEV), rnd(g, 140, 40, dtype=dt).to(DEV)
    return norm, lin, torch.tensor(off, device=DEV), off, x, t


def test_norm_product_loss_clip_step_together():
    """layer_norm -> grouped_linear -> loss -> backward -> clip -> step, against the same step in 64 bits."""
    norm, lin, ptr, off, x, t = _step_model(torch.float32)
    params = [norm.weight, norm.bias, lin.weight, lin.bias]
    ref = [p.detach().cpu().double().requires_grad_(True) for p in params]
    x64 = x.cpu().double()
    xh = (x64 - x64.mean(1, keepdim=True)) / (x64.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    h = xh * ref[0] + ref[1]
    y = torch.cat([h[off[q]:off[q + 1]] @ ref[2][q] + ref[3][q] for q in range(4)] + [torch.zeros(3, 40).double()])
    ((y - t.cpu().double()) ** 2).sum().backward()
    rn, factor = clip_reference([p.grad for p in ref], 0.5, 2.0)
    out = lin(norm(x), ptr)
    ((out - t) ** 2).sum().backward()
    total = mpgnn_amd.clip_grad_norm_(params, 0.5)
    # gradients of sums over at most 137 rows and 48 columns: relative to their own norm far below 2^-14
    assert abs(float(total) - rn) <= 2.0 ** -14 * rn
    for p, q in zip(params, ref):
        want = q.grad * factor
        assert float((p.grad.cpu().double() - want).norm()) <= 2.0 ** -14 * float(want.norm())
    before = [p.detach().clone() for p in params]
    torch.optim.SGD(params, lr=0.1).step()
    for p, a in zip(params, before):
        # torch's step may round a - 0.1 * grad once; in 64 bits here: the constant, the product and the result
        want = a.double().cpu() - 0.1 * p.grad.double().cpu()
        within(p, want, 2 * U * want.abs() + 2 * U * (0.1 * p.grad.double().cpu()).abs(), "step")


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_training_step_captured_and_replayed(dt):
    """The whole step in a graph, replayed between other work on new inputs: every replay equals the
    eager step bit for bit. ptr is data too: its values change between replays."""
    norm, lin, ptr, off, x, t = _step_model(dt)
    params = [norm.weight, norm.bias, lin.weight, lin.bias]
    sx, sp = x.clone(), ptr.clone()

    def step():
        grads = torch.autograd.grad((lin(norm(sx), sp).float() - t.float()).square().sum(), params)
        total, clipped = mpgnn_amd.clip_by_global_norm(grads, 0.5)
        return [total, *clipped]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for k in range(4):
        sx.copy_(rnd(gen(k), 140, 48, dtype=dt))
        sp.copy_(torch.tensor(offsets([30, 10 * k, 90 - 10 * k, 7], k)))
        graph.replay()
        got = [s.clone() for s in static]
        torch.cuda.synchronize()
        junk = torch.randn(1000, 1000, device=DEV).sum()  # eager work between the replays
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), k
        del junk


def test_two_graphs_and_another_stream():
    """Two captured backwards replayed on two streams at once, and a call on a stream of its own."""
    g = gen(60)
    off = offsets([700, 0, 1500, 300])
    ptr = torch.tensor(off, device=DEV)
    made, kept = [], []
    for k in range(2):
        x, w, b = (rnd(g, *s).to(DEV).requires_grad_(True) for s in ((2500, 128), (4, 128, 128), (4, 128)))
        dy = rnd(g, 2500, 128).to(DEV)

        def run(x=x, w=w, b=b, dy=dy):
            return torch.autograd.grad(mpgnn_amd.grouped_linear(mpgnn_amd.layer_norm(x), w, ptr, b), (x, w, b), dy)

        want = run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = run()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, c) for a, c in zip(other, want)), "another stream"
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static = run()
        made.append((graph, static, want, side))
        kept.append(run)  # the graph reads these inputs at every replay
    for _ in range(3):
        for graph, _, _, side in made:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
        for _, _, _, side in made:
            torch.cuda.current_stream().wait_stream(side)
        for _, static, want, _ in made:
            assert all(torch.equal(a, c) for a, c in zip(static, want))


def test_results_repeat_bitwise():
    g = gen(70)
    x, w = rnd(g, 6000, 96).to(DEV).requires_grad_(True), rnd(g, 3, 96, 80).to(DEV).requires_grad_(True)
    nw, nb = (rnd(g, 96).to(DEV).requires_grad_(True) for _ in range(2))
    ptr, dy = torch.tensor([0, 5000, 5000, 5990], device=DEV), rnd(g, 6000, 80).to(DEV)
    runs = []
    for _ in range(3):
        grads = torch.autograd.grad(mpgnn_amd.grouped_linear(mpgnn_amd.layer_norm(x, nw, nb), w, ptr), (x, w, nw, nb), dy)
        runs.append([*grads, *mpgnn_amd.clip_by_global_norm(grads, 0.1)[1]])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(r, runs[0]))


def _small_graph_data():
    from mpgnn_amd import data, main
    g = data.synthetic_graph(400, 4, 6, feat_dim=16, seed=3)
    gen_ = gen(90)
    idx = torch.randperm(400, generator=gen_)
    y = torch.randint(0, 3, (400,), generator=gen_)
    return main.Data(x=g.x, edge_index=g.edge_index, edge_type=g.edge_type, train_idx=idx[:200], train_y=y[idx[:200]],
                     val_idx=idx[200:300], val_y=y[idx[200:300]], test_idx=idx[300:], test_y=y[idx[300:]]).to(DEV)


def test_net_with_layer_norm_and_clipped_step():
    """Net(layer_norm=True): its forward and gradients equal those of the same model with torch's own
    LayerNorm modules in place; the training step then clips what it steps with."""
    from mpgnn_amd import main_rgcn
    data = _small_graph_data()
    torch.manual_seed(5)
    net = mpgnn_amd.Net(16, 32, 4, 32, 3, 3, layer_norm=True).to(DEV)
    assert sorted(set(net.state_dict()) - set(mpgnn_amd.Net(16, 32, 4, 32, 3, 3).state_dict())) == \
        ["norm1.bias", "norm1.weight", "norm2.bias", "norm2.weight"]
    with torch.no_grad():
        for p in (net.norm1.weight, net.norm2.weight):
            p.add_(torch.linspace(-0.5, 0.5, 32, device=DEV))
    ref = mpgnn_amd.Net(16, 32, 4, 32, 3, 3).to(DEV)
    ref.norm1, ref.norm2 = torch.nn.LayerNorm(32).to(DEV), torch.nn.LayerNorm(32).to(DEV)
    ref.load_state_dict(net.state_dict())
    outs = []
    for m in (net, ref):
        out = m(data.x, data.edge_index, data.edge_type)
        out[data.train_idx].gather(1, data.train_y[:, None]).sum().neg().backward()
        outs.append(out)
    # both sides' norms are fp32 with errors of about 2^-22; three layers and a log-softmax of them
    assert float((outs[0] - outs[1]).detach().abs().max()) <= 1e-4
    for (n, a), b in zip(net.named_parameters(), ref.parameters()):
        assert a.grad is not None, n
        assert float((a.grad - b.grad).norm()) <= 1e-4 * float(b.grad.norm()) + 1e-6, n
    opt = torch.optim.SGD(net.parameters(), lr=0.0)
    main_rgcn.mpgnn_train(net, opt, data, max_grad_norm=1e-3)
    total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in net.parameters()))
    assert 0.99e-3 <= total <= 1.001e-3


def test_loops_take_the_additions(monkeypatch):
    """The training loops with layer_norm and max_grad_norm, their epochs captured in a graph or not: the
    same scores. Left out, nothing changes."""
    from mpgnn_amd import main, main_rgcn
    data = _small_graph_data()
    scores = {}
    for graph in ("1", "0"):
        monkeypatch.setenv("MPGNN_LOOP_GRAPH", graph)
        torch.manual_seed(30)
        scores[graph, "rgcn"] = main_rgcn.mpgnn_parallel_multiple(data, 16, 32, 4, 32, 3, 2, epochs=8, verbose=False,
                                                                  layer_norm=True, max_grad_norm=0.5)
        torch.manual_seed(30)
        scores[graph, "mpgnn"] = main.mpgnn_parallel_multiple(data, 16, 32, 4, 32, 3, [[0, 1]], epochs=8,
                                                              max_grad_norm=0.5)
        torch.manual_seed(30)
        scores[graph, "plain"] = main_rgcn.mpgnn_parallel_multiple(data, 16, 32, 4, 32, 3, 2, epochs=8, verbose=False)
    assert scores["1", "rgcn"] == scores["0", "rgcn"]
    assert scores["1", "plain"] == scores["0", "plain"]
    assert all(0.0 <= float(v) <= 1.0 for v in scores.values())


def test_gpu_refusals():
    x = torch.zeros(4, 8, device=DEV)
    with pytest.raises(TypeError):
        mpgnn_amd.layer_norm(x.double())
    with pytest.raises(TypeError):
        mpgnn_amd.layer_norm(x, torch.ones(8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        mpgnn_amd.layer_norm(x.half(), torch.ones(8, device=DEV).half(), torch.ones(8, device=DEV))
    with pytest.raises(ValueError):
        mpgnn_amd.layer_norm(x, torch.ones(7, device=DEV))
    with pytest.raises(ValueError):
        mpgnn_amd.layer_norm(torch.zeros(4, 0, device=DEV))
    with pytest.raises(RuntimeError, match="CPU"):
        mpgnn_amd.layer_norm(x, torch.ones(8))
    w, ptr = torch.zeros(2, 8, 5, device=DEV), torch.tensor([0, 2, 4], device=DEV)
    with pytest.raises(RuntimeError, match="multiplied"):
        mpgnn_amd.grouped_linear(x[:, :7], w, ptr)
    with pytest.raises(ValueError):
        mpgnn_amd.grouped_linear(x, w, ptr[:2])
    with pytest.raises(TypeError):
        mpgnn_amd.grouped_linear(x, w, ptr.float())
    with pytest.raises(RuntimeError):
        mpgnn_amd.grouped_linear(x, w, ptr.cpu())
    with pytest.raises(TypeError):
        mpgnn_amd.grouped_linear(x, w.half(), ptr)
    with pytest.raises(ValueError):
        mpgnn_amd.grouped_linear(x, w, ptr, torch.zeros(2, 4, device=DEV))
    with pytest.raises(ValueError):
        mpgnn_amd.grouped_linear(x, torch.zeros(2, 8, 0, device=DEV), ptr)
    with pytest.raises(ValueError, match="twice"):
        mpgnn_amd.clip_by_global_norm([x], 1.0, out=[x, x][:1]) and mpgnn_amd.clip_by_global_norm([x, x], 1.0, out=[x, x])
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([x], -1.0)
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([x], math.nan)
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([x], 1.0, norm_type=1.0)
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([], 1.0)
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([x], 1.0, out=[torch.zeros(4, 9, device=DEV)[:, :8]])
    with pytest.raises(TypeError):
        mpgnn_amd.clip_by_global_norm([x.double()], 1.0)
    p = torch.nn.Parameter(torch.zeros(4, 8, device=DEV))
    p.grad = torch.ones(1, 8, device=DEV).expand(4, 8)
    with pytest.raises(ValueError, match="expanded"):
        mpgnn_amd.clip_grad_norm_([p], 1.0)
    y = mpgnn_amd.layer_norm(x.clone().requires_grad_(True))
    with pytest.raises(RuntimeError):  # differentiable once
        gx = torch.autograd.grad(y.sum(), y.grad_fn.next_functions[0][0].variable, create_graph=True)[0]
        gx.sum().backward()


def test_wrong_ptr_stays_inside_the_tensors():
    """A ptr that is negative, past the end or decreasing is clamped by the kernels: results of its
    groups are unspecified, rows of others and the memory around are not touched."""
    g = gen(2)
    x, w = rnd(g, 64, 32).to(DEV), rnd(g, 3, 32, 16).to(DEV)
    for vals in ([-5, 10, 20, 1 << 40], [0, 64, 64, 64], [100, 200, 300, 400], [-9, -8, -7, -6]):
        y = mpgnn_amd.grouped_linear(x, w, torch.tensor(vals, device=DEV))
        clamped = [min(max(v, 0), 64) for v in vals]
        ref, mag = gl_reference(x.cpu(), w.cpu(), None, clamped)
        within(y, ref, gl_tol(ref, mag, 32, torch.float32), vals)


def test_graphs_of_the_backward():
    """No second derivative by any argument, also where the incoming gradient is a constant; a graph is
    run once unless it is kept; a saved tensor that is written to is noticed."""
    g = gen(77)
    x, w = rnd(g, 6, 8).to(DEV).requires_grad_(True), rnd(g, 2, 8, 5).to(DEV).requires_grad_(True)
    ptr = torch.tensor([0, 2, 6], device=DEV)
    for f in (lambda t: mpgnn_amd.layer_norm(t), lambda t: mpgnn_amd.grouped_linear(t, w, ptr)):
        first = torch.autograd.grad(f(x).sum(), x)[0]
        gx = torch.autograd.grad(f(x).sum(), x, create_graph=True)[0]
        assert torch.equal(gx.detach(), first)
        with pytest.raises(RuntimeError, match="second derivative"):
            (gx * gx).sum().backward()
        y = f(x)
        for _ in range(2):
            assert torch.equal(torch.autograd.grad(y.sum(), x, retain_graph=True)[0], first)
        torch.autograd.grad(y.sum(), x)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y.sum(), x)
        z = x * 1.0
        y = f(z)
        z.mul_(2.0)
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()
    # the graph of another argument only
    y = mpgnn_amd.grouped_linear(x.detach(), w, ptr)
    dw = torch.autograd.grad(y.sum(), w)[0]
    assert torch.equal(dw, torch.autograd.grad(mpgnn_amd.grouped_linear(x, w, ptr).sum(), w)[0])


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("k, n", [(264, 328), (233, 331), (330, 259), (72, 840), (576, 264)])
def test_grouped_linear_tiles_between(k, n, dt):
    """Rows and columns enough for tiles of 128 x 128 in each direction, and too few for larger ones: aligned
    and odd widths, rows of no group, an empty group, a strided x. The 64-bit products run on the GPU."""
    sizes, before, behind = [1700, 0, 1, 990, 1633, 127], 2, 5
    g = gen(31)
    off = offsets(sizes, before)
    rows, groups = off[-1] + behind, len(sizes)
    x = rnd(g, rows, k + 8, dtype=dt).to(DEV)[:, 8:]
    w, b = rnd(g, groups, k, n, scale=k ** -0.5, dtype=dt).to(DEV), rnd(g, groups, n, dtype=dt).to(DEV)
    dy = rnd(g, rows, n, dtype=dt).to(DEV)
    leaves = [x.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
    y = mpgnn_amd.grouped_linear(leaves[0], leaves[1], torch.tensor(off, device=DEV), leaves[2])
    got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    for q in range(groups):
        lo, hi = off[q], off[q + 1]
        xg, wg, dg, bg = x[lo:hi].double(), w[q].double(), dy[lo:hi].double(), b[q].double()
        for a, ref, mag, length in [(got[0][lo:hi], xg @ wg + bg, xg.abs() @ wg.abs() + bg.abs(), k),
                                    (got[1][lo:hi], dg @ wg.t(), dg.abs() @ wg.abs().t(), n),
                                    (got[2][q], xg.t() @ dg, xg.abs().t() @ dg.abs(), hi - lo)]:
            assert bool(((a.double() - ref).abs() <= gl_tol(ref, mag, length, dt)).all()), (q, length)
        ref = dg.sum(0)
        tol = ((hi - lo) / 16 + 40) * U * dg.abs().sum(0) + half(dt) * ref.abs() + tiny(dt)
        assert bool(((got[3][q].double() - ref).abs() <= tol).all()), q
    out = [i for i in range(rows) if i < off[0] or i >= off[-1]]
    assert float(got[0][out].abs().max()) == 0.0 and float(got[1][out].abs().max()) == 0.0
    # an infinity and a NaN reach their own row, and the weight's row, alone
    x[700, 5], x[3000, 9] = math.inf, math.nan
    y2 = mpgnn_amd.grouped_linear(x, w, torch.tensor(off, device=DEV), b)
    rest = [i for i in range(rows) if i not in (700, 3000)]
    assert torch.equal(y2[rest], got[0][rest])
    assert bool(y2[3000].isnan().all()) and not bool(y2[700].isfinite().any())
    ref = x[700].double() @ w[0].double() + b[0].double()
    assert torch.equal(y2[700].double(), ref.to(dt).double())


def _one_step(seed, dt):
    """Norm, grouped product, their gradients and the clipping of these, as one list of tensors."""
    g = gen(seed)
    x, w = rnd(g, 300, 72, dtype=dt).to(DEV).requires_grad_(True), rnd(g, 3, 72, 40, dtype=dt).to(DEV).requires_grad_(True)
    lw, lb = rnd(g, 72, dtype=dt).to(DEV).requires_grad_(True), rnd(g, 72, dtype=dt).to(DEV).requires_grad_(True)
    ptr = torch.tensor([0, 100, 130, 300], device=DEV)
    y = mpgnn_amd.grouped_linear(mpgnn_amd.layer_norm(x, lw, lb), w, ptr)
    grads = torch.autograd.grad(y.float().square().mean(), [x, lw, lb, w])
    norm, clipped = mpgnn_amd.clip_by_global_norm(grads, 1e-3)
    return [y.detach(), *grads, norm, *clipped]


def test_threads_with_streams_of_their_own():
    """Several threads call at once (the calls leave the interpreter's lock), each on its own stream."""
    import threading
    kinds = [(s, TYPES[s % 3]) for s in range(6)]
    want = [_one_step(s, dt) for s, dt in kinds]
    torch.cuda.synchronize()
    got, errors = [None] * len(kinds), []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = _one_step(*kinds[i])
                torch.cuda.current_stream().synchronize()
        except Exception as exc:  # noqa: BLE001 - shown by the main thread
            errors.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(kinds))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(want, got):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_checkpointed_and_hooked():
    """Recomputed activations and saved-tensor hooks (packed to the host) give the same gradients."""
    from torch.utils.checkpoint import checkpoint
    g = gen(8)
    x, w = rnd(g, 50, 24).to(DEV).requires_grad_(True), rnd(g, 2, 24, 17).to(DEV).requires_grad_(True)
    ptr = torch.tensor([0, 20, 50], device=DEV)

    def f(t):
        return mpgnn_amd.grouped_linear(mpgnn_amd.layer_norm(t), w, ptr).square().sum()

    want = torch.autograd.grad(f(x), [x, w])
    again = torch.autograd.grad(checkpoint(f, x, use_reentrant=False), [x, w])
    with torch.autograd.graph.save_on_cpu():
        y = f(x)
    host = torch.autograd.grad(y, [x, w])
    for other in (again, host):
        assert all(torch.equal(a, b) for a, b in zip(want, other))


def test_odd_arguments():
    x = torch.ones(4, 8, device=DEV)
    for bad in (None, [1.0], "x"):
        with pytest.raises((TypeError, AttributeError)):
            mpgnn_amd.layer_norm(bad)
    with pytest.raises(TypeError):
        mpgnn_amd.layer_norm(x.to_sparse())
    with pytest.raises(TypeError):
        mpgnn_amd.clip_by_global_norm([x.to_sparse()], 1.0)
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([x], 1.0, out=[])
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([x], 1.0, out=[x.half()])
    with pytest.raises(ValueError):
        mpgnn_amd.grouped_linear(x, torch.ones(8, 5, device=DEV), torch.tensor([0, 4], device=DEV))
    assert mpgnn_amd.layer_norm(x, eps=1).dtype == torch.float32
    # one row, one element, no rows, all leading dimensions
    assert float(mpgnn_amd.layer_norm(torch.full((1, 1), 7.0, device=DEV))) == 0.0
    assert mpgnn_amd.layer_norm(torch.zeros(0, 8, device=DEV)).shape == (0, 8)
    assert mpgnn_amd.layer_norm(torch.zeros(8, device=DEV)).shape == (8,)
    v = torch.zeros(0, 8, device=DEV, requires_grad=True)
    lw = torch.ones(8, device=DEV, requires_grad=True)
    gv, gw = torch.autograd.grad(mpgnn_amd.layer_norm(v, lw).sum(), [v, lw])
    assert gv.shape == (0, 8) and float(gw.abs().max()) == 0.0
    w = torch.ones(2, 8, 5, device=DEV, requires_grad=True)
    y = mpgnn_amd.grouped_linear(v, w, torch.zeros(3, dtype=torch.int64, device=DEV))
    gv, gw = torch.autograd.grad(y.sum(), [v, w])
    assert gv.shape == (0, 8) and float(gw.abs().max()) == 0.0


@pytest.mark.parametrize("dt", TYPES, ids=str)
def test_overlapping_groups_stay_inside_the_workspace(dt):
    """A ptr that decreases makes groups overlap and have more chunks between them than there are slabs: the
    weight gradient writes neither behind its workspace nor behind its outputs."""
    import ctypes
    from mpgnn_amd import _lib
    code = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}[dt]
    g = gen(3)
    for rows, k, n in ((6000, 40, 24), (6000, 264, 200), (9000, 1200, 600)):
        x, dy = rnd(g, rows, k, dtype=dt).to(DEV), rnd(g, rows, n, dtype=dt).to(DEV)
        vals = [0, rows, 100, rows, 7, rows, 0, rows]
        groups = len(vals) - 1
        ptr = torch.tensor(vals, device=DEV)
        need = ctypes.c_int64()
        assert _lib.lib.mpgnn_grouped_linear_wgrad_workspace_bytes(rows, groups, k, n, ctypes.byref(need)) == 0
        pad = 1 << 20
        ws = torch.full((need.value + pad,), 0x5A, dtype=torch.uint8, device=DEV)
        dw = torch.full((groups * k * n + pad,), 7.0, dtype=dt, device=DEV)
        db = torch.full((groups * n + pad,), 7.0, dtype=dt, device=DEV)
        st = _lib.lib.mpgnn_grouped_linear_wgrad(x.data_ptr(), k, dy.data_ptr(), n, rows, code, groups, k, n,
                                                 ptr.data_ptr(), 64, dw.data_ptr(), db.data_ptr(), ws.data_ptr(),
                                                 torch.cuda.current_stream().cuda_stream)
        assert st == 0
        torch.cuda.synchronize()
        assert bool((ws[need.value:] == 0x5A).all()) and bool((dw[groups * k * n:] == 7.0).all())
        assert bool((db[groups * n:] == 7.0).all())


def test_tangents_and_traces_are_refused_on_the_gpu():
    """As on the CPU, and for a tangent that the backward meets on the incoming gradient."""
    from torch.autograd import forward_ad
    g = gen(91)
    x, w = rnd(g, 6, 8).to(DEV), rnd(g, 2, 8, 8).to(DEV)
    ptr = torch.tensor([0, 2, 6], device=DEV)
    calls = (lambda t: mpgnn_amd.layer_norm(t), lambda t: mpgnn_amd.grouped_linear(t, w, ptr))
    with forward_ad.dual_level():
        for f in calls + (lambda t: mpgnn_amd.clip_by_global_norm([w, t], 1.0),):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f(forward_ad.make_dual(x, x))
        for f in calls:
            xg = x.clone().requires_grad_(True)
            y = f(xg)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, xg, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
    for f in calls + (lambda t: mpgnn_amd.clip_by_global_norm([t], 1.0)[0],):
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(f, (x,))
        f(x)  # and nothing is left behind


@pytest.mark.parametrize("rows, f, dt", [(40000, 64, torch.float32), (5000, 771, torch.float32),
                                         (600, 20001, torch.float32), (600, 20001, torch.bfloat16),
                                         (5000, 771, torch.bfloat16)], ids=str)
def test_layer_norm_infinite_gradients_in_the_parameters_sums(rows, f, dt):
    """Infinities of one sign in a column of dy make its sums infinite, of both signs or a NaN no number, as the
    formula has it, whatever rows follow them in the same thread; the other columns are as without them."""
    g = gen(rows + f)
    x, dy = rnd(g, rows, f, dtype=dt), rnd(g, rows, f, dtype=dt)
    w, b = torch.ones(f, dtype=dt), torch.zeros(f, dtype=dt)
    xg, wg, bg = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = mpgnn_amd.layer_norm(xg, wg, bg)
    clean = torch.autograd.grad(y, (wg, bg), dy.to(DEV), retain_graph=True)
    dy[3, 5] = math.inf
    dy[2, 9] = -math.inf
    dy[rows - 1, 9] = -math.inf
    dy[3, 60], dy[11, 60] = math.inf, -math.inf
    dy[3, 33] = math.nan
    _, _, dw, db = ln_reference(x, w, b, dy, 1e-5)
    # dw[9] takes -inf * xhat of two rows and is what their signs make it: infinite or NaN
    for got, ref, old in zip(torch.autograd.grad(y, (wg, bg), dy.to(DEV)), (dw, db), clean):
        got = got.double().cpu()
        cols = [5, 9, 33, 60]
        assert torch.equal(torch.nan_to_num(got[cols], 1.0, 2.0, 3.0), torch.nan_to_num(ref[cols], 1.0, 2.0, 3.0)), got[cols]
        rest = torch.ones(f, dtype=torch.bool)
        rest[cols] = False
        assert torch.equal(got[rest], old.double().cpu()[rest])


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("n", [1, 3, 8, 17, 64, 1000, 9001, 50000])
def test_clip_norm_is_the_exact_one_rounded(n, dt):
    """Squares and sums in 64 bits and one rounding to fp32, by at most 2^-24 of the norm (the 64-bit sums of both
    sides add less than n * 2^-52): small lists, where errors of many vectors do not average out, and large ones."""
    for seed in range(12):
        t = rnd(gen(1000 * n + seed), n, scale=10.0 ** (seed % 5 - 2), dtype=dt)
        ref = float(t.double().square().sum().sqrt())
        norm, _ = mpgnn_amd.clip_by_global_norm([t.to(DEV)], 1.0)
        assert abs(float(norm.double()) - ref) <= (U + n * 2.0 ** -51) * ref, (seed, float(norm), ref)


def test_clip_overlapping_and_neighbouring_tensors():
    """Views that share elements with another tensor of the list are refused before anything is written; neighbours in
    one bucket, and strided slices that interleave, are clipped as tensors of their own."""
    flat = rnd(gen(92), 4096, scale=3.0).to(DEV)
    kept = flat.clone()
    a, b = flat[:1000], flat[1000:3000]
    for tensors, out in (([flat, a], None), ([b, flat[2999:3001]], None), ([a, b[:1000]], [b[:1000], a]),
                         ([flat[:64]], [flat[1:65]]), ([a, b], [flat[3000:4000], flat[500:2500]])):
        with pytest.raises(ValueError, match="overlaps"):
            if out is None:
                params = [torch.nn.Parameter(t.clone()) for t in tensors]
                for p, t in zip(params, tensors):
                    p.grad = t
                mpgnn_amd.clip_grad_norm_(params, 1.0)
            else:
                mpgnn_amd.clip_by_global_norm(tensors, 1.0, out=out)
        assert torch.equal(flat, kept)
    assert mpgnn_amd.clip_by_global_norm([flat, a], 1.0)[1][1].shape == a.shape  # new tensors: the inputs may overlap
    parts = [flat[:1000], flat[1000:3000], flat[3000:3000], flat[3000:]]
    norm, _ = mpgnn_amd.clip_by_global_norm(parts[::-1], 1.0, out=parts[::-1])
    ref = kept.double().cpu()
    n = float(ref.square().sum().sqrt())
    # the factor's division and sum, its product with the element and the norm round: five roundings
    within(flat, ref / (n + 1e-6), 6 * U * ref.abs() / n, "neighbours")
    grid = kept.view(64, 64).clone()
    params = [torch.nn.Parameter(torch.zeros(64, 40, device=DEV)), torch.nn.Parameter(torch.zeros(64, 24, device=DEV))]
    params[0].grad, params[1].grad = grid[:, :40], grid[:, 40:]
    mpgnn_amd.clip_grad_norm_(params, 1.0)
    within(grid, (ref / (n + 1e-6)).view(64, 64), (6 * U * ref.abs() / n).view(64, 64), "interleaved")


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("rows, k, n", [(48, 40, 24), (2000, 264, 200), (2001, 233, 331), (30000, 256, 1024)], ids=str)
def test_decreasing_ptr_stays_inside_the_outputs(rows, k, n, dt):
    """Groups that overlap because ptr decreases: forward and input gradient write neither before nor behind their
    outputs (the overlapped rows' values are unspecified)."""
    from mpgnn_amd import _lib
    code = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}[dt]
    g = gen(rows + k)
    pad = 1 << 16
    x, dy = rnd(g, rows, k, dtype=dt).to(DEV), rnd(g, rows, n, dtype=dt).to(DEV)
    for vals in ([0, rows, 0, rows, 0], [rows, 0], [rows // 2, 3, rows, 5, rows + 9, -4], [rows, rows // 3, 1]):
        groups = len(vals) - 1
        w = rnd(g, groups, k, n, dtype=dt).to(DEV)
        for bits, it in ((64, torch.int64), (32, torch.int32)):
            ptr = torch.tensor(vals, device=DEV, dtype=it)
            for call, r, width, cols in ((_lib.lib.mpgnn_grouped_linear_fwd, x, k, n),
                                         (_lib.lib.mpgnn_grouped_linear_dgrad, dy, n, k)):
                out = torch.full((2 * pad + rows * cols,), 7.0, dtype=dt, device=DEV)
                bias = (None,) if r is x else ()
                st = call(r.data_ptr(), rows, width, code, w.data_ptr(), groups, k, n, *bias, ptr.data_ptr(), bits,
                          out[pad:].data_ptr(), torch.cuda.current_stream().cuda_stream)
                assert st == _lib.MPGNN_OK
                torch.cuda.synchronize()
                assert bool((out[:pad] == 7.0).all()) and bool((out[pad + rows * cols:] == 7.0).all()), (vals, bits)


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("off", [0, 1, 2, 3, 5])
def test_layer_norm_slices_at_every_offset(off, dt):
    """Column slices that start at any element against the definition, whichever loads their alignment takes."""
    g = gen(40 + off)
    rows, f = 65, 264
    wide = rnd(g, rows, f + 9, scale=2.0, shift=0.5, dtype=dt)
    ref = ln_reference(wide[:, off:off + f], None, None, None, 1e-5)
    _, ty = ln_tolerances(wide[:, off:off + f], ref, dt, ln_depth(f))
    within(mpgnn_amd.layer_norm(wide.to(DEV)[:, off:off + f]), ref[0], ty, off)


def test_views_that_negate_their_memory():
    """The imaginary part of a conjugate is a view whose memory holds the negative: as its values, in every place."""
    g = gen(93)
    neg = torch._neg_view
    x, w, b = (rnd(g, *s).to(DEV) for s in ((6, 8), (2, 8, 5), (2, 5)))
    v, dy, dz = rnd(g, 8).to(DEV), rnd(g, 6, 8).to(DEV), rnd(g, 6, 5).to(DEV)
    ptr = torch.tensor([0, 2, 6], device=DEV)
    one = torch.complex(rnd(g, 1), rnd(g, 1)).to(DEV).conj().imag  # contiguous by its only element
    assert one.is_neg() and one.is_contiguous()
    norm, (clipped,) = mpgnn_amd.clip_by_global_norm([one], 1e3)
    assert torch.equal(clipped, one.clone()) and float(norm) == abs(float(one))
    for t in (x, x[:, 1:7], x.t()):
        assert torch.equal(mpgnn_amd.layer_norm(neg(t)), mpgnn_amd.layer_norm(-t))
    assert torch.equal(mpgnn_amd.layer_norm(x, neg(v), neg(v)), mpgnn_amd.layer_norm(x, -v, -v))
    plain = mpgnn_amd.grouped_linear(-x, -w, ptr, -b)
    assert torch.equal(mpgnn_amd.grouped_linear(neg(x), neg(w), ptr, neg(b)), plain)
    for f, d in ((lambda t: mpgnn_amd.layer_norm(t, v), dy), (lambda t: mpgnn_amd.grouped_linear(t, w, ptr), dz)):
        leaf = x.clone().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(f(leaf), leaf, neg(d))[0], torch.autograd.grad(f(leaf), leaf, -d)[0])
        assert torch.equal(torch.autograd.grad(f(neg(leaf)), leaf, d)[0], torch.autograd.grad(f(-leaf), leaf, d)[0])
    a, c = x.clone(), neg(x.clone())
    p = [torch.nn.Parameter(x.clone()), torch.nn.Parameter(x.clone())]
    p[0].grad, p[1].grad = a, c
    mpgnn_amd.clip_grad_norm_(p, 1.0)
    assert torch.equal(c, -a) and float(a.abs().max()) < float(x.abs().max())
    with pytest.raises(ValueError):
        mpgnn_amd.clip_by_global_norm([x], 1.0, out=[neg(x.clone())])


@pytest.mark.parametrize("rows", [9, 700])
@pytest.mark.parametrize("e, f", [(-100, 60), (-108, 20), (-116, 40), (-126, 60), (60, -126)], ids=str)
def test_grouped_linear_fp32_small_magnitudes(rows, e, f):
    """fp32 products of operands near the smallest normal numbers: the third (and second) bf16 piece ends at the
    subnormal step 2^-133, so that each operand is off by half of that at most on top of the usual error."""
    g = gen(rows + f)
    x, dy = rnd(g, rows, 96) * 2.0 ** e, rnd(g, rows, 72) * 2.0 ** e
    w = rnd(g, 2, 96, 72) * 2.0 ** f
    off = [0, rows // 3, rows]
    (y, ym), (dx, dxm), (_, _), _ = gl_reference(x, w, None, off, dy)
    xg, wg = x.to(DEV).requires_grad_(True), w.to(DEV)
    got = mpgnn_amd.grouped_linear(xg, wg, torch.tensor(off, device=DEV))
    got.backward(dy.to(DEV))
    ones = torch.ones_like
    (_, ys), (_, dxs), _, _ = gl_reference(ones(x), w, None, off, ones(dy))  # sums of |w|
    (_, yx), (_, dxd), _, _ = gl_reference(x, ones(w), None, off, dy)        # sums of |x|, of |dy|
    lost = 2.0 ** -134
    within(got, y, gl_tol(y, ym, 96, torch.float32) + lost * (ys + yx), "y")
    within(xg.grad, dx, gl_tol(dx, dxm, 72, torch.float32) + lost * (dxs + dxd), "dx")


@pytest.mark.parametrize("dt", TYPES, ids=str)
@pytest.mark.parametrize("groups, rows, bits", [(253, 1000, 64), (254, 9000, 32), (255, 5, 64), (256, 9000, 64),
                                                (257, 3000, 32), (510, 40000, 64), (513, 700, 64), (2700, 8192, 64),
                                                (70001, 50000, 32), (1 << 20, 300000, 64)], ids=str)
def test_grouped_linear_many_groups(groups, rows, bits, dt):
    """Group counts around the ways of the search for a workgroup's tile and far above them: uneven groups, many empty,
    rows before the first and behind the last. A million of them ends as soon as any other call."""
    k, n = 8, 5
    g = gen(groups + rows)
    sizes = torch.bincount(torch.randint(0, groups, (rows - 3,), generator=g) ** 2 // groups, minlength=groups)
    before = 2
    ptr = torch.cat([torch.tensor([before]), before + sizes.cumsum(0)])
    x, w, b, dy = (rnd(g, *s, dtype=dt) for s in ((rows, k), (groups, k, n), (groups, n), (rows, n)))
    of = torch.repeat_interleave(torch.arange(groups), sizes)  # the group of each of the rows that have one
    lo, hi = before, before + len(of)
    xd, wd, dd = x.double()[lo:hi], w.double()[of], dy.double()[lo:hi]

    def rows_of(t):  # zeros for the rows of no group
        out = torch.zeros(rows, t.shape[1], dtype=torch.float64)
        out[lo:hi] = t
        return out

    def sums_of(t):
        return torch.zeros(groups, *t.shape[1:], dtype=torch.float64).index_add_(0, of, t)

    prod = xd[:, :, None] * wd
    bd = b.double()[of]
    xg, wg, bg = (t.to(DEV).requires_grad_(True) for t in (x, w, b))
    y = mpgnn_amd.grouped_linear(xg, wg, ptr.to(DEV, torch.int64 if bits == 64 else torch.int32), bg)
    y.backward(dy.to(DEV))
    within(y, rows_of(prod.sum(1) + bd), gl_tol(rows_of(prod.sum(1) + bd), rows_of(prod.abs().sum(1) + bd.abs()), k, dt), "y")
    back = dd[:, None, :] * wd
    within(xg.grad, rows_of(back.sum(2)), gl_tol(rows_of(back.sum(2)), rows_of(back.abs().sum(2)), n, dt), "dx")
    outer = xd[:, :, None] * dd[:, None, :]
    longest = int(sizes.max())
    dw, dwm = sums_of(outer), sums_of(outer.abs())
    within(wg.grad, dw, gl_tol(dw, dwm, longest, dt), "dw")
    db, dbm = sums_of(dd), sums_of(dd.abs())
    within(bg.grad, db, longest * U * dbm + half(dt) * db.abs() + tiny(dt), "db")


def test_clip_refuses_an_out_with_a_tangent():
    """What is written would keep the tangent of what it held before."""
    from torch.autograd import forward_ad
    x = rnd(gen(94), 6, 8).to(DEV)
    with forward_ad.dual_level():
        o = forward_ad.make_dual(torch.zeros_like(x), torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            mpgnn_amd.clip_by_global_norm([x], 1.0, out=[o])
        assert float(forward_ad.unpack_dual(o).primal.abs().max()) == 0.0
