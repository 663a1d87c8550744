"""Layer norm with its gradients to second order (``ubio_molfm_b200.norm``) against a 64-bit restatement.

Tolerances.  u = 2^-24 is fp32's half step.  Every rounding of the fp32 evaluation changes one of the terms of
the formulas by a relative u; no output has more than L + 40 of them on any path, L = ceil(W / 32) + 5 being
the longest chain of a row sum (32 lanes, then five exchanges) and 40 covering the exponential (2 units), the
divisions and the rest.  The normalised value itself comes from a difference: |d xh| <= (L + 8) u (1 + A)(1 + X)
with A = max|x| r and X = max|xh| of the row, which enters every term at most once through act, act' or act''
(bounded by 1.1, 1.1 and 0.5 in slope).  So every output is within (L + 40) u (1 + A)(1 + X) of the sum of its
terms' magnitudes (``_majorants``), plus half a step of its own type; a column sum in fp32 chains of at most 128
rows adds 160 u of the sum of magnitudes.
"""
import math

import pytest
import torch

U = 2.0 ** -24
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
EPS = 1e-5

SHAPES = [(1, 1), (5, 2), (1, 16), (257, 16), (33, 128), (7, 130), (64, 260), (19, 513), (1100, 96), (5, 1024),
          (3, 1025), (2, 4096), (3, 9001)]


def _act(z, silu):
    if not silu:
        return z, torch.ones_like(z), torch.zeros_like(z)
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s)), s * (1 - s) * (2 + z * (1 - 2 * s))


def reference(x, w, b, silu, g=None, u=None, p=None, q=None):
    """All outputs in 64 bits: y; dx, dw, db; gg, gx, gw, gb."""
    x, w, b = x.double(), w.double(), b.double()
    mean = x.mean(1, keepdim=True)
    r = 1 / ((x - mean).square().mean(1, keepdim=True) + EPS).sqrt()
    xh = (x - mean) * r
    y, d1, d2 = _act(xh * w + b, silu)
    out = dict(y=y)
    if g is None:
        return out
    g = g.double()
    a = g * d1
    h = a * w
    m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    out.update(dx=r * (h - m1 - xh * m2), dw=(a * xh).sum(0), db=a.sum(0))
    if u is None:
        return out
    u, p, q = u.double(), p.double(), q.double()
    c = (u * xh).mean(1, keepdim=True)
    t = r * (u - u.mean(1, keepdim=True) - xh * c)
    v = w * t + p * xh + q
    e = g * d2 * v
    k = e * w + a * p - r * (u * m2 + h * c)
    out.update(gg=d1 * v, gw=(a * t + e * xh).sum(0), gb=e.sum(0),
               gx=r * (k - k.mean(1, keepdim=True) - xh * (k * xh).mean(1, keepdim=True)
                       - xh * (h * t).mean(1, keepdim=True)))
    return out


def _majorants(x, w, b, g, u=None, p=None, q=None):
    """The sums of magnitudes of every output's terms, times the error per unit of them (see above)."""
    x, w, b, g = x.double(), w.double().abs(), b.double().abs(), g.double().abs()
    L = math.ceil(x.shape[1] / 32) + 5
    mean = x.mean(1, keepdim=True)
    r = 1 / ((x - mean).square().mean(1, keepdim=True) + EPS).sqrt()
    xh = ((x - mean) * r).abs()
    A = x.abs().amax(1, keepdim=True) * r
    per = (L + 40) * U * (1 + A) * (1 + xh.amax(1, keepdim=True))
    xh = xh + 1          # |xh| and the unit that a difference's error is measured in
    a = 1.1 * g
    h = a * w
    m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    out = dict(y=1.1 * per * (xh * w + b), dx=per * r * (h + m1 + xh * m2),
               dw=((per + 160 * U) * a * xh).sum(0), db=((per + 160 * U) * a).sum(0))
    if u is None:
        return out
    u, p, q = u.double().abs(), p.double().abs(), q.double().abs()
    c = (u * xh).mean(1, keepdim=True)
    t = r * (u + u.mean(1, keepdim=True) + xh * c)
    v = w * t + p * xh + q
    e = 0.5 * g * v
    k = e * w + a * p + r * (u * m2 + h * c)
    out.update(gg=per * 1.1 * v, gw=((per + 160 * U) * (a * t + e * xh)).sum(0), gb=((per + 160 * U) * e).sum(0),
               gx=per * r * (k + k.mean(1, keepdim=True) + xh * ((k * xh).mean(1, keepdim=True)
                                                                 + (h * t).mean(1, keepdim=True))))
    return out


def _close(got, ref, major, what):
    got64 = got.detach().double()
    tol = major + HALF[got.dtype] * (ref.abs() + major) + TINY[got.dtype]
    bad = ~((got64 - ref).abs() <= tol)
    assert not bool(bad.any()), (what, float((got64 - ref).abs().max()), float(tol.max()), int(bad.sum()))


def _inputs(rows, width, dtype, seed=0, device=DEV):
    gen = torch.Generator().manual_seed(1000 * seed + rows * 7 + width)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x = (r(rows, width) * (0.3 + torch.rand(rows, 1, generator=gen)) + r(rows, 1)).to(dtype)
    g, u = (0.5 * r(rows, width)).to(dtype), r(rows, width).to(dtype)
    w, b, p, q = 1 + 0.3 * r(width), 0.3 * r(width), r(width), r(width)
    return [t.to(device) for t in (x, w, b, g, u, p, q)]


def _run(x, w, b, silu, g, second=None):
    from ubio_molfm_b200.norm import layer_norm

    x, w, b, g = (t.detach().requires_grad_(True) for t in (x, w, b, g))
    y = layer_norm(x, w, b, EPS, "silu" if silu else None)
    if second is None:
        dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
        return dict(y=y, dx=dx, dw=dw, db=db)
    u, p, q = second
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g, create_graph=True)
    gg, gx, gw, gb = torch.autograd.grad((dx, dw, db), (g, x, w, b), (u, p, q))
    return dict(y=y, dx=dx, dw=dw, db=db, gg=gg, gx=gx, gw=gw, gb=gb)


# ------------------------------------------------------------------------------------------------
# the formulas themselves (CPU, 64 bits): against autograd and against differences
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("silu", [False, True])
def test_reference_formulas_equal_autograd_and_differences(silu):
    x, w, b, g, u, p, q = (t.double() for t in _inputs(6, 12, torch.float32, device="cpu"))
    ref = reference(x, w, b, silu, g, u, p, q)
    xs, ws, bs, gs = (t.clone().requires_grad_(True) for t in (x, w, b, g))
    y = torch.nn.functional.layer_norm(xs, (12,), ws, bs, EPS)
    y = torch.nn.functional.silu(y) if silu else y
    first = torch.autograd.grad(y, (xs, ws, bs), gs, create_graph=True)
    second = torch.autograd.grad(first, (gs, xs, ws, bs), (u, p, q), allow_unused=True)
    for name, t in zip(("y", "dx", "dw", "db", "gg", "gx", "gw", "gb"), (y, *first, *second)):
        t = torch.zeros_like(ref[name]) if t is None else t.detach()
        assert float((t - ref[name]).abs().max()) <= 1e-12 * max(1.0, float(t.abs().max())), name
    # central differences along a direction: error h^2 (third derivatives of order 10) + 1e-16 / h
    h = 1e-5
    d = [torch.randn(t.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
         for i, t in enumerate((x, w, b, g))]

    def energy(s):
        return float((reference(x + s * d[0], w + s * d[1], b + s * d[2], silu)["y"] * g).sum())

    def paired(s):
        o = reference(x + s * d[0], w + s * d[1], b + s * d[2], silu, g + s * d[3])
        return float((o["dx"] * u).sum() + (o["dw"] * p).sum() + (o["db"] * q).sum())

    slope = float((ref["dx"] * d[0]).sum() + (ref["dw"] * d[1]).sum() + (ref["db"] * d[2]).sum())
    assert abs((energy(h) - energy(-h)) / (2 * h) - slope) <= 1e-6 * max(1.0, abs(slope))
    slope = float((ref["gx"] * d[0]).sum() + (ref["gw"] * d[1]).sum() + (ref["gb"] * d[2]).sum()
                  + (ref["gg"] * d[3]).sum())
    assert abs((paired(h) - paired(-h)) / (2 * h) - slope) <= 1e-6 * max(1.0, abs(slope))


def test_refusals():
    from ubio_molfm_b200.norm import layer_norm

    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(torch.zeros(3, 4))


def test_c_abi_refuses_bad_arguments():
    """Checked on the host before any device work: the addresses are never read."""
    import ctypes

    from ubio_molfm_b200 import _lib

    lib = _lib.load()
    d = ctypes.c_void_p(4096)
    fwd, bwd, bwd2 = lib.e2a_layer_norm_fwd, lib.e2a_layer_norm_bwd, lib.e2a_layer_norm_bwd2

    def ok(rows=4, W=8, ldx=8, dtype=0, act=0, x=d):
        return fwd(x, ldx, dtype, None, None, rows, W, EPS, act, d, d, d, None)

    assert ok(rows=0) == 0
    assert ok(rows=-1) == 1 and ok(W=0) == 1 and ok(ldx=-1) == 1 and ok(act=2) == 1 and ok(x=None) == 1
    assert ok(dtype=3) == 1 and ok(dtype=3, rows=0) == 1
    assert lib.e2a_layer_norm_bwd_workspace_bytes(0, 8) == 0
    need = lib.e2a_layer_norm_bwd_workspace_bytes(4, 8)
    assert need >= 2 * 8 * 4
    args = (d, 8, d, 8, 0, None, None, d, d, 4, 8, 0, d, d, d)
    assert bwd(*args, None, 0, None) == 3 and bwd(*args, d, need - 1, None) == 3
    assert bwd(None, *args[1:], d, need, None) == 1
    need2 = lib.e2a_layer_norm_bwd2_workspace_bytes(4, 8)
    args2 = (d, 8, d, 8, d, 8, 0, None, None, d, d, None, None, 4, 8, 0, d, d, d, d)
    assert bwd2(*args2, d, need2 - 1, None) == 3
    assert bwd2(*args2[:4], None, *args2[5:], d, need2, None) == 1


# ------------------------------------------------------------------------------------------------
# the kernels
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_layer_norm_and_gradients_to_second_order(rows, width, dtype, silu):
    x, w, b, g, u, p, q = _inputs(rows, width, dtype)
    ref, major = reference(x, w, b, silu, g, u, p, q), _majorants(x, w, b, g, u, p, q)
    first = _run(x, w, b, silu, g)
    for k, t in first.items():
        assert t.dtype == (dtype if k in ("y", "dx") else torch.float32) and t.is_contiguous()
        _close(t, ref[k], major[k], k)
    for k, t in _run(x, w, b, silu, g, (u, p, q)).items():
        _close(t, ref[k], major[k], k)
        if k in first:
            assert torch.equal(t, first[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("rows,width,dtype", [
    (40000, 16, torch.float32), (20011, 64, torch.float32), (70001, 128, torch.float32), (9001, 512, torch.float32),
    (3001, 771, torch.float32), (600, 8200, torch.float32), (150001, 3, torch.float16), (50001, 25, torch.bfloat16),
    (50003, 26, torch.float16), (40001, 77, torch.bfloat16), (30007, 131, torch.float16), (20001, 250, torch.bfloat16),
    (20011, 300, torch.float16), (9001, 771, torch.bfloat16), (5003, 1203, torch.float16), (3001, 3001, torch.bfloat16),
    (1201, 4089, torch.float16), (1201, 4091, torch.bfloat16)])
def test_many_rows(rows, width, dtype):
    """More rows than the device holds at once, past the fp32 chains' length, at every way of reading them."""
    x, w, b, g, u, p, q = _inputs(rows, width, dtype)
    ref, major = reference(x, w, b, True, g, u, p, q), _majorants(x, w, b, g, u, p, q)
    got = _run(x, w, b, True, g, (u, p, q))
    for k, t in got.items():
        _close(t, ref[k], major[k], k)
    again = _run(x, w, b, True, g, (u, p, q))
    for k in got:
        assert torch.equal(got[k], again[k]), k      # the same bits every time


@pytest.mark.gpu
@pytest.mark.parametrize("width", [12, 128, 520])
@pytest.mark.parametrize("layout", ["row stride", "offset", "transposed", "repeated rows", "3d", "1d"])
def test_layouts(layout, width):
    from ubio_molfm_b200.norm import layer_norm

    x, w, b, g, u, p, q = _inputs(24, width, torch.float32)
    if layout == "row stride":
        x = torch.cat([x, 7 * x], 1)[:, :width]
    elif layout == "offset":
        big = torch.zeros(24, width + 5, device=DEV)
        big[:, 1:width + 1] = x
        x = big[:, 1:width + 1]
    elif layout == "transposed":
        x = x.t().contiguous().t()
    elif layout == "repeated rows":
        x = x[:1].expand(24, width)
    assert x.shape == (24, width)
    ref, major = reference(x, w, b, True, g, u, p, q), _majorants(x, w, b, g, u, p, q)
    shape = {"3d": (2, 12, width), "1d": None}.get(layout, (24, width))
    if shape is None:
        x, g, u = x[0], g[0], u[0]
        ref = reference(x[None], w, b, True, g[None], u[None], p, q)
        major = _majorants(x[None], w, b, g[None], u[None], p, q)
        shape = (width,)
    xi = (x if layout not in ("3d",) else x.reshape(shape)).detach().requires_grad_(True)
    wi, bi, gi = (t.detach().clone().requires_grad_(True) for t in (w, b, g.reshape(shape)))
    y = layer_norm(xi, wi, bi, EPS, "silu")
    assert y.shape == shape
    dx, dw, db = torch.autograd.grad(y, (xi, wi, bi), gi, create_graph=True)
    gg, gx, gw, gb = torch.autograd.grad((dx, dw, db), (gi, xi, wi, bi), (u.reshape(shape), p, q))
    for k, t in dict(y=y, dx=dx, dw=dw, db=db, gg=gg, gx=gx, gw=gw, gb=gb).items():
        _close(t.reshape(ref[k].shape), ref[k], major[k], k)


@pytest.mark.gpu
def test_upstream_gradients_that_repeat():
    """A cotangent that autograd hands over as an expanded scalar (the gradient of a sum)."""
    from ubio_molfm_b200.norm import layer_norm

    x, w, b, g, u, p, q = _inputs(50, 96, torch.float32)
    ones = torch.ones_like(x)
    ref, major = reference(x, w, b, True, ones), _majorants(x, w, b, ones)
    xi, wi, bi = (t.detach().clone().requires_grad_(True) for t in (x, w, b))
    layer_norm(xi, wi, bi, EPS, "silu").sum().backward()
    for k, t in dict(dx=xi.grad, dw=wi.grad, db=bi.grad).items():
        _close(t, ref[k], major[k], k)


@pytest.mark.gpu
@pytest.mark.parametrize("affine", ["none", "weight", "bias", "frozen", "half"])
def test_affine_forms(affine):
    from ubio_molfm_b200.norm import layer_norm

    x, w, b, g, u, p, q = _inputs(37, 160, torch.bfloat16 if affine == "half" else torch.float32)
    if affine == "half":
        w, b = w.bfloat16(), b.bfloat16()
    one, zero = torch.ones(160, device=DEV), torch.zeros(160, device=DEV)
    rw, rb = (one if affine in ("none", "bias") else w), (zero if affine in ("none", "weight") else b)
    ref, major = reference(x, rw, rb, True, g, u, 0 * p, 0 * q), _majorants(x, rw, rb, g, u, 0 * p, 0 * q)
    learn = affine != "frozen"
    xi, gi = x.clone().requires_grad_(True), g.clone().requires_grad_(True)
    wi = None if affine in ("none", "bias") else w.clone().requires_grad_(learn)
    bi = None if affine in ("none", "weight") else b.clone().requires_grad_(learn)
    y = layer_norm(xi, wi, bi, EPS, "silu")
    _close(y, ref["y"], major["y"], "y")
    leaves = [t for t in (xi, wi, bi) if t is not None and t.requires_grad]
    names = [n for n, t in (("x", xi), ("w", wi), ("b", bi)) if t is not None and t.requires_grad]
    for n, t, leaf in zip(names, torch.autograd.grad(y, leaves, gi, retain_graph=True), leaves):
        assert t.dtype == leaf.dtype
        _close(t, ref["d" + n], major["d" + n], "d" + n)
    (dx,) = torch.autograd.grad(y, xi, gi, create_graph=True)
    for n, t in zip(["g"] + names, torch.autograd.grad(dx, [gi] + leaves, u)):
        _close(t, ref["g" + n], major["g" + n], "g" + n)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [96, 77, 9001])
def test_column_gradients_alone(width):
    """An input without gradient (the first layer's): only dw and db are formed, and they are the same."""
    from ubio_molfm_b200.norm import layer_norm

    x, w, b, g, u, p, q = _inputs(70, width, torch.float32)
    want = _run(x, w, b, True, g)
    wi, bi = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    layer_norm(x, wi, bi, EPS, "silu").backward(g)
    assert torch.equal(wi.grad, want["dw"]) and torch.equal(bi.grad, want["db"])
    (db,) = torch.autograd.grad(layer_norm(x, None, bi, EPS), bi, g)
    ref, major = reference(x, torch.ones_like(w), b, False, g), _majorants(x, torch.ones_like(w), b, g)
    _close(db, ref["db"], major["db"], "db")


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["w", "b"])
def test_second_order_of_one_column_gradient(which):
    """Only dw (or db) is differentiated on: the cotangent of dx is absent."""
    from ubio_molfm_b200.norm import layer_norm

    x, w, b, g, u, p, q = _inputs(20, 48, torch.float32)
    z = torch.zeros_like
    ref = reference(x, w, b, True, g, z(u), p if which == "w" else z(p), q if which == "b" else z(q))
    major = _majorants(x, w, b, g, z(u), p if which == "w" else z(p), q if which == "b" else z(q))
    xi, wi, bi, gi = (t.clone().requires_grad_(True) for t in (x, w, b, g))
    y = layer_norm(xi, wi, bi, EPS, "silu")
    (d,) = torch.autograd.grad(y, wi if which == "w" else bi, gi, create_graph=True)
    for n, t in zip("gxwb", torch.autograd.grad(d, (gi, xi, wi, bi), p if which == "w" else q)):
        _close(t, ref["g" + n], major["g" + n], "g" + n)


@pytest.mark.gpu
def test_rows_do_not_see_each_other():
    """A row of NaN or infinities leaves the other rows' outputs as they were; its own become NaN."""
    x, w, b, g, u, p, q = _inputs(64, 128, torch.float32)
    clean = _run(x, w, b, True, g, (u, p, q))
    x = x.clone()
    x[5, 3], x[40, 100], x[41] = float("nan"), float("inf"), float("-inf")
    got = _run(x, w, b, True, g, (u, p, q))
    hit = torch.zeros(64, dtype=torch.bool, device=DEV)
    hit[[5, 40, 41]] = True
    for k in ("y", "dx", "gg", "gx"):
        assert torch.equal(got[k][~hit], clean[k][~hit]), k
        assert bool(got[k][hit].isnan().all()), k


@pytest.mark.gpu
def test_constant_rows_and_no_rows():
    from ubio_molfm_b200.norm import layer_norm

    w, b = torch.full((32,), 2.0, device=DEV), torch.full((32,), 0.5, device=DEV)
    y = layer_norm(torch.full((3, 32), 7.0, device=DEV), w, b, EPS)
    assert bool((y == 0.5).all())             # variance 0: xh is 0 exactly
    for width in (3, 12, 100, 1000, 5000):    # 7 k is exact, and so is the mean
        y = layer_norm(torch.full((2, width), 7.0, device=DEV), bias=torch.full((width,), 0.5, device=DEV))
        assert bool((y == 0.5).all()), width
    x = torch.zeros(0, 32, device=DEV, requires_grad=True)
    w.requires_grad_(True)
    y = layer_norm(x, w, b, EPS)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 32) and dx.shape == (0, 32) and bool((dw == 0).all())


@pytest.mark.gpu
def test_gpu_refusals():
    from ubio_molfm_b200.norm import layer_norm

    x = torch.zeros(3, 8, device=DEV)
    with pytest.raises(TypeError):
        layer_norm(x.double())
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(7, device=DEV))
    with pytest.raises(TypeError):
        layer_norm(x, torch.ones(8, device=DEV, dtype=torch.float16))
    with pytest.raises(ValueError):
        layer_norm(x, activation="gelu")
    with pytest.raises(ValueError):
        layer_norm(torch.zeros(3, 0, device=DEV))
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(8))
    xi = torch.randn(3, 8, device=DEV, requires_grad=True)
    y = layer_norm(xi, activation="silu")
    (d1,) = torch.autograd.grad(y.square().sum(), xi, create_graph=True)
    with pytest.raises(RuntimeError, match="third"):
        torch.autograd.grad(d1.square().sum(), xi, create_graph=True)


@pytest.mark.gpu
def test_other_stream_and_captured_graph():
    from ubio_molfm_b200.norm import layer_norm

    x, w, b, g, u, p, q = _inputs(300, 128, torch.float32)
    want = _run(x, w, b, True, g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(x, w, b, True, g)
    torch.cuda.current_stream().wait_stream(s)
    for k in want:
        assert torch.equal(want[k], got[k]), k
    del got
    # captured once, replayed on other values
    xi, wi, bi = x.clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        torch.autograd.grad(layer_norm(xi, wi, bi, EPS, "silu"), (xi, wi, bi), g)
    torch.cuda.current_stream().wait_stream(s)
    with torch.cuda.graph(graph):
        y = layer_norm(xi, wi, bi, EPS, "silu")
        grads = torch.autograd.grad(y, (xi, wi, bi), g)
    for seed in (3, 4):
        x2 = _inputs(300, 128, torch.float32, seed)[0]
        with torch.no_grad():
            xi.copy_(x2)
        graph.replay()
        want = _run(x2, w, b, True, g)
        for t, k in zip((y, *grads), ("y", "dx", "dw", "db")):
            assert torch.equal(t, want[k]), k


@pytest.mark.gpu
def test_offsets_past_32_bits():
    from ubio_molfm_b200.norm import layer_norm

    rows, width = (1 << 22) + 3, 520            # 2.2e9 values
    x = torch.randn(1, width, device=DEV).bfloat16()
    y = layer_norm(x.expand(rows, width))
    assert torch.equal(y[-1], layer_norm(x)[0]) and torch.equal(y[rows // 2], y[0])
    g = y[:1].expand(rows, width)
    xi = x.expand(rows, width).detach().requires_grad_(True)
    (dx,) = torch.autograd.grad(layer_norm(xi), xi, g)
    assert torch.equal(dx[-1], dx[0]) and torch.equal(dx[rows // 2 + 1], dx[0])
