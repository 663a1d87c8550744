"""Layer norm of rows away from zero, constant or nearly so, of extreme values, and wider than a warp's registers hold
(``ubio_molfm_b200.norm``), against a 64-bit restatement.

Tolerances.  u = 2^-24.  The forward takes every value's difference to the row's first one, which is exact for values
within a factor of two of each other and otherwise off by u of the difference; mean, variance and what follows are
sums and products of those differences, in chains of at most L = 40 roundings whatever the width (16 values a thread
in pairs, 5 exchanges, 16 warps; loops over wider rows add up in 64 bits).  So xh is off by at most
(L + 40) u (1 + X), X = max|xh|, if the first value is not itself far out: |x_0 - mean| r <= X covers that, too.  No term
grows with |x|.  The backward takes x - mean with the mean rounded to fp32: at most u |mean| r more in xh, 0 where the
mean is a constant row's value.  Outputs then as in ``test_layer_norm``: each is within ``per`` = (L + 40) u (1 + X)
+ u A' (1 + X), A' = |mean| r or 0, of the sum of its terms' magnitudes, and half a step of its type."""
import pytest
import torch
from test_layer_norm import DEV, EPS, HALF, TINY, U, _inputs, _majorants, _run, reference

L = 40


def _per(x, exact_mean):
    """This file's error per unit of magnitude, a row; ``exact_mean``: the rows whose mean is one of their values."""
    x = x.double()
    mean = x.mean(1, keepdim=True)
    r = 1 / ((x - mean).square().mean(1, keepdim=True) + EPS).sqrt()
    X = ((x - mean) * r).abs().amax(1, keepdim=True)
    return (L + 40) * U * (1 + X) + torch.where(exact_mean, 0 * r, U * mean.abs() * r * (1 + X))


def _majorants_with(per, x, w, b, g, u, p, q):
    """The sums of magnitudes of every output's terms times ``per``."""
    x, w, b, g, u, p, q = x.double(), *(t.double().abs() for t in (w, b, g, u, p, q))
    mean = x.mean(1, keepdim=True)
    r = 1 / ((x - mean).square().mean(1, keepdim=True) + EPS).sqrt()
    xh = ((x - mean) * r).abs() + 1          # and the unit that a difference's error is measured in
    a = 1.1 * g
    h = a * w
    m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
    c = (u * xh).mean(1, keepdim=True)
    t = r * (u + u.mean(1, keepdim=True) + xh * c)
    v = w * t + p * xh + q
    e = 0.5 * g * v
    k = e * w + a * p + r * (u * m2 + h * c)
    cols = per + 160 * U
    return dict(y=1.1 * per * (xh * w + b), dx=per * r * (h + m1 + xh * m2), dw=(cols * a * xh).sum(0),
                db=(cols * a).sum(0), gg=per * 1.1 * v, gw=(cols * (a * t + e * xh)).sum(0), gb=(cols * e).sum(0),
                gx=per * r * (k + k.mean(1, keepdim=True)
                              + xh * ((k * xh).mean(1, keepdim=True) + (h * t).mean(1, keepdim=True))))


def _close(got, ref, major, what):
    got64 = got.detach().double()
    tol = major + HALF[got.dtype] * (ref.abs() + major) + TINY[got.dtype]
    off = (got64 - ref).abs()
    bad = ~(off <= tol)
    assert not bool(bad.any()), (what, float(off[bad].max()), float((off / tol).max()), int(bad.sum()))


def _rows(width, dtype, seed):
    """Constant rows whose values are no short binary fractions, nearly constant ones, an ordinary row far from zero."""
    gen = torch.Generator().manual_seed(seed + width)
    z = torch.randn(8, width, generator=gen, dtype=torch.float64)
    base = torch.tensor([0.1, 100.3, 1000.1, -77.7, 3e7, 100.3, 1000.1, -30.0], dtype=torch.float64)[:, None]
    spread = torch.tensor([0, 0, 0, 0, 0, 0.01, 0.3, 1.0], dtype=torch.float64)[:, None]
    x = base + spread * z
    if dtype == torch.float16:
        x[4] = 2049.0
    x = x.to(dtype).to(DEV)
    constant = (x == x[:, :1]).all(1, keepdim=True)
    return x, constant


WIDTHS = [3, 12, 100, 512, 1000, 1001, 4096, 5000, 6001, 8192, 9001]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("width", WIDTHS + [100_003, 1 << 20])
def test_constant_and_nearly_constant_rows(width, dtype):
    """A constant row's outputs are the bias's, exactly."""
    from ubio_molfm_b200.norm import layer_norm

    x, constant = _rows(width, dtype, 1)
    w, b = _inputs(1, width, torch.float32)[1:3]
    y = layer_norm(x, w, b, EPS)
    c = constant.squeeze(1)
    assert int(c.sum()) >= 5 and torch.equal(y[c], b.to(dtype).expand(int(c.sum()), width))
    ref = reference(x, w, b, False)["y"]
    every = torch.ones_like(constant)            # no row's error may grow with its mean here
    xh = reference(x, torch.ones_like(w), torch.zeros_like(b), False)["y"].abs()
    _close(y, ref, _per(x, every) * (w.abs() * (1 + xh) + b.abs()), "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("width", WIDTHS)
def test_gradients_of_constant_and_nearly_constant_rows(width, dtype):
    x, constant = _rows(width, dtype, 2)
    _, w, b, g, u, p, q = _inputs(8, width, dtype)
    ref = reference(x, w, b, True, g, u, p, q)
    major = _majorants_with(_per(x, constant), x, w, b, g, u, p, q)
    for k, t in _run(x, w, b, True, g, (u, p, q)).items():
        _close(t, ref[k], major[k], k)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 3, 12, 100, 128, 1000, 6001, 9001])
@pytest.mark.parametrize("value", [2e36, 1e38, -3.4028234663852886e38])
def test_rows_of_one_extreme_value(width, value):
    """The type's lowest value as a mask leaves it, and others whose sum or product with 1 / sqrt(eps) passes fp32's
    range: xh is 0, y the activated bias, and the gradients are those of xh = 0."""
    _, w, b, g, u, p, q = _inputs(4, width, torch.float32)
    x = torch.full((4, width), value, device=DEV)
    ref = reference(torch.zeros_like(x), w, b, True, g, u, p, q)
    zero = torch.zeros_like(x)
    major = _majorants_with(_per(zero, zero[:, :1] == 0), zero, w, b, g, u, p, q)
    for k, t in _run(x, w, b, True, g, (u, p, q)).items():
        _close(t, ref[k], major[k], k)
    y = _run(x, w, b, False, g)["y"]
    assert torch.equal(y, b.expand(4, width))
