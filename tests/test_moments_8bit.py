"""The 8-bit moments of ``ubio_molfm_b200.optim.AdamW``: the format and its roundings as stated, by value.

256 values share the power of two of the largest magnitude.  Over it a value is a small float of 4 exponent and 3
(first moment, with a sign) or 4 (square root of the second moment) fraction bits; it is rounded up where its part
below the last place plus an offset from an additive sequence over (element, step) reaches one, never past the largest
code, and a root over 0 stays over 0.  The restatement below has no bit patterns in it; the kernel's codes and scales
have to equal it bit for bit, since the moments' fp32 operations are each rounded once in a stated order."""
import math

import numpy as np
import pytest
import torch

DEV = "cuda"
F = np.float32
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# 32-bit fractions by which an offset moves from element to element and from step to step, by fraction bits
STEPS = {3: (0xDB4F0B91, 0xBBE05633), 4: (0xA0F2EC75, 0x89E18285)}


def offsets(n, t, fraction):
    """The offsets in [0, 1) of elements 0..n-1 at step t, in the places that the format's fp32 value has left."""
    a, b = STEPS[fraction]
    whole = [(i * a + t * b) % 2 ** 32 for i in range(n)]
    return np.array([w // 2 ** (9 + fraction) for w in whole]) / 2.0 ** (23 - fraction)


def pack(x, offset, fraction):
    """Codes and block scales of fp32 values ``x``."""
    n = x.size
    mag = np.abs(x.astype(np.float64))
    blocks = np.zeros(-(-n // 256) * 256)
    blocks[:n] = mag
    top = blocks.reshape(-1, 256).max(1)
    e = np.clip(np.floor(np.log2(np.maximum(top, 1e-300))).astype(int), -100, 126)
    y = mag / np.exp2(np.repeat(e, 256)[:n].astype(np.float64))
    y = np.where(y < 2.0 ** -14, np.round(y * 2.0 ** 37) / 2.0 ** 37, y)     # what is left of fp32 down there
    with np.errstate(divide="ignore"):
        k = np.maximum(np.floor(np.log2(y)), -14)
    places = y / np.exp2(k - fraction)
    low = np.floor(places)
    low = low + ((places - low) + offset >= 1)
    code = np.minimum((low + (k + 14) * 2 ** fraction).astype(int), 2 ** (4 + fraction) - 1)
    if fraction == 4:
        code = np.maximum(code, x > 0)
    else:
        code = code + 128 * (x < 0)
    return code.astype(np.uint8), (e + 127).astype(np.uint8)


def unpack(code, scale, fraction):
    mag = (code & 127 if fraction == 3 else code).astype(np.int64)
    exp, frac = mag >> fraction, mag & (2 ** fraction - 1)
    y = np.where(exp == 0, frac * 2.0 ** (-14 - fraction), (1 + frac * 2.0 ** -fraction) * np.exp2(exp - 15.0))
    y = y * np.exp2(np.repeat(scale.astype(np.float64), 256)[:code.size] - 127)
    if fraction == 3:
        y = np.where(code > 127, -y, y)
    return y.astype(F)


def step32(p, g, m, v, t, lr, b1, b2, eps, wd, coef=None):
    """One step in float32, every operation rounded on its own; all arrays float32."""
    size, root = F(lr / (1 - b1 ** t)), F(1 / math.sqrt(1 - b2 ** t))
    if coef is not None:
        g = g * coef
    m = m * F(b1) + g * F(1 - b1)
    v = v * F(b2) + (g * g) * F(1 - b2)
    with np.errstate(all="ignore"):
        return p * F(1 - lr * wd) - m / (np.sqrt(v) * root + F(eps)) * size, m, v


# ------------------------------------------------------------------------------------------------
# the format
# ------------------------------------------------------------------------------------------------
def _sequence_bound(step):
    """How far the share of t < T with frac(t step / 2^32 + c) above a threshold can be from its measure, times T: at
    most the sum of the partial quotients of the continued fraction up to the first denominator over T, and one."""
    T, a, b, total, q0, q1 = 4096, 2 ** 32, step, 1, 0, 1
    while b and q1 <= T:
        k = a // b
        total += k
        a, b, q0, q1 = b, a % b, q1, k * q1 + q0
    return T, total


@pytest.mark.parametrize("fraction", [3, 4])
def test_a_fixed_value_is_held_within_a_place_and_right_in_the_mean(fraction):
    """But for what lies over the largest code, which stays there.  The offsets have 23 - fraction bits, which moves
    a threshold by at most 2^-19 of a place."""
    x = np.exp(np.random.default_rng(0).uniform(-9, 0, 256)).astype(F)
    x[0], x[1] = 1.75, 1.97                     # the block's power of two, and a value over either largest code
    T, total = _sequence_bound(STEPS[fraction][1])
    place = np.exp2(np.maximum(np.floor(np.log2(x.astype(np.float64))), -14) - fraction)
    held = np.zeros(256)
    for t in range(T):
        y = unpack(*pack(x, offsets(256, t, fraction), fraction), fraction).astype(np.float64)
        assert (np.abs(y - x) <= place).all()
        held += y
    far = np.abs(held / T - x)
    assert (far[2:] <= (total / T + 2.0 ** -19) * place[2:]).all() and far[0] == 0
    assert held[1] / T == 2 - 2.0 ** -fraction


def test_corner_values():
    x = np.zeros(512, F)
    x[3], x[300], x[301] = 1e-20, 5.0, -1e-30
    code, scale = pack(x, np.full(512, 0.999), 3)
    assert scale[1] == 129 and code[301] & 127 <= 1 and (code[:3] == 0).all()
    assert abs(unpack(code, scale, 3)[3] - 1e-20) <= 1e-20 / 8
    s, sc = pack(np.abs(x), np.zeros(512), 4)
    assert s[301] == 1 and unpack(s, sc, 4)[301] == F(4 * 2.0 ** -18)    # over 0 stays over 0
    assert (unpack(*pack(np.zeros(256, F), np.full(256, 0.999), 3), 3) == 0).all()
    # rounding up does not pass the largest code, whatever the offset
    for fraction in (3, 4):
        code, scale = pack(np.full(256, 1.999, F), np.full(256, 0.999), fraction)
        assert (code == 2 ** (4 + fraction) - 1).all() and (scale == 127).all()


@pytest.mark.parametrize("kind", ["random", "constant"])
def test_what_is_held_over_4000_steps(kind):
    """What the kernel's comment and the optimiser's documentation say of the format, on 16 blocks: with random
    gradients of differing size the held sqrt(v) is 1.4% low in the mean (0.5% is five standard errors of 4,096 values
    with a spread of 10%, of which those of a block are half dependent) and a block's largest value about 40%; with
    gradients that never change a block stays where its largest value first meets the largest code, at 1/8 to 1/4.

    The latter: from 31/16 to 2 a root grows by 32/31 in one step, 0.999 + 0.001 (g / s)^2 >= (32/31)^2, only while
    s <= 0.1225 g.  So it stays at 0.1225 to 0.245 of g; the exact root has come to (1 - 0.999^4000)^(1/2) = 0.9908 of g,
    hence 0.1236 to 0.2473 of that.  The block's other values, up to 1/16 smaller here, grow to the same code."""
    n, T, b2 = 4096, 4000, 0.999
    rng = np.random.default_rng(5)
    size = np.exp(rng.normal(0, 1, n)) if kind == "random" else np.linspace(0.5, 1, n)
    v, exact, held = np.zeros(n, F), np.zeros(n), None
    a, b = STEPS[4]
    index = np.arange(n, dtype=np.uint64) * np.uint64(a)
    for t in range(1, T + 1):
        g = (size * (rng.normal(size=n) if kind == "random" else 1)).astype(F)
        v = v * F(b2) + g * g * F(1 - b2)
        exact = exact * b2 + (1 - b2) * g.astype(np.float64) ** 2
        offset = ((index + np.uint64(t * b)) & np.uint64(2 ** 32 - 1)) >> np.uint64(13)
        held = unpack(*pack(np.sqrt(v), offset / 2.0 ** 19, 4), 4)
        v = held * held
    ratio = held / np.sqrt(exact)
    top = np.sqrt(exact).reshape(-1, 256).argmax(1)
    largest = ratio.reshape(-1, 256)[np.arange(n // 256), top]
    if kind == "random":
        assert abs(ratio.mean() - 0.986) <= 0.01 and ratio.std() <= 0.12
        assert 0.4 <= largest.mean() <= 0.8
    else:
        assert 0.1236 <= largest.min() and largest.max() <= 0.2473
        assert ratio.max() <= 0.2473 * 17 / 16


# ------------------------------------------------------------------------------------------------
# the kernel
# ------------------------------------------------------------------------------------------------
def _np(t):
    return t.detach().float().cpu().numpy()


def _grad(n, dtype, seed):
    gen = torch.Generator().manual_seed(104729 + seed)
    return (10.0 ** ((seed % 5) - 3) * torch.randn(n, generator=gen)).to(dtype)


def _same_p(got, before, want, dtype):
    """The update is within 16 u of its terms (reciprocals and roots of one or two units), and one step of the
    parameter's type where that is narrower."""
    up = np.abs(want.astype(np.float64) - before) + 0.2 * np.abs(before)
    tol = 16 * U * (np.abs(before) + up) + 1e-44
    if dtype != torch.float32:
        tol += 2 * HALF[dtype] * np.abs(want) + (2.0 ** -24 if dtype == torch.float16 else 0)
    return bool((np.abs(got.astype(np.float64) - want) <= tol).all())


def _check_state(st, m, v, t):
    """The held codes and scales of one tensor are those of moments ``m`` and ``v``; returns what they stand for."""
    n = m.size
    cm, sm = pack(m, offsets(n, t, 3), 3)
    cv, sv = pack(np.sqrt(v), offsets(n, t, 4), 4)
    for name, want in (("exp_avg", cm), ("exp_avg_scale", sm), ("exp_avg_sq", cv), ("exp_avg_sq_scale", sv)):
        got = st[name].cpu().numpy()
        assert np.array_equal(got, want), (t, name, int((got != want).sum()))
    s = unpack(cv, sv, 4)
    return unpack(cm, sm, 3), s * s


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_codes_and_scales_bit_for_bit(dtype, clip):
    from ubio_molfm_b200.optim import AdamW

    sizes = [1, 255, 256, 257, 0, 1000, 4099, 40001]
    lr, b1, b2, eps, wd = 3e-3, 0.9, 0.99, 1e-8, 0.05
    gen = torch.Generator().manual_seed(3)
    ps = [torch.nn.Parameter((0.1 * torch.randn(n, generator=gen)).to(dtype).to(DEV)) for n in sizes]
    opt = AdamW(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=8, max_grad_norm=clip)
    ref = [dict(p=_np(p), m=np.zeros(p.numel(), F), v=np.zeros(p.numel(), F)) for p in ps]
    for t in range(1, 6):
        for k, p in enumerate(ps):
            p.grad = _grad(p.numel(), dtype, 29 * t + k).to(DEV)
        opt.step()
        gs = [_np(p.grad) for p in ps]
        coef = None
        if clip is not None:
            norm = F(math.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in gs)))
            assert float(opt.last_grad_norm) == float(norm)
            coef = np.minimum(F(clip) / (norm + F(1e-6)), F(1))
        for p, r, g in zip(ps, ref, gs):
            new, m, v = step32(r["p"], g, r["m"], r["v"], t, lr, b1, b2, eps, wd, coef)
            st = opt.state[p]
            assert int(st["step"]) == t and _same_p(_np(p), r["p"], new, dtype)
            r["p"] = _np(p)
            if p.numel():
                r["m"], r["v"] = _check_state(st, m, v, t)
    m, v = opt.moments()
    for k, r in enumerate(ref):
        o, n = opt._group_state(0).offset[k], ps[k].numel()
        end = -(-n // 256) * 256
        assert np.array_equal(_np(m[o:o + n]), r["m"]) and np.array_equal(_np(v[o:o + n]), r["v"])
        assert not bool(m[o + n:o + end].any()) and not bool(v[o + n:o + end].any())     # nothing between tensors


@pytest.mark.gpu
def test_extreme_magnitudes_and_the_largest_code():
    """Squares near fp32's largest, moments below 2^-100, one value among zeros, and moments between the largest
    code and the next power of two, in whole blocks and in one that the tensor's end cuts short."""
    from ubio_molfm_b200.optim import AdamW

    n = 5 * 256 + 100
    g = np.zeros(n, F)
    rng = np.random.default_rng(2)
    g[:256] = np.linspace(-3e18, 3e18, 256)
    g[256:512] = 1e-37 * rng.normal(size=256)
    g[700] = 1.0
    g[768:] = rng.choice([-1, 1], n - 768) * rng.uniform(1.9, 2.0, n - 768) / F(0.1)
    g[1024:] *= F(math.sqrt(10.0))               # sqrt(0.001) g between 1.9 and 2, too
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    p.grad = torch.from_numpy(g).to(DEV)
    opt = AdamW([p], lr=1e-2, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    z = np.zeros(n, F)
    r = dict(p=z, m=z, v=z)
    for t in (1, 2, 3):
        opt.step()
        new, m, v = step32(r["p"], g, r["m"], r["v"], t, 1e-2, 0.9, 0.999, 1e-8, 0.0)
        assert _same_p(_np(p), r["p"], new, torch.float32)
        r["p"] = _np(p)
        r["m"], r["v"] = _check_state(opt.state[p], m, v, t)
    assert bool(torch.isfinite(torch.stack(opt.moments())).all())


@pytest.mark.gpu
def test_late_steps_wrap_the_sequences():
    """Offsets are sums modulo 2^32 of (element, step): steps near the largest step count."""
    from ubio_molfm_b200.optim import AdamW

    n = 3000
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = AdamW([p], lr=1e-3, state_bits=8)
    held = opt.flat_state()
    held["step"].fill_(2 ** 31 - 3)
    z = np.zeros(n, F)
    p.grad = _grad(n, torch.float32, 1).to(DEV)
    opt.step()
    _, m, v = step32(z, _np(p.grad), z, z, 2 ** 31 - 2, 1e-3, 0.9, 0.999, 1e-8, 1e-2)
    _check_state(opt.state[p], m, v, 2 ** 31 - 2)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, 1e-8])
def test_second_moments_below_the_normal_range(eps):
    """Gradients of order 1 beside ones whose squares are subnormal, in whole blocks and in one that is cut short: a
    second moment over 0 keeps a root over 0, and with eps = 0 the update has it in its denominator."""
    from ubio_molfm_b200.optim import AdamW

    n = 4 * 256 + 99
    rng = np.random.default_rng(8)
    g = rng.normal(size=n)
    tiny = rng.random(n) < 0.5
    g[tiny] = rng.choice([-1, 1], tiny.sum()) * np.exp(rng.uniform(np.log(4e-21), np.log(2e-17), tiny.sum()))
    g[300:400] = 0
    g = g.astype(F)
    p0 = rng.normal(size=n).astype(F)
    if eps == 0:
        g[300:400] = 1.0                         # 0 / 0 is not a number, here as in the formula
    p = torch.nn.Parameter(torch.from_numpy(p0.copy()).to(DEV))
    p.grad = torch.from_numpy(g).to(DEV)
    opt = AdamW([p], lr=1e-2, betas=(0.9, 0.999), eps=eps, weight_decay=0.0, state_bits=8)
    r = dict(p=p0, m=np.zeros(n, F), v=np.zeros(n, F))
    for t in (1, 2, 3):
        opt.step()
        new, m, v = step32(r["p"], g, r["m"], r["v"], t, 1e-2, 0.9, 0.999, eps, 0.0)
        assert ((v > 0) == (g != 0)).all() and np.isfinite(new).all()
        assert _same_p(_np(p), r["p"], new, torch.float32), t
        r["p"] = _np(p)
        r["m"], r["v"] = _check_state(opt.state[p], m, v, t)
