"""AdamW over many tensors (32- and 8-bit moments) and the global gradient norm (``ubio_molfm_b200.optim``).

The moments' fp32 operations are each rounded once in a stated order, so the reference below, the same order in
numpy's float32, has to agree bit for bit: in 32-bit moments and in every 8-bit code.  The parameter's update takes
reciprocals and roots within one or two units: with u = 2^-24 the update has relative errors of 2 u (root), u (sum
with eps), 2 u (reciprocal), u (product) and at most half of the moments', the reference's own about as many, and
p decay and the difference 2 u each: |dp| <= 16 u (|p| + |update|), and one step of the parameter's type where that
is narrower (``_same_p``)."""
import copy
import ctypes
import io
import math
from array import array

import numpy as np
import pytest
import torch

DEV = "cuda"
U = 2.0 ** -24
F = np.float32
SIZES = [1, 255, 256, 257, 0, 1000, 4099, 70001]
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


# ------------------------------------------------------------------------------------------------
# the 8-bit format, by value (not by bit patterns)
# ------------------------------------------------------------------------------------------------
def _offsets(n, t):
    """Offsets in [0, 1) of the first and second moments' roundings for elements 0..n-1 at step t."""
    low = np.uint64(0xFFFFFFFF)
    u = (np.arange(n, dtype=np.uint64) * np.uint64(0xDB4F0B91) + np.uint64(t) * np.uint64(0xBBE05633)) & low
    u = ((u ^ (u >> np.uint64(16))) * np.uint64(0xA0F2EC75)) & low
    u = ((u ^ (u >> np.uint64(15))) * np.uint64(0x89E18285)) & low
    u = u ^ (u >> np.uint64(16))
    return (u >> np.uint64(12)).astype(np.float64) / 2 ** 20, (u & np.uint64(0x7FFFF)).astype(np.float64) / 2 ** 19


def pack(x, offset, fraction):
    """Codes and block scales of fp32 values ``x``; ``offset`` in [0, 1) decides which way a value is rounded."""
    n = x.size
    nb = -(-n // 256)
    xb = np.zeros(nb * 256)
    xb[:n] = np.abs(x.astype(np.float64))
    top = xb.reshape(nb, 256).max(1, initial=0)
    e = np.floor(np.log2(np.maximum(top, 1e-300))).astype(int)
    e = np.clip(e + (top >= np.exp2(e) * (2 - 2.0 ** -fraction)), -100, 126)     # room to round up
    y = np.abs(x.astype(np.float64)) / np.exp2(np.repeat(e, 256)[:n].astype(np.float64))
    with np.errstate(divide="ignore"):
        k = np.maximum(np.floor(np.log2(y)), -14)
    small = y < 2.0 ** -14
    y = np.where(small, np.round(y * 2.0 ** 37) / 2.0 ** 37, y)     # what is left of fp32 down there
    k = np.where(small & (y >= 2.0 ** -14), -14, k)
    steps = y / np.exp2(k - fraction)                                # in units of the code's last place
    low = np.floor(steps)
    low = low + ((steps - low) + offset >= 1)
    code = (low + (k + 14) * 2 ** fraction).astype(int)              # the binades follow one another
    code = np.minimum(code, 2 ** (4 + fraction) - 1)
    if fraction == 4:
        code = np.maximum(code, (x > 0).astype(int))
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
    return p * F(1 - lr * wd) - m / (np.sqrt(v) * root + F(eps)) * size, m, v


def clip_coef(norm, most):
    return np.minimum(F(most) / (F(norm) + F(1e-6)), F(1))


@pytest.mark.parametrize("fraction", [3, 4])
def test_format_is_unbiased_and_close(fraction):
    """Each held value is within one place of the value.  A rounding's error has a standard deviation of at most
    half a place, the mean of T = 4,096 of them of 1/128: six of those, for 256 values."""
    rng = np.random.default_rng(0)
    x = np.exp(rng.uniform(-9, 0, 256)).astype(F)
    x[0] = 1.9
    T = 4096
    held = np.zeros(256)
    place = np.exp2(np.maximum(np.floor(np.log2(x.astype(np.float64))), -14) - fraction)
    for t in range(T):
        code, scale = pack(x, _offsets(256, t)[fraction - 3], fraction)
        y = unpack(code, scale, fraction).astype(np.float64)
        assert (np.abs(y - x) <= place).all()
        held += y / T
    assert (np.abs(held - x) <= 6 / 128 * place).all()


def test_a_slowly_growing_average_keeps_growing():
    """The largest value of a block, raised by 0.1 % a step through its whole binade and held in 8 bits in
    between, follows (round-to-nearest, or a largest code to stop at, would keep it where it is)."""
    n = 4096
    start = np.random.default_rng(0).uniform(1, 2, n).astype(F)
    held, x = start, 1.0
    for t in range(1, 1001):
        held = unpack(*pack(held * F(1.001), _offsets(n, t)[1], 4), 4)
        x *= 1.001
    # a step raises a value by a place of 1/32 to 1/16 of it with probability 0.001 over that: a relative variance
    # of at most 0.001 / 16 a step, 0.25^2 in 1,000 of them, 0.25 / 64 for the mean of 4,096; five of those
    assert abs(float((held / start).mean()) / x - 1) <= 5 * 0.25 / 64


def test_format_corner_values():
    x = np.zeros(512, F)
    x[3], x[300], x[301] = 1e-20, 5.0, -1e-30
    code, scale = pack(x, np.full(512, 0.999), 3)
    assert scale[1] == 129 and code[301] & 127 <= 1 and (code[:3] == 0).all()
    assert abs(unpack(code, scale, 3)[3] - 1e-20) <= 1e-20 / 8
    s, sc = pack(np.abs(x), np.zeros(512), 4)
    assert s[301] == 1 and unpack(s, sc, 4)[301] == F(4 * 2.0 ** -18)    # over 0 stays over 0
    assert (unpack(*pack(np.zeros(256, F), np.full(256, 0.999), 3), 3) == 0).all()


# ------------------------------------------------------------------------------------------------
# refusals, on the host
# ------------------------------------------------------------------------------------------------
def test_constructor_refusals():
    from ubio_molfm_b200.optim import AdamW, grad_norm

    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(state_bits=16), dict(max_grad_norm=0.0), dict(max_grad_norm=float("nan")), dict(betas=(1.0, 0.9)),
                dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(lr=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            AdamW(p, **bad)
    with pytest.raises(ValueError):
        AdamW([p[0], p[0]])
    p[0].grad = torch.ones(3)
    with pytest.raises(ValueError, match="CUDA"):
        AdamW(p).step()
    with pytest.raises(ValueError, match="CUDA"):
        grad_norm([torch.ones(3)])


def unlike_gradients():
    """Parameters whose gradients are not of their type, size or device, with the error each is to raise."""
    def of(device, grad, data=None):
        p = torch.nn.Parameter(torch.zeros(4, device=device))
        if grad != torch.float32:
            p.grad_dtype = grad
        p.grad = torch.ones(4, dtype=grad, device=device)
        if data is not None:
            p.data = data
        return p

    return [(lambda dev: of(dev, torch.bfloat16), TypeError), (lambda dev: of(dev, torch.float64), TypeError),
            (lambda dev: of(dev, torch.float32, torch.zeros(4, dtype=torch.bfloat16, device=dev)), TypeError),
            (lambda dev: of(dev, torch.float32, torch.zeros(1000, device=dev)), ValueError),
            (lambda dev: of(dev, torch.float32, torch.zeros(2, device=dev)), ValueError)]


def test_unlike_gradients_are_refused_on_the_host():
    from ubio_molfm_b200.optim import _gradients

    for make, error in unlike_gradients():
        with pytest.raises(error, match="gradient"):
            _gradients([make("cpu")])
    p = torch.nn.Parameter(torch.zeros(4, 2))
    p.grad = torch.arange(8.0).reshape(2, 4).t()
    assert torch.equal(_gradients([p])[0], p.grad) and _gradients([p])[0].is_contiguous()


def test_streams_are_of_cuda_devices():
    from ubio_molfm_b200 import _lib

    with pytest.raises((ValueError, RuntimeError, AssertionError)):      # no device to ask, or not one of CUDA's
        _lib.stream_of(torch.device("cpu"))


def test_c_abi_refuses_bad_arguments():
    """Every check comes before device work: the addresses are never read."""
    from ubio_molfm_b200 import _lib

    lib = _lib.load()
    dev = ctypes.c_void_p(1 << 20)

    def call(p=(4096, 8192), g=(12288, 16384), numel=(10, 300), off=(0, 256), slot=(0, 1), dtype=0, bits=32, m=dev,
             scale=dev, elements=768, b1=0.9, b2=0.999, eps=1e-8, norm=None, most=1.0, ws=dev, size=1 << 12, step=dev):
        keep = [array("Q", p), array("Q", g), array("q", numel), array("q", off), array("i", slot)]
        return lib.e2a_adamw_step(*[a.buffer_info()[0] for a in keep], len(numel), dtype, bits, m, dev, scale, dev,
                                  elements, step, 1e-3, None, b1, b2, eps, 0.0, norm, most, ws, size, None)

    bad = [dict(dtype=3), dict(bits=16), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(norm=dev, most=0.0),
           dict(m=None), dict(step=None), dict(bits=8, scale=None), dict(numel=(10, -1)), dict(p=(0, 8192)),
           dict(p=(4098, 8192)), dict(g=(12288, 16386)), dict(off=(0, 128)), dict(off=(256, 0)), dict(slot=(1, 0)),
           dict(slot=(1, 1)), dict(elements=512 + 128), dict(slot=(-1, 0))]
    for kw in bad:
        assert call(**kw) == 1, kw
    assert call(ws=None) == 3 and call(size=15) == 3
    # memory that a parameter shares with another parameter or a gradient
    assert call(p=(4096, 4096)) == 1 and call(p=(4096, 4096 + 36)) == 1 and call(g=(4096, 16384)) == 1
    assert call(g=(8192 + 1196, 16384)) == 1
    n = array("q", [0])
    t, k = array("Q", [4096]), array("q", [7])
    assert lib.e2a_sum_squares(t.buffer_info()[0], k.buffer_info()[0], 1, 5, dev, 64, n.buffer_info()[0], None) == 1
    assert lib.e2a_sum_squares(t.buffer_info()[0], k.buffer_info()[0], 1, 0, dev, 0, n.buffer_info()[0], None) == 3
    assert lib.e2a_sum_squares(None, None, 0, 0, None, 0, n.buffer_info()[0], None) == 0 and n[0] == 0
    assert lib.e2a_norm_of_squares(None, 0, None, None) == 1 and lib.e2a_norm_of_squares(None, 4, dev, None) == 1
    assert lib.e2a_grad_norm(t.buffer_info()[0], k.buffer_info()[0], 1, 0, dev, 0, dev, None) == 3
    assert lib.e2a_grad_norm(t.buffer_info()[0], k.buffer_info()[0], -1, 0, dev, 64, dev, None) == 1
    assert lib.e2a_moments_unpack(None, None, None, None, 5, None, None, None) == 1


# ------------------------------------------------------------------------------------------------
# the step
# ------------------------------------------------------------------------------------------------
def _same_p(got, before, want, dtype=torch.float32):
    """``got`` is ``want`` (float32) but for the update's last units; ``before``: the parameter before the step."""
    up = np.abs(want.astype(np.float64) - before) + 0.2 * np.abs(before)
    tol = 16 * U * (np.abs(before) + up) + 1e-44
    if dtype != torch.float32:
        tol += 2 * HALF[dtype] * np.abs(want) + (2.0 ** -24 if dtype == torch.float16 else 0)
    return bool((np.abs(got.astype(np.float64) - want) <= tol).all())


def _params(sizes, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ps = []
    for k, n in enumerate(sizes):
        p = torch.nn.Parameter((0.1 * torch.randn(n, generator=gen)).to(dtype).to(DEV))
        p.grad = _grad(n, dtype, 100 * seed + k).to(DEV)
        ps.append(p)
    return ps


def _grad(n, dtype, seed):
    gen = torch.Generator().manual_seed(7919 + seed)
    return (10.0 ** ((seed % 5) - 3) * torch.randn(n, generator=gen)).to(dtype)


def _np(t):
    return t.detach().float().cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [None, 0.5, 1e6])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_equal_the_stated_arithmetic_bit_for_bit(dtype, bits, clip):
    from ubio_molfm_b200.optim import AdamW

    ps = _params(SIZES, dtype)
    lr, b1, b2, eps, wd = 3e-3, 0.9, 0.99, 1e-8, 0.05
    opt = AdamW(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits, max_grad_norm=clip)
    ref = [dict(p=_np(p), m=np.zeros(p.numel(), F), v=np.zeros(p.numel(), F)) for p in ps]
    for t in range(1, 5):
        for k, p in enumerate(ps):
            p.grad = _grad(p.numel(), dtype, 31 * t + k).to(DEV)
        opt.step()
        gs = [_np(p.grad) for p in ps]
        coef = None
        if clip is not None:
            norm = F(math.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in gs)))
            assert float(opt.last_grad_norm) == float(norm)
            coef = clip_coef(norm, clip)
        for k, (p, r, g) in enumerate(zip(ps, ref, gs)):
            new, m, v = step32(r["p"], g, r["m"], r["v"], t, lr, b1, b2, eps, wd, coef)
            st = opt.state[p]
            assert int(st["step"]) == t
            assert _same_p(_np(p), r["p"], new, dtype), (t, k)
            r["p"] = _np(p)
            if bits == 32:
                r["m"], r["v"] = m, v
                assert np.array_equal(_np(st["exp_avg"]), m) and np.array_equal(_np(st["exp_avg_sq"]), v), (t, k)
            elif p.numel():
                om, ov = _offsets(p.numel(), t)
                cm, sm = pack(m, om, 3)
                cv, sv = pack(np.sqrt(v), ov, 4)
                for name, want in (("exp_avg", cm), ("exp_avg_scale", sm), ("exp_avg_sq", cv), ("exp_avg_sq_scale", sv)):
                    assert np.array_equal(st[name].cpu().numpy(), want), (t, k, name)
                s = unpack(cv, sv, 4)
                r["m"], r["v"] = unpack(cm, sm, 3), s * s
    m, v = opt.moments()
    for k, r in enumerate(ref):
        o = opt._group_state(0).offset[k]
        n = ps[k].numel()
        assert np.array_equal(_np(m[o:o + n]), r["m"]) and np.array_equal(_np(v[o:o + n]), r["v"])
        end = -(-n // 256) * 256
        assert not bool(m[o + n:o + end].any()) and not bool(v[o + n:o + end].any())     # nothing between tensors


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_one_step_against_the_formula_in_64_bits(bits):
    """Per element at most 3 roundings in m and 4 in v, of terms below |m| + |g| and v + g^2; the quotient of
    them by sqrt(v) root + eps adds 6 (root halves v's relative error), size, decay and the last difference 4:
    |dp| <= 16 u (|p| + |update terms|).  beta's own rounding is one of the roundings."""
    from ubio_molfm_b200.optim import AdamW

    ps = _params([5000, 300], torch.float32, 5)
    opt = AdamW(ps, lr=1e-2, betas=(0.9, 0.999), weight_decay=0.1, state_bits=bits, max_grad_norm=0.3)
    before = [p.detach().double().clone() for p in ps]
    norm = torch.cat([p.grad.double() for p in ps]).norm()
    opt.step()
    assert abs(float(opt.last_grad_norm) - float(norm)) <= U * float(norm)
    coef = min(1.0, 0.3 / (float(norm) + 1e-6))
    for p, p0 in zip(ps, before):
        g = p.grad.double() * coef
        m, v = 0.1 * g, 0.001 * g * g
        up = 1e-2 / (1 - 0.9) * m / ((v / (1 - 0.999)).sqrt() + 1e-8)
        want = p0 * (1 - 1e-2 * 0.1) - up
        assert bool(((p.double() - want).abs() <= 16 * U * (p0.abs() + up.abs())).all())
        if bits == 32:
            assert bool(((opt.state[p]["exp_avg"].double() - m).abs() <= 4 * U * m.abs()).all())
            assert bool(((opt.state[p]["exp_avg_sq"].double() - v).abs() <= 6 * U * v).all())


@pytest.mark.gpu
def test_follows_pytorch_over_steps():
    """20 steps beside torch.optim.AdamW in 64 bits: each step's rounding is below 16 u (|p| + lr-sized update),
    and a step's update depends on the last only through the moments, which carry relative errors of a few u."""
    from ubio_molfm_b200.optim import AdamW

    ps = _params([1000, 77], torch.float32, 6)
    qs = [torch.nn.Parameter(p.detach().double()) for p in ps]
    opt = AdamW(ps, lr=1e-2, weight_decay=0.1)
    ref = torch.optim.AdamW(qs, lr=1e-2, weight_decay=0.1)
    for t in range(20):
        for k, (p, q) in enumerate(zip(ps, qs)):
            p.grad = _grad(p.numel(), torch.float32, 50 * t + k).to(DEV)
            q.grad = p.grad.double()
        opt.step()
        ref.step()
    for p, q in zip(ps, qs):
        assert float((p.double() - q).detach().abs().max()) <= 20 * 16 * U * (float(q.detach().abs().max()) + 1e-2 * 10)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_views_and_unaligned_memory(bits):
    """1,300 tensors, each at an odd element of one allocation: no vector load fits, and the gaps stay."""
    from ubio_molfm_b200.optim import AdamW

    sizes = [(37 * k) % 301 + 1 for k in range(1300)]
    starts = np.concatenate([[1], 1 + np.cumsum([n + 3 for n in sizes])])
    p_all = torch.randn(int(starts[-1]), device=DEV)
    g_all = torch.randn(int(starts[-1]), device=DEV)
    before = p_all.clone()
    ps = []
    for n, o in zip(sizes, starts):
        ps.append(torch.nn.Parameter(p_all[o:o + n]))
        ps[-1].grad = g_all[o:o + n]
    opt = AdamW(ps, lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    opt.step()
    inside = torch.zeros_like(p_all, dtype=torch.bool)
    for n, o in zip(sizes, starts):
        inside[o:o + n] = True
    assert torch.equal(p_all[~inside], before[~inside])
    g64 = g_all[inside].double().cpu().numpy()
    coef = clip_coef(F(math.sqrt(float((g64 ** 2).sum()))), 1.0)
    zero = np.zeros(g64.size, F)
    want, _, _ = step32(_np(before[inside]), g64.astype(F), zero, zero, 1, 1e-2, 0.9, 0.999, 1e-8, 1e-2, coef)
    assert _same_p(_np(p_all[inside]), _np(before[inside]), want)
    assert bool((opt.flat_state()["step"] == 1).all())


@pytest.mark.gpu
def test_parameters_without_gradient_and_groups():
    from ubio_molfm_b200.optim import AdamW

    ps = _params([100, 200, 300, 50], torch.float32, 2)
    ps.append(torch.nn.Parameter(torch.randn(70, device=DEV, dtype=torch.bfloat16)))
    ps[4].grad = torch.ones_like(ps[4])
    start = [p.detach().clone() for p in ps]
    opt = AdamW([dict(params=[ps[0], ps[1], ps[4]], weight_decay=0.0), dict(params=ps[2:4], lr=0.5)], lr=1e-3)
    ps[1].grad = None
    opt.step()
    assert torch.equal(ps[1], start[1]) and not torch.equal(ps[0], start[0])
    assert float((ps[2].detach() - start[2]).abs().min()) > 0.3           # the second group's lr: the first step is lr sign(g)
    ps[1].grad = torch.ones_like(ps[1])
    opt.step()
    assert [int(opt.state[p]["step"]) for p in ps] == [2, 1, 2, 2, 2]
    # the late parameter's first step has its own bias correction: lr g / (|g| + eps), no decay
    want, _, _ = step32(_np(start[1]), np.ones(200, F), np.zeros(200, F), np.zeros(200, F), 1, 1e-3, 0.9, 0.999, 1e-8, 0.0)
    assert _same_p(_np(ps[1]), _np(start[1]), want)
    for p in ps:
        p.grad = None
    opt.step()                                                    # nothing to do
    assert [int(opt.state[p]["step"]) for p in ps] == [2, 1, 2, 2, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_step_with_a_non_finite_norm_changes_nothing(bits, bad):
    from ubio_molfm_b200.optim import AdamW

    ps = _params([300, 1000], torch.float32, 3)
    opt = AdamW(ps, state_bits=bits, max_grad_norm=1.0)
    opt.step()
    held = [p.detach().clone() for p in ps] + [t.clone() for t in opt.flat_state().values()]
    good = ps[1].grad.clone()
    ps[1].grad[17] = bad
    opt.step()
    assert not math.isfinite(float(opt.last_grad_norm))
    now = [p.detach() for p in ps] + list(opt.flat_state().values())
    assert all(torch.equal(a, b) for a, b in zip(held, now))
    ps[1].grad = good
    opt.step()
    assert int(opt.state[ps[0]]["step"]) == 2


@pytest.mark.gpu
def test_non_finite_gradients_without_clipping():
    """32 bits: the element is NaN, the others are not touched by it.  8 bits: its block of 256 moments stands
    for NaN from then on, the other blocks do not."""
    from ubio_molfm_b200.optim import AdamW

    for bits in (32, 8):
        ps, qs = _params([700], torch.float32, 4), _params([700], torch.float32, 4)
        ps[0].grad[300] = float("nan")
        a, b = AdamW(ps, state_bits=bits), AdamW(qs, state_bits=bits)
        a.step()
        b.step()
        hit = torch.zeros(700, dtype=torch.bool, device=DEV)
        hit[300] = True
        assert bool(ps[0][hit].isnan().all()) and torch.equal(ps[0][~hit], qs[0][~hit])
        m, v = (t[:700] for t in a.moments())
        m0, v0 = (t[:700] for t in b.moments())
        if bits == 8:
            hit[256:512] = True
        assert bool(m[hit].isnan().all()) and bool(v[hit].isnan().all())
        assert torch.equal(m[~hit], m0[~hit]) and torch.equal(v[~hit], v0[~hit])


@pytest.mark.gpu
def test_extreme_magnitudes_in_8_bits():
    from ubio_molfm_b200.optim import AdamW

    p = torch.nn.Parameter(torch.zeros(1024, device=DEV))
    g = torch.zeros(1024)
    g[:256] = torch.linspace(-3e18, 3e18, 256)          # squares near fp32's largest
    g[256:512] = 1e-37 * torch.randn(256)               # moments below 2^-100
    g[700] = 1.0                                        # one among zeros
    p.grad = g.to(DEV)
    opt = AdamW([p], lr=1e-2, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    opt.step()
    z = np.zeros(1024, F)
    want, m, v = step32(z, g.numpy(), z, z, 1, 1e-2, 0.9, 0.999, 1e-8, 0.0)
    om, ov = _offsets(1024, 1)
    (cm, sm), (cv, sv) = pack(m, om, 3), pack(np.sqrt(v), ov, 4)
    st = opt.state[p]
    assert _same_p(_np(p), z, want)
    for name, w in (("exp_avg", cm), ("exp_avg_scale", sm), ("exp_avg_sq", cv), ("exp_avg_sq_scale", sv)):
        assert np.array_equal(st[name].cpu().numpy(), w), name
    assert bool(torch.isfinite(torch.stack(opt.moments())).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_copies_and_pickles_continue_alike(bits):
    from ubio_molfm_b200.optim import AdamW

    def fresh():
        return _params([300, 700, 64], torch.bfloat16, 8)

    ps = fresh()
    opt = AdamW([dict(params=ps[:2]), dict(params=ps[2:], lr=0.1)], state_bits=bits)
    opt.step()
    opt.step()
    saved = io.BytesIO()
    torch.save(dict(opt=opt.state_dict(), p=[p.detach() for p in ps]), saved)
    saved.seek(0)
    held = torch.load(saved, map_location="cpu")
    qs = fresh()
    for q, t in zip(qs, held["p"]):
        q.data.copy_(t)
    other = AdamW([dict(params=qs[:2]), dict(params=qs[2:])], state_bits=bits)
    other.load_state_dict(held["opt"])
    assert other.param_groups[1]["lr"] == 0.1
    rs, third = copy.deepcopy((ps, opt))
    for r, p in zip(rs, ps):
        r.grad = p.grad
    for o in (opt, other, third):
        o.step()
    for p, q, r in zip(ps, qs, rs):
        assert torch.equal(p, q) and torch.equal(p, r)
    for gi in (0, 1):
        for a, b, c in zip(opt.flat_state(gi).values(), other.flat_state(gi).values(), third.flat_state(gi).values()):
            assert torch.equal(a, b) and torch.equal(a, c) and a.data_ptr() != c.data_ptr()
    with pytest.raises(ValueError, match="bit"):
        AdamW([dict(params=qs[:2]), dict(params=qs[2:])], state_bits=40 - bits).load_state_dict(held["opt"])
    with pytest.raises(ValueError, match="shape"):
        AdamW([dict(params=qs[1:]), dict(params=qs[:1])], state_bits=bits).load_state_dict(held["opt"])


@pytest.mark.gpu
def test_caches_and_saved_tensors_see_the_step():
    from ubio_molfm_b200.optim import AdamW

    p = torch.nn.Parameter(torch.ones(10, device=DEV))
    y = (p * p).sum()
    p.grad = torch.ones(10, device=DEV)
    before = p._version
    AdamW([p]).step()
    assert p._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_with_a_tensor_lr(bits):
    """One captured step replayed three times, the learning rate changed in between, equals eager steps; a
    second optimiser's captured step replayed between them changes nothing."""
    from ubio_molfm_b200.optim import AdamW

    def make(seed, lr):
        ps = _params([5000, 33], torch.float32, seed)
        return ps, AdamW(ps, lr=lr, state_bits=bits, max_grad_norm=1.0)

    eager, opt = make(9, 1e-3)
    lr = torch.tensor(1e-3, device=DEV)
    ps, cap = make(9, lr)
    qs, other = make(11, 1e-2)
    for o in (cap, other):
        o.flat_state()                                  # the state is made before the capture
    graphs = []
    for o in (cap, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o.step()
        graphs.append(g)
    for t, value in enumerate((1e-3, 5e-4, 2e-3)):
        for k in range(2):
            new = _grad(eager[k].numel(), torch.float32, 70 + 3 * t + k).to(DEV)
            eager[k].grad.copy_(new)
            ps[k].grad.copy_(new)
        lr.fill_(value)
        opt.param_groups[0]["lr"] = float(F(value))
        graphs[0].replay()
        graphs[1].replay()
        opt.step()
        for a, b in zip(eager, ps):
            assert torch.equal(a, b), t
    for a, b in zip(opt.flat_state().values(), cap.flat_state().values()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_other_stream_and_other_layouts():
    from ubio_molfm_b200.optim import AdamW, grad_norm

    a, b = _params([3000], torch.float32, 12), _params([3000], torch.float32, 12)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        opt = AdamW(a, max_grad_norm=1.0)
        opt.step()
    torch.cuda.current_stream().wait_stream(s)
    AdamW(b, max_grad_norm=1.0).step()
    assert torch.equal(a[0], b[0])
    # a gradient with another layout than the parameter's
    g = torch.randn(30, 40, device=DEV)
    p, q = (torch.nn.Parameter(torch.ones(40, 30, device=DEV)) for _ in range(2))
    p.grad, q.grad = g.t(), g.t().contiguous()
    for t in (p, q):
        AdamW([t], max_grad_norm=1.0).step()
    assert torch.equal(p, q)
    r = torch.nn.Parameter(torch.ones(30, 40, device=DEV).t())
    r.grad = g.t()
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([r]).step()
    d = torch.nn.Parameter(torch.ones(3, device=DEV, dtype=torch.float64))
    d.grad = torch.ones_like(d)
    with pytest.raises(TypeError):
        AdamW([d]).step()
    with pytest.raises(TypeError):
        grad_norm([d])
    w = torch.nn.Parameter(torch.zeros(8, device=DEV))
    w.grad = w.data                                      # a gradient in the parameter's own memory
    with pytest.raises(RuntimeError, match="argument"):
        AdamW([w]).step()


@pytest.mark.gpu
def test_learning_rates_as_tensors_and_schedules():
    from ubio_molfm_b200.optim import AdamW

    a, b, c = (_params([500], torch.float32, 13) for _ in range(3))
    oa, ob = AdamW(a, lr=2e-3), AdamW(b, lr=torch.tensor(2e-3))
    oc = AdamW(c, lr=4e-3)
    torch.optim.lr_scheduler.LambdaLR(oc, lambda epoch: 0.5)          # takes the optimiser, sets lr to 2e-3
    for o in (oa, ob, oc):
        o.step()
    assert torch.equal(a[0], c[0])
    # 2e-3 as a float32 tensor is off by at most 2^-24 of itself, and so is the update of at most 2e-3
    assert float((a[0] - b[0]).detach().abs().max()) <= 2e-3 * 2 * U + 2 * U * float(a[0].detach().abs().max())
    d = _params([8], torch.float32, 1)
    with pytest.raises(ValueError, match="lr"):
        AdamW(d, lr=torch.tensor(1e-3, dtype=torch.float64, device=DEV)).step()


@pytest.mark.gpu
def test_sparse_gradients_are_refused():
    from ubio_molfm_b200.optim import AdamW, grad_norm

    e = torch.nn.Embedding(10, 4, sparse=True).to(DEV)
    e(torch.tensor([1, 2], device=DEV)).sum().backward()
    with pytest.raises(TypeError):
        AdamW(e.parameters()).step()
    with pytest.raises(TypeError):
        grad_norm([e.weight.grad])


@pytest.mark.gpu
def test_unlike_gradients_are_refused():
    from ubio_molfm_b200.optim import AdamW

    for make, error in unlike_gradients():
        for bits in (32, 8):
            p, q = make(DEV), torch.nn.Parameter(torch.ones(5, device=DEV))
            q.grad = torch.ones(5, device=DEV)
            opt = AdamW([q, p], state_bits=bits, max_grad_norm=1.0)
            with pytest.raises(error, match="gradient"):
                opt.step()
            assert (q == 1).all() and (p == 0).all() and not opt.flat_state()["step"].any()
            p.grad = None
            opt.step()
            assert (q != 1).all() and opt.flat_state()["step"].tolist() == [1, 0]


@pytest.mark.gpu
def test_more_than_2_to_the_32_elements():
    """Elements 2^32 apart have the same mixed bits: with the same values in every block of 256, the block that
    starts there becomes what the first one becomes."""
    from ubio_molfm_b200.optim import AdamW, grad_norm

    n, tail = (1 << 32) + 256 * 3 + 100, 256
    block = torch.randn(256, device=DEV).bfloat16()
    p = torch.nn.Parameter(torch.empty(n, dtype=torch.bfloat16, device=DEV))
    whole = n // 256 * 256
    with torch.no_grad():
        p[:whole].view(-1, 256).copy_(block)
        p[whole:] = block[:n - whole]
    p.grad = p.detach().clone()
    want = math.sqrt(float(block.double().square().sum()) * (n // 256) + float(block[:n - whole].double().square().sum()))
    assert abs(float(grad_norm([p.grad])) - want) <= (U + 1e-9) * want
    opt = AdamW([p], lr=1e-2, state_bits=8)
    for _ in range(2):
        opt.step()
    st = opt.flat_state()
    at = 1 << 32
    assert torch.equal(p[at:at + tail], p[:tail]) and not torch.equal(p[:tail].detach(), block)
    for k in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(st[k][at:at + tail], st[k][:tail])
        assert not bool(st[k][n:].any())
    # the last block, cut short: its moments have the first one's values or, where its largest value is smaller,
    # a smaller scale; its parameters do not depend on that after one step more than the moments' own rounding
    assert bool(torch.isfinite(p[-100:]).all()) and not torch.equal(p[-100:].detach(), block[:100])


# ------------------------------------------------------------------------------------------------
# the norm
# ------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [0], [7, 0, 100000], [300] * 1100, [5_000_001, 33]])
def test_grad_norm(sizes):
    """Squares and sums are in 64 bits (errors below 1e-10 relative), the result is rounded once."""
    from ubio_molfm_b200.optim import grad_norm

    ts = [_grad(n, (torch.float32, torch.bfloat16, torch.float16)[k % 3], k).to(DEV) for k, n in enumerate(sizes)]
    want = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    got = grad_norm(ts)
    assert got.shape == () and got.dtype == torch.float32 and got.device == ts[0].device
    assert abs(float(got) - want) <= (U + 1e-10) * want
    assert torch.equal(got, grad_norm(ts))
    strided = [t[::2] for t in ts]
    want = math.sqrt(sum(float(t.double().square().sum()) for t in strided))
    assert abs(float(grad_norm(strided)) - want) <= (U + 1e-10) * want


@pytest.mark.gpu
def test_grad_norm_corners():
    from ubio_molfm_b200.optim import grad_norm

    assert float(grad_norm([])) == 0.0
    big = torch.full((4,), 1e38, device=DEV)
    assert abs(float(grad_norm([big])) - 2e38) <= U * 2e38          # the squares pass fp32's range
    assert math.isinf(float(grad_norm([big] * 9)))                  # so does this norm itself
    assert math.isnan(float(grad_norm([big, torch.tensor([float("nan")], device=DEV)])))
    tiny = torch.full((10000,), 1e-38, device=DEV)
    assert abs(float(grad_norm([tiny])) - 1e-36) <= 2 * U * 1e-36 + 1e-6 * U
