"""The training operators' cases: what is timed, their plain forms and their values in 64 bits.

Operators (``ubio_molfm_b200.norm`` and ``ubio_molfm_b200.optim``):

* ``ln``    layer norm, optionally with SiLU: forward and backward with the weight's and bias's gradients;
* ``ln2``   the same with the second-order backward that a loss on forces = -dE/dpos asks for;
* ``adamw`` one AdamW step over all tensors of a model, moments in 32 or in 8 bits, optionally with the
  gradients clipped to a global norm;
* ``gnorm`` the global L2 norm of all gradients.

``own`` selects the framework's calls; otherwise ``run`` computes the same in elementary torch operations.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
LR, BETA1, BETA2, ADAM_EPS, DECAY, MAX_NORM = 2e-4, 0.9, 0.999, 1e-8, 0.01, 1.0
STEP0 = 10          # steps taken before the timed one
BLOCK = 256         # elements that share one scale of an 8-bit moment; tensors start at its multiples


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------
def listed():
    return [
        # the small model's edge MLP (16 wide) on one 40-atom periodic box: latency
        dict(name="ln edges small", op="ln", rows=2560, width=16, dtype="f32", act=True),
        # the full model's edge MLP (128 wide) on the 20,000-atom layer's 640,210 edges
        dict(name="ln edges", op="ln", rows=640210, width=128, dtype="f32", act=True),
        # the Q / K scalar MLP (512 wide) on the nodes of the 97,865-atom system
        dict(name="ln nodes", op="ln", rows=97865, width=512, dtype="f32", act=True),
        # a plain norm of wide half-precision features (generic)
        dict(name="ln wide bf16", op="ln", rows=16384, width=4096, dtype="bf16", act=False),
        # rows that no vector load divides (generic, odd)
        dict(name="ln odd f16", op="ln", rows=12345, width=769, dtype="f16", act=False),
        # force-loss training of the 20,000-atom layer's edge MLP
        dict(name="ln2 edges", op="ln2", rows=640210, width=128, dtype="f32", act=True),
        # the optimiser's step on the small model (32 channels, 2 layers): latency over many tiny tensors
        dict(name="adamw small", op="adamw", model="small", dtype="f32", bits=32, clip=False),
        # the full-size model (256 channels, 4 layers, 240 tensors) as it is trained: fp32, clipped
        dict(name="adamw full", op="adamw", model="full", dtype="f32", bits=32, clip=True),
        # the same with moments in 8 bits
        dict(name="adamw full 8-bit", op="adamw", model="full", dtype="f32", bits=8, clip=True),
        # a large bf16 model's 101 tensors of ragged sizes (generic)
        dict(name="adamw large bf16 8-bit", op="adamw", model="ragged", tensors=101, total=120_000_000, sizes=7,
             dtype="bf16", bits=8, clip=False),
        # the clipping norm alone: the full-size model, and large ragged bf16 gradients
        dict(name="gnorm full", op="gnorm", model="full", dtype="f32"),
        dict(name="gnorm large bf16", op="gnorm", model="ragged", tensors=101, total=240_000_001, sizes=9,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln", "ln", "ln2", "adamw", "adamw", "gnorm"])
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    if op in ("ln", "ln2"):
        width = _log(rng, 8, 8192)
        if rng.random() < 0.5:
            width = (width + 7) // 8 * 8
        most = (64_000_000 if op == "ln" else 40_000_000) // width
        return dict(op=op, rows=_log(rng, 1, max(2, min(1_000_000, most))), width=width, dtype=dtype,
                    act=rng.random() < 0.6)
    case = dict(op=op, model="ragged", tensors=_log(rng, 1, 300), total=_log(rng, 1000, 60_000_000),
                sizes=rng.randrange(1 << 20), dtype=dtype)
    if op == "adamw":
        case.update(bits=rng.choice([32, 8]), clip=rng.random() < 0.5)
    return case


def _model_sizes(channels, heads, head_dim, basis, layers, head_mul):
    """Numbers of elements of the backbone's and energy head's trainable tensors."""
    C, hid, qk = channels, min(128, basis // 2), heads * head_dim // 2
    out = [256 * C, 30 * C, 30 * C, 2 * C * C, C, C * C, C, 256 * C, basis * heads, basis, 300 * basis, 300 * basis]
    for _ in range(3):
        out += [hid * 3 * basis, hid, hid, hid, hid * hid, hid, hid, hid, C * hid, C]
    out += [3 * C * 2 * C, C]
    for _ in range(layers):
        out += [3 * C, C, 256 * 128, 256 * 128]
        out += [hid * (basis + 256), hid, hid, hid, hid * hid, hid, hid, hid, 2 * heads * hid, 2 * heads]
        for _ in range(2):
            out += [3 * qk * C, qk, 3 * qk * C, qk * 3 * qk, qk, qk, qk, 2 * qk * qk, 2 * qk]
        hc = head_mul * heads
        out += [3 * C * C, C, C * hc, 3 * C * hc, 2 * C * hc, 3 * hc * C, C, 3 * C, C]
        out += [3 * C * C, C, 3 * C * C, 3 * C, 3 * C * C, C]
    return out + [3 * C, C, C * C, C, C * C, C, C, 1]


def _sizes(case):
    if case["model"] == "full":
        return _model_sizes(256, 128, 8, 256, 4, 2)
    if case["model"] == "small":
        return _model_sizes(32, 8, 8, 32, 2, 4)
    rng = random.Random(case["sizes"])
    n, total = case["tensors"], case["total"]
    share = [math.exp(rng.uniform(-4, 0)) for _ in range(n)]
    k = total / sum(share)
    return [max(1, int(s * k)) for s in share]


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _views(flat, offsets, sizes):
    return [flat[o:o + n] for o, n in zip(offsets, sizes)]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    if case["op"] in ("ln", "ln2"):
        n, w = case["rows"], case["width"]
        # rows of differing mean and spread, as a linear's outputs have
        x = (_randn(gen, n, w) * (0.5 + torch.rand(n, 1, generator=gen, device=DEV)) + 0.5 * _randn(gen, n, 1)).to(dt)
        st = dict(x=x.requires_grad_(True), w=(1 + 0.2 * _randn(gen, w)).requires_grad_(True),
                  b=(0.2 * _randn(gen, w)).requires_grad_(True), g=(0.1 * _randn(gen, n, w)).to(dt))
        if case["op"] == "ln2":
            st["g"].requires_grad_(True)
            st["u"] = (0.1 * _randn(gen, n, w)).to(dt)
        return dict(case=case, **st)
    sizes = _sizes(case)
    starts = np.concatenate([[0], np.cumsum([-(-n // BLOCK) * BLOCK for n in sizes])])
    total, offsets = int(starts[-1]), [int(o) for o in starts[:-1]]
    # zero in the gaps between tensors, where nothing is computed
    ends = torch.tensor([o + n for o, n in zip(offsets, sizes)], device=DEV)
    reps = torch.tensor(np.diff(starts), device=DEV)
    inside = torch.arange(total, device=DEV) < torch.repeat_interleave(ends, reps, output_size=total)
    # gradients whose size differs from tensor to tensor
    scale = 1e-3 * torch.exp(1.5 * _randn(gen, len(sizes))).repeat_interleave(reps, output_size=total) * inside
    g = (_randn(gen, total) * scale).to(dt)
    st = dict(case=case, sizes=sizes, g=g, grads=_views(g, offsets, sizes))
    if case["op"] == "gnorm":
        return st
    p = (0.06 * _randn(gen, total) * inside).to(dt)
    m = 0.3 * _randn(gen, total) * scale
    v = (0.7 + 0.6 * torch.rand(total, generator=gen, device=DEV)) * scale * scale
    st.update(p=p, step=torch.full((len(sizes),), STEP0, dtype=torch.int32, device=DEV))
    if case["bits"] == 8:
        index = (torch.arange(total, device=DEV) - torch.repeat_interleave(
            torch.tensor(offsets, device=DEV), reps, output_size=total)).view(-1, BLOCK)
        st["index"] = index
        st["m"], st["ms"] = _pack(m.view(-1, BLOCK), _dither(index, st["step"][:1], 0), 3)
        st["v"], st["vs"] = _pack(v.sqrt().view(-1, BLOCK), _dither(index, st["step"][:1], 1), 4)
    else:
        st["m"], st["v"] = m, v
    if own:
        from ubio_molfm_b200.optim import AdamW

        params = [torch.nn.Parameter(t) for t in _views(p, offsets, sizes)]
        for q, t in zip(params, st["grads"]):
            q.grad = t
        opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"],
                    max_grad_norm=MAX_NORM if case["clip"] else None)
        held = opt.flat_state(0)
        held["step"].copy_(st["step"])
        held["exp_avg"].copy_(st["m"].view(-1))
        held["exp_avg_sq"].copy_(st["v"].view(-1))
        if case["bits"] == 8:
            held["exp_avg_scale"].copy_(st["ms"].view(-1))
            held["exp_avg_sq_scale"].copy_(st["vs"].view(-1))
        st["opt"], st["held"] = opt, held
    return st


# ------------------------------------------------------------------------------------------------
# 8-bit moments, in elementary operations.  A block of 256 values shares the power of two of its largest
# magnitude; a value over it is a small float of 4 exponent bits and 3 (signed first moment) or 4 (square
# root of the second moment) fraction bits, rounded up with the probability that a fixed sequence over
# elements and steps gives.
# ------------------------------------------------------------------------------------------------
# odd 32-bit fractions of the powers of the root of x^5 = x + 1: additive sequences with independent steps
_INDEX_STEP = (0xDB4F0B91, 0xA0F2EC75)
_TIME_STEP = (0xBBE05633, 0x89E18285)


def _dither(index, step, which):
    """Uniform values below 2^20 (first moment) or 2^19 (second), [blocks, 256]."""
    u = (index * _INDEX_STEP[which] + step.long() * _TIME_STEP[which]) & 0xFFFFFFFF
    return (u >> (12 + which)).int()


def _pack(x, dither, fraction):
    mag = x.abs()
    b = (mag.amax(1, keepdim=True).view(torch.int32) >> 23).clamp(27, 253)
    z = mag * ((254 - b) << 23).view(torch.float32) * 2.0 ** -112
    top = 127 if fraction == 3 else 255
    code = ((z.view(torch.int32) + dither) >> (23 - fraction)).clamp(max=top)
    if fraction == 3:
        code = code | ((x < 0).int() << 7)
    else:
        code = torch.maximum(code, (x > 0).int())   # a second moment over zero stays over zero
    return code.to(torch.uint8), b.to(torch.uint8)


def _unpack(code, b, fraction):
    code = code.int()
    mag = code & 127 if fraction == 3 else code
    y = (mag << (23 - fraction)).view(torch.float32) * 2.0 ** 112 * (b.int() << 23).view(torch.float32)
    return torch.where(code > 127, -y, y) if fraction == 3 else y


# ------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "ln":
        return _run_ln(state)
    if op == "ln2":
        return _run_ln2(state)
    if op == "gnorm":
        return _run_gnorm(state)
    return _run_adamw(state)


def _run_ln(st):
    act = st["case"]["act"]
    if own:
        from ubio_molfm_b200.norm import layer_norm

        y = layer_norm(st["x"], st["w"], st["b"], EPS, "silu" if act else None)
        dx, dw, db = torch.autograd.grad(y, (st["x"], st["w"], st["b"]), st["g"])
        return dict(y=y, dx=dx, dw=dw, db=db)
    with torch.no_grad():
        x, w, b, g = st["x"].float(), st["w"], st["b"], st["g"].float()
        xc = x - x.mean(1, keepdim=True)
        r = 1 / (xc.square().mean(1, keepdim=True) + EPS).sqrt()
        xh = xc * r
        z = xh * w + b
        y, a = z, g
        if act:
            s = 1 / (1 + torch.exp(-z))
            y = z * s
            a = g * s * (1 + z * (1 - s))
        h = a * w
        dx = r * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
        dw = (a * xh).sum(0, dtype=torch.float64).float()
        db = a.sum(0, dtype=torch.float64).float()
        dt = st["x"].dtype
        return dict(y=y.to(dt), dx=dx.to(dt), dw=dw, db=db)


def _run_ln2(st):
    act = st["case"]["act"]
    if own:
        from ubio_molfm_b200.norm import layer_norm

        y = layer_norm(st["x"], st["w"], st["b"], EPS, "silu" if act else None)
        (dx,) = torch.autograd.grad(y, st["x"], st["g"], create_graph=True)
        gg, gx, gw, gb = torch.autograd.grad(dx, (st["g"], st["x"], st["w"], st["b"]), st["u"])
        return dict(y=y, dx=dx, gg=gg, gx=gx, gw=gw, gb=gb)
    with torch.no_grad():
        x, w, b, g, u = st["x"].float(), st["w"], st["b"], st["g"].float(), st["u"].float()
        xc = x - x.mean(1, keepdim=True)
        r = 1 / (xc.square().mean(1, keepdim=True) + EPS).sqrt()
        xh = xc * r
        z = xh * w + b
        if act:
            s = 1 / (1 + torch.exp(-z))
            y = z * s
            d1 = s * (1 + z * (1 - s))
            d2 = s * (1 - s) * (2 + z * (1 - 2 * s))
        else:
            y, d1, d2 = z, torch.ones_like(z), torch.zeros_like(z)
        a = g * d1
        h = a * w
        m1, m2 = h.mean(1, keepdim=True), (h * xh).mean(1, keepdim=True)
        dx = r * (h - m1 - xh * m2)
        # the gradients of S = <dx, u>; t = the norm's Jacobian applied to u
        c = (u * xh).mean(1, keepdim=True)
        t = r * (u - u.mean(1, keepdim=True) - xh * c)
        e = g * d2 * (w * t)
        k = e * w - r * (u * m2 + h * c)
        gx = r * (k - k.mean(1, keepdim=True) - xh * (k * xh).mean(1, keepdim=True) - xh * (h * t).mean(1, keepdim=True))
        gg = d1 * (w * t)
        gw = (a * t + e * xh).sum(0, dtype=torch.float64).float()
        gb = e.sum(0, dtype=torch.float64).float()
        dt = st["x"].dtype
        return dict(y=y.to(dt), dx=dx.to(dt), gg=gg.to(dt), gx=gx.to(dt), gw=gw, gb=gb)


def _norm(g):
    return g.double().square().sum().sqrt().float()


def _run_gnorm(st):
    if own:
        from ubio_molfm_b200.optim import grad_norm

        return dict(norm=grad_norm(st["grads"]))
    return dict(norm=_norm(st["g"]))


def _run_adamw(st):
    case = st["case"]
    if own:
        opt, held = st["opt"], st["held"]
        opt.step()
        m, v = opt.moments(0) if case["bits"] == 8 else (held["exp_avg"], held["exp_avg_sq"])
        return dict(p=st["p"], m=m, v=v, step=held["step"])
    with torch.no_grad():
        p, g = st["p"].float(), st["g"].float()
        if case["clip"]:
            g = g * (MAX_NORM / (_norm(st["g"]) + 1e-6)).clamp(max=1.0)
        st["step"] += 1
        t = st["step"][0].double()
        size = (LR / (1 - torch.exp2(t * math.log2(BETA1)))).float()
        root = (1 / (1 - torch.exp2(t * math.log2(BETA2))).sqrt()).float()
        if case["bits"] == 8:
            shape = st["m"].shape
            p, g = p.view(shape), g.view(shape)
            m = _unpack(st["m"], st["ms"], 3)
            s = _unpack(st["v"], st["vs"], 4)
            v = s * s
        else:
            m, v = st["m"], st["v"]
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + (g * g) * (1 - BETA2)
        new = p * (1 - LR * DECAY) - m / (v.sqrt() * root + ADAM_EPS) * size
        st["p"].copy_(new.view(-1))
        if case["bits"] == 8:
            st["m"], st["ms"] = _pack(m, _dither(st["index"], st["step"][:1], 0), 3)
            st["v"], st["vs"] = _pack(v.sqrt(), _dither(st["index"], st["step"][:1], 1), 4)
            m, s = _unpack(st["m"], st["ms"], 3), _unpack(st["v"], st["vs"], 4)
            v = s * s
        else:
            st["m"], st["v"] = m, v
        return dict(p=st["p"], m=m.view(-1), v=v.view(-1), step=st["step"])


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------
def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] in ("ln", "ln2"):
        n = case["rows"] * case["width"]
        if case["op"] == "ln":   # x, g in; y, dx out
            return dict(bytes=4 * n * size + 16 * case["width"], flops=n * (36 if case["act"] else 20))
        # x, g, u in; y, dx and the gradients of g and x out
        return dict(bytes=7 * n * size + 16 * case["width"], flops=n * (80 if case["act"] else 45))
    n = sum(_sizes(case))
    if case["op"] == "gnorm":
        return dict(bytes=n * size, flops=2 * n)
    # parameter in and out, gradient in, both moments in and out (8-bit ones also out as their values)
    moments = 16 if case["bits"] == 32 else 4 + 8
    return dict(bytes=n * (3 * size + moments), flops=n * (18 if case["clip"] else 15))


# ------------------------------------------------------------------------------------------------
# the same from the definitions in 64 bits: autograd of the definition, and the update's formula
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("ln", "ln2"):
        x, w, b, g = (st[k].detach().double().requires_grad_(True) for k in ("x", "w", "b", "g"))
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        y = (x - mean) * torch.rsqrt(var + EPS) * w + b
        if case["act"]:
            y = y * torch.sigmoid(y)
        if case["op"] == "ln":
            dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
            return dict(y=y.detach(), dx=dx, dw=dw, db=db)
        (dx,) = torch.autograd.grad(y, x, g, create_graph=True)
        grads = torch.autograd.grad(dx, (g, x, w, b), st["u"].double(), allow_unused=True)
        gg, gx, gw, gb = (torch.zeros_like(q) if t is None else t for t, q in zip(grads, (g, x, w, b)))
        return dict(y=y.detach(), dx=dx.detach(), gg=gg, gx=gx, gw=gw, gb=gb)
    g = st["g"].double()
    if case["op"] == "gnorm":
        return dict(norm=torch.linalg.vector_norm(g))
    if case["clip"]:
        g = g * min(1.0, MAX_NORM / (float(torch.linalg.vector_norm(g)) + 1e-6))
    t = STEP0 + 1
    if case["bits"] == 8:
        m0 = _unpack(st["m"], st["ms"], 3).double().view(-1)
        v0 = _unpack(st["v"], st["vs"], 4).double().view(-1).square()
    else:
        m0, v0 = st["m"].double(), st["v"].double()
    m = torch.lerp(g, m0, BETA1)
    v = torch.lerp(g.square(), v0, BETA2)
    mhat, vhat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = st["p"].double() * (1 - LR * DECAY) - LR * mhat / (vhat.sqrt() + ADAM_EPS)
    held = case["bits"] == 8     # an 8-bit moment is rounded by the operator's own sequence
    return dict(p=p, m=None if held else m, v=None if held else v, step=None)
