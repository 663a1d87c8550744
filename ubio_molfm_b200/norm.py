"""Layer norm for training: ``act(LayerNorm(x) * weight + bias)`` with every gradient, to second order.

:func:`layer_norm` is what ``nn.LayerNorm`` (followed by ``nn.SiLU``, module_utils.py:2151-2178, 2240-2274)
computes in the radial and scalar MLPs.  Beside it, :func:`ubio_molfm_b200.linear.ln_silu` is the eval-mode
form (constant weights, first order).  The backward gives the input's, weight's and bias's gradients, and
is itself differentiable once, as a loss on forces = -dE/dpos needs (``create_graph=True``).
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check, require_cuda, stream_of

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTIVATIONS = {None: 0, "silu": 1}


def _rows(t, width):
    """``t`` as [rows, width] with unit inner stride, and its row stride (a copy only where no such view
    exists; rows that repeat, stride 0, are read in place)."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if width > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _f32(t):
    """A contiguous fp32 vector (itself where it is one) and its address; None stays None."""
    if t is None:
        return None, None
    if t.dtype != torch.float32 or not t.is_contiguous():
        t = t.contiguous().to(torch.float32)
    return t, t.data_ptr()


def _columns(lib_bytes, rows, width, dev):
    """Storage of a column-sum pass: (dw, db) [width] fp32 and the workspace."""
    dw, db = torch.empty((2, width), dtype=torch.float32, device=dev).unbind(0)
    ws = torch.empty(max(lib_bytes(rows, width), 1), dtype=torch.uint8, device=dev)
    return dw, db, ws


def _backward(x, g, weight, bias, stats, act, need_x, need_cols):
    """``(dx, dw, db)`` of rows: dx in x's dtype (or None), dw / db [width] in fp32 (or None)."""
    lib = _lib.load()
    width, dev = x.shape[-1], x.device
    x2, ldx = _rows(x, width)
    g2, ldg = _rows(g, width)
    rows = x2.shape[0]
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    dw = db = ws = None
    if need_cols:
        dw, db, ws = _columns(lib.e2a_layer_norm_bwd_workspace_bytes, rows, width, dev)
    w, w_at = _f32(weight)
    b, b_at = _f32(bias)
    at = stats.data_ptr()
    check(lib.e2a_layer_norm_bwd(x2.data_ptr(), ldx, g2.data_ptr(), ldg, _DTYPES[x.dtype], w_at, b_at, at,
                                 at + 4 * rows, rows, width, act, dx.data_ptr() if need_x else None,
                                 dw.data_ptr() if need_cols else None, db.data_ptr() if need_cols else None,
                                 ws.data_ptr() if need_cols else None, ws.numel() if need_cols else 0,
                                 stream_of(dev)), "e2a_layer_norm_bwd")
    return dx, dw, db


def _cast(t, like):
    if t is None or like is None:
        return None
    return t if like.dtype == torch.float32 else t.to(like.dtype)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, act):
        lib = _lib.load()
        width, dev = x.shape[-1], x.device
        x2, ldx = _rows(x, width)
        rows = x2.shape[0]
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        stats = torch.empty((2, rows), dtype=torch.float32, device=dev)
        w, w_at = _f32(weight)
        b, b_at = _f32(bias)
        at = stats.data_ptr()
        check(lib.e2a_layer_norm_fwd(x2.data_ptr(), ldx, _DTYPES[x.dtype], w_at, b_at, rows, width, eps, act,
                                     y.data_ptr(), at, at + 4 * rows, stream_of(dev)), "e2a_layer_norm_fwd")
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, g):
        x, weight, bias, stats = ctx.saved_tensors
        if torch.is_grad_enabled():
            # create_graph=True: the backward as an op of its own, with the second-order kernel behind it
            dx, dw, db = _LayerNormBackwardFn.apply(g, x, weight, bias, stats, ctx.act)
            return dx, dw, db, None, None
        need = ctx.needs_input_grad
        dx, dw, db = _backward(x, g, weight, bias, stats, ctx.act, need[0], need[1] or need[2])
        return dx, _cast(dw, weight) if need[1] else None, _cast(db, bias) if need[2] else None, None, None


class _LayerNormBackwardFn(torch.autograd.Function):
    """``(dx, dw, db)`` of the layer norm at upstream gradient ``g`` as a differentiable op."""

    @staticmethod
    def forward(ctx, g, x, weight, bias, stats, act):
        ctx.set_materialize_grads(False)
        dx, dw, db = _backward(x, g, weight, bias, stats, act, True, weight is not None or bias is not None)
        ctx.save_for_backward(g, x, weight, bias, stats)
        ctx.act = act
        return dx, _cast(dw, weight), _cast(db, bias)

    @staticmethod
    def backward(ctx, u, p, q):
        if torch.is_grad_enabled():
            raise RuntimeError("layer_norm: gradients of third and higher order are not supported")
        g, x, weight, bias, stats = ctx.saved_tensors
        if u is None and p is None and q is None:
            return None, None, None, None, None, None
        lib = _lib.load()
        width, dev = x.shape[-1], x.device
        if u is None:
            u = torch.zeros((), dtype=x.dtype, device=dev).expand(x.shape)
        x2, ldx = _rows(x, width)
        g2, ldg = _rows(g, width)
        u2, ldu = _rows(u, width)
        rows = x2.shape[0]
        (w, w_at), (b, b_at), (p, p_at), (q, q_at) = _f32(weight), _f32(bias), _f32(p), _f32(q)
        d_g = torch.empty(x.shape, dtype=x.dtype, device=dev)
        d_x = torch.empty(x.shape, dtype=x.dtype, device=dev)
        dw, db, ws = _columns(lib.e2a_layer_norm_bwd2_workspace_bytes, rows, width, dev)
        cols = ctx.needs_input_grad[2] or ctx.needs_input_grad[3]
        at = stats.data_ptr()
        check(lib.e2a_layer_norm_bwd2(x2.data_ptr(), ldx, g2.data_ptr(), ldg, u2.data_ptr(), ldu, _DTYPES[x.dtype],
                                      w_at, b_at, at, at + 4 * rows, p_at, q_at, rows, width, ctx.act, d_g.data_ptr(),
                                      d_x.data_ptr(), dw.data_ptr() if cols else None, db.data_ptr() if cols else None,
                                      ws.data_ptr(), ws.numel(), stream_of(dev)), "e2a_layer_norm_bwd2")
        return d_g, d_x, _cast(dw, weight) if cols else None, _cast(db, bias) if cols else None, None, None


def _check_affine(name, t, x):
    if t is None:
        return
    if t.dim() != 1 or t.shape[0] != x.shape[-1]:
        raise ValueError(f"{name} must be [{x.shape[-1]}], got {list(t.shape)}")
    if t.dtype not in (torch.float32, x.dtype):
        raise TypeError(f"{name} must be float32 or {x.dtype}, got {t.dtype}")
    if t.device != x.device:
        raise ValueError(f"{name} is on {t.device}, the input on {x.device}")


def layer_norm(x, weight=None, bias=None, eps=1e-5, activation=None):
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` over the last dimension (biased variance).

    ``x`` [..., width] in float32, bfloat16 or float16 on CUDA, any strides; ``weight`` / ``bias`` [width] in
    float32 or x's dtype, or None (1 / 0); ``activation`` None or ``"silu"``.  The result is contiguous in
    x's dtype, the arithmetic fp32 with one rounding at the end.  Differentiable twice in x, weight and bias
    (a third order raises).  Gradients are bitwise reproducible."""
    require_cuda(x, weight, bias)
    if x.dtype not in _DTYPES:
        raise TypeError(f"layer_norm takes float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm needs a last dimension of at least one value")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation={activation!r}: expected None or 'silu'")
    _check_affine("weight", weight, x)
    _check_affine("bias", bias, x)
    if x.device.index == torch.cuda.current_device():
        return _LayerNormFn.apply(x, weight, bias, float(eps), _ACTIVATIONS[activation])
    with torch.cuda.device(x.device):
        return _LayerNormFn.apply(x, weight, bias, float(eps), _ACTIVATIONS[activation])
