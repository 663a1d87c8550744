"""Layer norm for training: ``act(LayerNorm(x) * weight + bias)`` with every gradient, to second order.

:func:`layer_norm` is what ``nn.LayerNorm`` (followed by ``nn.SiLU``, module_utils.py:2151-2178, 2240-2274)
computes in the radial and scalar MLPs.  Beside it, :func:`ubio_molfm_b200.linear.ln_silu` is the eval-mode
form (constant weights, first order).  The backward gives the input's, weight's and bias's gradients, and
is itself differentiable once, as a loss on forces = -dE/dpos needs (``create_graph=True``).
"""
from __future__ import annotations

from . import _lib

_ACTIVATIONS = {None: 0, "silu": 1}


def layer_norm(x, weight=None, bias=None, eps=1e-5, activation=None):
    """``act((x - mean) / sqrt(var + eps) * weight + bias)`` over the last dimension (biased variance).

    ``x`` [..., width] in float32, bfloat16 or float16 on CUDA, any strides; ``weight`` / ``bias`` [width] in
    float32 or x's dtype, or None (1 / 0); ``activation`` None or ``"silu"``.  The result is contiguous in
    x's dtype, the arithmetic fp32 with one rounding at the end.  Differentiable twice in x, weight and bias
    (a third order raises); column gradients that a backward does not reach are not formed.  Gradients are
    bitwise reproducible."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation={activation!r}: expected None or 'silu'")
    return _lib.load_torch().e2a_layer_norm(x, weight, bias, eps, _ACTIVATIONS[activation])
