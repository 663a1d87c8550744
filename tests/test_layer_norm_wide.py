"""Layer norm's backward and second order at 4,097 to 8,192 columns (``ubio_molfm_b200.norm``), the widest rows that teams
of threads hold in registers, with ``test_layer_norm``'s restatement and tolerances."""
import pytest
import torch
from test_layer_norm import _close, _inputs, _majorants, _run, reference


@pytest.mark.gpu
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,width", [(7, 4104), (5, 5000), (5, 6001), (300, 6001), (6, 8192), (400, 8192)])
def test_gradients_from_4097_to_8192_columns(rows, width, dtype, silu):
    x, w, b, g, u, p, q = _inputs(rows, width, dtype)
    ref, major = reference(x, w, b, silu, g, u, p, q), _majorants(x, w, b, g, u, p, q)
    first = _run(x, w, b, silu, g)
    for k, t in first.items():
        _close(t, ref[k], major[k], k)
    got = _run(x, w, b, silu, g, (u, p, q))
    for k, t in got.items():
        _close(t, ref[k], major[k], k)
        assert k not in first or torch.equal(t, first[k]), k
    if rows > 100:
        again = _run(x, w, b, silu, g, (u, p, q))
        assert all(torch.equal(got[k], again[k]) for k in got)
