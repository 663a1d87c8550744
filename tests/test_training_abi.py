"""The training operators' C entry points refuse addresses that their kernels could not read or write: every check is on
the host, before any device work, so the addresses are never touched."""
import ctypes
from array import array

import pytest

OK = 1 << 20
ARG = 1


def at(address):
    return ctypes.c_void_p(address) if address else None


def _lib():
    from ubio_molfm_b200 import _lib

    return _lib.load()


@pytest.mark.parametrize("dtype,odd", [(0, 2), (1, 1), (2, 1)])
def test_layer_norm(dtype, odd):
    lib = _lib()
    rows = OK + odd

    def fwd(x=OK, gamma=0, beta=0, y=OK, mean=OK, rstd=OK):
        return lib.e2a_layer_norm_fwd(at(x), 8, dtype, at(gamma), at(beta), 4, 8, 1e-5, 0, at(y), at(mean), at(rstd), None)

    for bad in (dict(x=rows), dict(y=rows), dict(gamma=OK + 2), dict(beta=OK + 1), dict(mean=OK + 2), dict(rstd=OK + 2)):
        assert fwd(**bad) == ARG, bad

    def bwd(x=OK, dy=OK, gamma=0, mean=OK, rstd=OK, dx=OK, dgamma=OK, dbeta=OK, ws=OK):
        return lib.e2a_layer_norm_bwd(at(x), 8, at(dy), 8, dtype, at(gamma), None, at(mean), at(rstd), 4, 8, 0, at(dx),
                                      at(dgamma), at(dbeta), at(ws), 1 << 20, None)

    for bad in (dict(x=rows), dict(dy=rows), dict(dx=rows), dict(gamma=OK + 2), dict(mean=OK + 2), dict(rstd=OK + 1),
                dict(dgamma=OK + 2), dict(dbeta=OK + 2), dict(ws=OK + 8)):
        assert bwd(**bad) == ARG, bad

    def bwd2(x=OK, dy=OK, u=OK, p=0, q=0, d_dy=OK, dx=OK, dgamma=OK, ws=OK):
        return lib.e2a_layer_norm_bwd2(at(x), 8, at(dy), 8, at(u), 8, dtype, None, None, at(OK), at(OK), at(p), at(q), 4, 8,
                                       0, at(d_dy), at(dx), at(dgamma), None, at(ws), 1 << 20, None)

    for bad in (dict(x=rows), dict(dy=rows), dict(u=rows), dict(d_dy=rows), dict(dx=rows), dict(p=OK + 2), dict(q=OK + 2),
                dict(dgamma=OK + 2), dict(ws=OK + 8)):
        assert bwd2(**bad) == ARG, bad


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_and_its_moments(bits):
    lib = _lib()
    tables = [array("Q", [4096]), array("Q", [8192]), array("q", [10]), array("q", [0]), array("i", [0])]

    def step(m=OK, v=OK, count=OK, lr=0, norm=0, ws=OK):
        return lib.e2a_adamw_step(*[t.buffer_info()[0] for t in tables], 1, 0, bits, at(m), at(v), at(OK), at(OK), 256,
                                  at(count), 1e-3, at(lr), 0.9, 0.999, 1e-8, 0.0, at(norm), 1.0, at(ws), 1 << 12, None)

    off = 8 if bits == 32 else 2
    for bad in (dict(m=OK + off), dict(v=OK + off), dict(count=OK + 2), dict(lr=OK + 2), dict(norm=OK + 2), dict(ws=OK + 8)):
        assert step(**bad) == ARG, bad

    def unpack(m=OK, v=OK, a=OK, b=OK):
        return lib.e2a_moments_unpack(at(m), at(v), at(OK), at(OK), 256, at(a), at(b), None)

    for bad in (dict(m=OK + 2), dict(v=OK + 1), dict(a=OK + 4), dict(b=OK + 8)):
        assert unpack(**bad) == ARG, bad


def test_gradient_norm():
    lib = _lib()
    t, n, count = array("Q", [4096]), array("q", [7]), array("q", [0])
    where = t.buffer_info()[0], n.buffer_info()[0]
    assert lib.e2a_sum_squares(*where, 1, 0, at(OK + 4), 1 << 20, count.buffer_info()[0], None) == ARG
    assert lib.e2a_norm_of_squares(at(OK + 4), 4, at(OK), None) == ARG
    assert lib.e2a_norm_of_squares(at(OK), 4, at(OK + 2), None) == ARG
    assert lib.e2a_grad_norm(*where, 1, 0, at(OK + 4), 1 << 20, at(OK), None) == ARG
