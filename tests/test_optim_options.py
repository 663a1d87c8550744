"""What ``ubio_molfm_b200.optim.AdamW`` refuses: options that it does not have and values that it cannot take."""
import pytest
import torch

DEV = "cuda"


def _param(n, seed):
    gen = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV))
    p.grad = torch.randn(n, generator=gen).to(DEV)
    return p


def _twin(p):
    q = torch.nn.Parameter(p.detach().clone())
    q.grad = p.grad.clone()
    return q


def test_epsilons_below_the_normal_range_are_refused():
    """The update of an element without gradient would be 0 times an infinite reciprocal."""
    import ctypes
    from array import array

    from ubio_molfm_b200 import _lib
    from ubio_molfm_b200.optim import AdamW

    p = torch.nn.Parameter(torch.zeros(3))
    for eps in (1e-38, 1e-44, 5e-324):
        with pytest.raises(ValueError, match="eps"):
            AdamW([p], eps=eps)
    for eps in (0.0, 2.0 ** -126, 1e-8):
        AdamW([p], eps=eps)
    dev = ctypes.c_void_p(1 << 20)
    keep = [array("Q", [4096]), array("Q", [8192]), array("q", [10]), array("q", [0]), array("i", [0])]
    assert _lib.load().e2a_adamw_step(*[a.buffer_info()[0] for a in keep], 1, 0, 32, dev, dev, None, None, 256, dev,
                                      1e-3, None, 0.9, 0.999, 1e-40, 0.0, None, 0.0, dev, 1 << 12, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_the_smallest_epsilon(bits):
    """Elements without gradient keep their value, the others take the step of an eps below their roots' last place."""
    from ubio_molfm_b200.optim import AdamW

    p = _param(1000, 3)
    p.grad[::3] = 0
    q = _twin(p)
    before = p.detach().clone()
    AdamW([p], lr=1e-2, eps=2.0 ** -126, weight_decay=0.0, state_bits=bits).step()
    AdamW([q], lr=1e-2, eps=1e-30, weight_decay=0.0, state_bits=bits).step()
    assert torch.equal(p[::3], before[::3])
    assert float((p - q).detach().abs().max()) <= 16 * 2.0 ** -24 * 4       # |p| + |update| <= 4 here
