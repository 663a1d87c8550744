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


@pytest.mark.parametrize("option", [dict(maximize=True), dict(amsgrad=True), dict(differentiable=True),
                                    dict(decoupled_weight_decay=False), dict(state_bits=8), dict(max_grad_norm=1.0)])
def test_options_that_it_does_not_have_are_refused(option):
    from ubio_molfm_b200.optim import AdamW

    p, q = (torch.nn.Parameter(torch.zeros(3)) for _ in range(2))
    with pytest.raises(ValueError, match=next(iter(option))):
        AdamW([dict(params=[p], **option)])
    opt = AdamW([p])
    with pytest.raises(ValueError, match=next(iter(option))):
        opt.add_param_group(dict(params=[q], **option))
    assert len(opt.param_groups) == 1
    held = opt.state_dict()
    held["param_groups"][0].update(option)
    with pytest.raises(ValueError, match=next(iter(option))):
        opt.load_state_dict(held)
    opt.param_groups[0].update(option)
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match=next(iter(option))):
        opt.step()


def test_options_that_change_nothing_are_taken():
    """PyTorch's own AdamW state without them set, a scheduler's keys, a user's own."""
    from ubio_molfm_b200.optim import AdamW

    p = torch.nn.Parameter(torch.zeros(3))
    theirs = torch.optim.AdamW([p], lr=0.5)
    opt = AdamW([dict(params=[p], name="head", initial_lr=1e-3)])
    opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5
    opt.step()


@pytest.mark.gpu
def test_a_refused_learning_rate_leaves_all_groups_as_they_were():
    from ubio_molfm_b200.optim import AdamW

    ps = [_param(30, 1), _param(40, 2)]
    opt = AdamW([dict(params=[ps[0]]), dict(params=[ps[1]], lr=torch.tensor(1e-3, dtype=torch.float64, device=DEV))])
    before, versions = [p.detach().clone() for p in ps], [p._version for p in ps]
    with pytest.raises(ValueError, match="lr"):
        opt.step()
    assert all(torch.equal(p, b) for p, b in zip(ps, before)) and int(opt.flat_state(0)["step"]) == 0
    assert ps[1]._version == versions[1]
