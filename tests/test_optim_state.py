"""What ``ubio_molfm_b200.optim.AdamW`` does with parameters and states that change between its steps."""
import collections
import copy

import pytest
import torch

DEV = "cuda"


def _param(n, seed, grad=None):
    gen = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(n, generator=gen).to(DEV))
    p.grad = (torch.randn(n, generator=gen) if grad is None else torch.full((n,), grad)).to(DEV)
    return p


def _twin(p):
    q = torch.nn.Parameter(p.detach().clone())
    q.grad = p.grad.clone()
    return q


def _pair(sizes, bits, seed=0, **kw):
    from ubio_molfm_b200.optim import AdamW

    ps = [_param(n, seed + k) for k, n in enumerate(sizes)]
    return ps, AdamW(ps, lr=1e-2, state_bits=bits, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_replaced_parameter_starts_anew(bits):
    from ubio_molfm_b200.optim import AdamW

    ps, opt = _pair([300, 500, 70], bits)
    opt.step()
    opt.step()
    new = _param(500, 50)
    same, other = _twin(new), _twin(ps[0])
    fresh = AdamW([same], lr=1e-2, state_bits=bits)
    held = {k: t.clone() for k, t in opt.state[ps[0]].items()}
    opt.param_groups[0]["params"][1] = new
    opt.step()
    fresh.step()
    assert torch.equal(new, same) and int(opt.state[new]["step"]) == 1
    for k in fresh.state[same]:
        assert torch.equal(opt.state[new][k], fresh.state[same][k]), k
    # the others went on from where they were
    assert int(opt.state[ps[0]]["step"]) == 3 and int(opt.state[ps[2]]["step"]) == 3
    cont = AdamW([other], lr=1e-2, state_bits=bits)
    for k, t in cont._group_state(0).view(0, other).items():
        t.copy_(held[k])
    cont.step()
    assert torch.equal(other, ps[0])
    del opt.state[ps[1]]                             # the state of a parameter that is no longer there
    assert new in opt.state and len(opt.state_dict()["state"]) == 3
    opt.step()
    assert int(opt.state[new]["step"]) == 2 and int(opt.state[ps[0]]["step"]) == 4


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["clear", "new dict", "del", "pop", "empty entry"])
def test_a_cleared_state_starts_anew(bits, how):
    from ubio_molfm_b200.optim import AdamW

    ps, opt = _pair([300, 500], bits)
    opt.step()
    opt.step()
    gone = ps if how in ("clear", "new dict") else ps[1:]
    if how == "clear":
        opt.state.clear()
    elif how == "new dict":
        opt.state = collections.defaultdict(dict)
    elif how == "del":
        del opt.state[ps[1]]
    elif how == "pop":
        opt.state.pop(ps[1])
    else:
        opt.state[ps[1]] = {}
    twins = [_twin(p) for p in gone]
    fresh = AdamW(twins, lr=1e-2, state_bits=bits)
    opt.step()
    fresh.step()
    for p, q in zip(gone, twins):
        assert torch.equal(p, q) and int(opt.state[p]["step"]) == 1
        for k in fresh.state[q]:
            assert torch.equal(opt.state[p][k], fresh.state[q][k]), k
    assert int(opt.state[ps[0]]["step"]) == (1 if len(gone) == 2 else 3)
    opt.step()
    fresh.step()
    assert all(torch.equal(p, q) for p, q in zip(gone, twins))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_groups_removed_and_reordered(bits):
    """Two groups of like sizes that change places, and one that goes: every parameter keeps its own moments."""
    from ubio_molfm_b200.optim import AdamW

    ps = [_param(400, k) for k in range(3)]
    qs = [_twin(p) for p in ps]
    opt, ref = (AdamW([dict(params=[t], lr=10.0 ** -(2 + k)) for k, t in enumerate(ts)], state_bits=bits)
                for ts in (ps, qs))
    opt.step()
    ref.step()
    opt.param_groups.reverse()
    del opt.param_groups[1]
    opt.step()
    ref.step()
    assert torch.equal(ps[0], qs[0]) and torch.equal(ps[2], qs[2]) and not torch.equal(ps[1], qs[1])
    for p, q in ((ps[0], qs[0]), (ps[2], qs[2])):
        for k in ref.state[q]:
            assert torch.equal(opt.state[p][k], ref.state[q][k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_replaced_state_tensors_are_used(bits):
    ps, opt = _pair([300, 40], bits)
    opt.step()
    copy_of = {k: t.clone() for k, t in opt.state[ps[0]].items()}
    opt.step()
    for k, t in copy_of.items():
        opt.state[ps[0]][k] = t
    opt.step()
    assert int(opt.state[ps[0]]["step"]) == 2 and int(opt.state[ps[1]]["step"]) == 3
    opt.state[ps[0]]["exp_avg"] = torch.zeros(7, device=DEV)
    with pytest.raises(ValueError, match="state"):
        opt.step()


@pytest.mark.gpu
def test_a_list_that_grows_or_shrinks():
    ps, opt = _pair([30, 40], 32)
    opt.step()
    late = _param(50, 9)
    opt.param_groups[0]["params"].append(late)
    opt.step()
    assert int(opt.state[late]["step"]) == 1 and int(opt.state[ps[0]]["step"]) == 2
    del opt.param_groups[0]["params"][0]
    before = ps[0].detach().clone()
    opt.step()
    assert torch.equal(ps[0], before) and int(opt.state[ps[1]]["step"]) == 3 and int(opt.state[late]["step"]) == 2


@pytest.mark.gpu
def test_a_saved_state_of_other_shapes_is_refused():
    from ubio_molfm_b200.optim import AdamW

    ps, opt = _pair([600, 30], 8)
    opt.step()
    for key in ("exp_avg_scale", "exp_avg_sq_scale", "step"):
        held = copy.deepcopy(opt.state_dict())
        held["state"][0][key] = held["state"][0][key].reshape(-1)[:1] if key != "step" else torch.ones(2)
        other = AdamW(ps, lr=0.5, state_bits=8)
        with pytest.raises(ValueError, match="shape"):
            other.load_state_dict(held)
        assert other.param_groups[0]["lr"] == 0.5 and not other.state


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("when", ["new", "cleared"])
def test_state_is_not_made_inside_a_capture(bits, when):
    """Its zeros would be captured and every replay would start from them."""
    ps, opt = _pair([300, 20], bits)
    if when == "cleared":
        opt.step()
        opt.state.clear()
    before = [p.detach().clone() for p in ps]
    with pytest.raises(RuntimeError, match="flat_state"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, b) for p, b in zip(ps, before))
    opt.flat_state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for t in (1, 2):
        graph.replay()
        assert int(opt.state[ps[0]]["step"]) == t


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("how", ["clear", "entry", "load", "swap"])
def test_a_captured_step_stays_good_when_the_state_is_laid_out_again(bits, how):
    """The state of the same parameters keeps its memory: replays go on from what it was set to."""
    ps, opt = _pair([300, 300, 20], bits)
    qs, eager = _pair([300, 300, 20], bits)
    opt.flat_state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    graph.replay()
    for _ in range(2):
        eager.step()
    at = {k: t.data_ptr() for k, t in opt.flat_state().items()}
    for o, ts in ((opt, ps), (eager, qs)):
        if how == "clear":
            o.state.clear()
        elif how == "entry":
            o.state[ts[1]] = {}
        elif how == "swap":
            o.state[ts[0]], o.state[ts[1]] = o.state[ts[1]], o.state[ts[0]]
        else:
            saved = copy.deepcopy(o.state_dict())
            o.step() if o is eager else graph.replay()
            o.load_state_dict(saved)
        held = o.flat_state()
        assert not (how == "clear" and any(bool(t.any()) for t in held.values()))
        if o is opt:
            assert at == {k: t.data_ptr() for k, t in held.items()}
    graph.replay()
    eager.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        for k in eager.state[q]:
            assert torch.equal(opt.state[p][k], eager.state[q][k]), k
