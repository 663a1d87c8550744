"""The operators of a training step together: layer norm inside the model's force-loss training, the clipped
AdamW step, and ``E2FormerModelInterface.train_step`` that runs them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

SMALL = dict(irreps_node_embedding="32x0e+32x1e+32x2e", num_layers=2, max_neighbors=None, max_radius=5.0,
             number_of_basis=32, num_attn_heads=8, attn_scalar_head=8, irreps_head="4x0e+4x1e+4x2e",
             norm_layer="rms_norm_sh", alpha_drop=0.0, tp_type="QK_alpha", attn_type="so2-first-order",
             atom_type_cnt=256, avg_degree=23.0)


def _potential(fused, seed=31):
    from ubio_molfm_b200.model import E2FormerPotential
    from ubio_molfm_b200.synthetic import seeded_params_

    pot = E2FormerPotential(fused_layer_norm=fused, **SMALL)
    seeded_params_(pot.decoder, seed)
    seeded_params_(pot.energy_head, seed + 1)
    return pot.to(DEV)


def _box(seed=12, n=40, L=7.0):
    rng = np.random.default_rng(seed)
    return (rng.random((n, 3)) * L).astype(np.float32), rng.choice([1, 6, 7, 8], n), np.eye(3, dtype=np.float32) * L


def _molecules():
    from ubio_molfm_b200.interface import collate_systems

    rng = np.random.default_rng(5)
    systems = []
    for n in (7, 12, 1, 9):
        systems.append(dict(atoms=rng.choice([1, 6, 8], n), coords=rng.random((n, 3)) * 4 + 1, charge=0, multiplicity=1))
    return collate_systems(systems, device=DEV)


def test_fused_layer_norm_gives_the_training_gradients():
    """Parameter gradients of E^2 + sum |F|^2 with and without the fused layer norm.  Either is held to 1e-4 of
    each parameter's largest entry against the 64-bit model (test_double_backward.py), so they differ by at most
    2e-4."""
    pos, Z, cell = _box()
    grads = []
    for fused in (False, True):
        pot = _potential(fused).train()
        energy, forces = pot(torch.tensor(pos, device=DEV), torch.tensor(Z, device=DEV), torch.tensor(cell), (True,) * 3)
        (energy.square().sum() + forces.square().sum()).backward()
        grads.append({k: p.grad for k, p in pot.named_parameters() if p.grad is not None})
    assert grads[0].keys() == grads[1].keys() and any("net.1.weight" in k for k in grads[0])
    for k, a in grads[0].items():
        b = grads[1][k]
        assert float((a - b).abs().max()) <= 2e-4 * max(float(a.abs().max()), 1e-12), k


def test_fused_layer_norm_leaves_eval_mode_alone():
    pos, Z, cell = _box()
    out = [_potential(f).eval()(torch.tensor(pos, device=DEV), torch.tensor(Z, device=DEV), torch.tensor(cell),
                                (True,) * 3) for f in (False, True)]
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


@pytest.mark.parametrize("bits", [32, 8])
def test_train_step(bits):
    """One step equals its parts done by hand: loss, gradients, the clipping norm and AdamW's first update (lr
    sign(g) where |g| is far from eps, weights decayed), and eval mode sees the new weights."""
    from ubio_molfm_b200.interface import E2FormerModelInterface
    from ubio_molfm_b200.model import E2FormerPotential
    from ubio_molfm_b200.optim import AdamW

    batch = _molecules()
    gen = torch.Generator().manual_seed(3)
    energy, forces = torch.randn(4, generator=gen), 0.1 * torch.randn(*batch["pos"].shape, generator=gen)
    pot = _potential(True)
    iface = E2FormerModelInterface(model=pot, device=DEV)
    opt = AdamW(pot.parameters(), lr=1e-3, weight_decay=0.01, state_bits=bits, max_grad_norm=0.5)
    iface.predict(batch)                               # fills eval mode's caches of merged weights
    before = {k: p.detach().clone() for k, p in pot.named_parameters()}
    loss = iface.train_step(batch, energy, forces, opt, energy_weight=2.0, force_weight=3.0)
    assert not pot.training and loss.shape == () and not loss.requires_grad

    # by hand, on a copy with the old weights
    ref = _potential(True)
    ref.load_state_dict({**ref.state_dict(), **before})
    ri = E2FormerModelInterface(model=ref, device=DEV)
    ref.train()
    out = ri.predict(batch)
    n = batch["atom_masks"].sum(-1)
    de = (out["pred_energy"] - energy.to(DEV)) / n
    df = (out["pred_forces"] - forces.to(DEV))[batch["atom_masks"]]
    want = 2.0 * de.square().mean() + 3.0 * df.square().sum(-1).mean()
    want.backward()
    # the batch's energies are summed by atomics: a few fp32 units (2^-24) of either
    assert abs(float(loss) - float(want.detach())) <= 1e-5 * float(want.detach())
    grads = {k: p.grad for k, p in ref.named_parameters() if p.grad is not None}
    norm = torch.sqrt(sum(g.double().square().sum() for g in grads.values()))
    assert abs(float(opt.last_grad_norm) - float(norm)) <= 1e-4 * float(norm)
    coef = min(1.0, 0.5 / (float(norm) + 1e-6))
    moved = 0
    for k, p in pot.named_parameters():
        if k not in grads:
            assert torch.equal(p.detach(), before[k]), k
            continue
        g = grads[k] * coef
        sure = g.abs() > 1e-3 * g.abs().max() + 1e-6    # elements whose gradient is known to 1e-4 of the largest
        step = before[k] * (1 - 1e-3 * 0.01) - p.detach()
        # lr |g| / (|g| + eps): within eps / |g| <= 1e-2 and the gradient's own 10 % of lr
        assert bool(((step[sure] - 1e-3 * g[sure].sign()).abs() <= 1e-4 + 1e-6 * before[k][sure].abs()).all()), k
        moved += int(sure.sum())
    assert moved > 1000

    # eval mode after the step: the same as a model that was built with the new weights
    fresh = E2FormerPotential(**SMALL).to(DEV)
    fresh.load_state_dict(pot.state_dict())
    a, b = iface.predict(batch), E2FormerModelInterface(model=fresh, device=DEV).predict(batch)
    assert torch.equal(a["pred_forces"], b["pred_forces"])


def test_train_step_runs_on_and_refuses_bad_targets():
    from ubio_molfm_b200.interface import E2FormerModelInterface, collate_systems
    from ubio_molfm_b200.optim import AdamW

    batch = _molecules()
    pot = _potential(True)
    iface = E2FormerModelInterface(model=pot, device=DEV)
    opt = AdamW(pot.parameters(), lr=1e-4, state_bits=8, max_grad_norm=10.0)
    zero_e, zero_f = torch.zeros(4), torch.zeros_like(batch["pos"])
    box = collate_systems([dict(atoms=_box()[1], coords=_box()[0], cell=_box()[2], pbc=[True] * 3)], device=DEV)
    assert bool(torch.isfinite(iface.train_step(box, torch.zeros(1), torch.zeros_like(box["pos"]), opt)))    # periodic
    for _ in range(3):
        assert bool(torch.isfinite(iface.train_step(batch, zero_e, zero_f, opt)))
    for bad_e, bad_f in ((torch.zeros(3), zero_f), (torch.zeros(1), zero_f), (zero_e, zero_f[:, :5]), (zero_e, zero_f[0])):
        with pytest.raises(ValueError, match="targets"):
            iface.train_step(batch, bad_e, bad_f, opt)
    assert not pot.training
    # targets that are not finite: the step is left out, weights and states stay
    held = [p.detach().clone() for p in pot.parameters()] + [t.clone() for t in opt.flat_state().values()]
    iface.train_step(batch, torch.full((4,), float("nan")), zero_f, opt)
    now = [p.detach() for p in pot.parameters()] + list(opt.flat_state().values())
    assert all(torch.equal(x, y) for x, y in zip(held, now))
