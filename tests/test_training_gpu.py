"""The training operators together, as a training uses them: a model with block norms, its force loss
and gradients on the kernels, and AdamW over all its weights."""
import pytest
import torch

from _util import assert_close
from oracle import adamw_oracle
from test_model_gpu import brute_neighbors, random_system

pytestmark = pytest.mark.gpu


def build(channels, lmax, layers, seed=5, **kwargs):
    from mace_ictc.models import MACEICTC
    from oracle.model_ops import OracleOps
    torch.manual_seed(seed)
    options = dict(channels=channels, lmax=lmax, num_interactions=layers, avg_num_neighbors=10.0, block_norm=True,
                   block_scale=0.7, **kwargs)
    model = MACEICTC(**options)
    with torch.no_grad():
        for norm in [*model.block_norms, model.input_norm]:
            for p in norm.parameters():
                p.mul_(1 + 0.2 * torch.randn_like(p))
    twin = MACEICTC(**options, ops=OracleOps())
    twin.load_state_dict(model.state_dict())
    return model, twin.double()


def batch_of(graphs, device, dtype):
    """Positions, atomic numbers and a block-diagonal graph of several periodic cells."""
    parts, offset = [], 0
    for k, n in enumerate(graphs):
        pos, species, side = random_system(n, seed=40 + k)
        src, dst, shift = brute_neighbors(pos, side, 5.0)
        cell = torch.eye(3, dtype=torch.float64) * side
        parts.append((pos, torch.tensor([1, 6, 8])[species], torch.full((n,), k), src + offset, dst + offset,
                      torch.round(shift / side), cell.unsqueeze(0)))
        offset += n
    out = [torch.cat(x).to(device) for x in zip(*parts)]
    return [x.to(dtype) if x.is_floating_point() else x for x in out]


@pytest.mark.parametrize("lmax, layers", [(1, 2), (2, 3), (3, 2)])
def test_forces_and_force_loss_gradients_match_oracle(lmax, layers, cuda_device):
    pos, species, side = random_system(26, seed=60 + lmax)
    src, dst, shift = brute_neighbors(pos, side, 5.0)
    model, twin = build(16, lmax, layers)
    model = model.to(cuda_device)
    gen = torch.Generator().manual_seed(1)
    target = torch.randn(26, 3, generator=gen, dtype=torch.float64)

    def run(m, p, sp, s, d, sh, t):
        energy, forces = m.energy_and_forces(p, sp, s, d, sh, training=True)
        loss = energy.square().sum() / 26 ** 2 + 100.0 * (forces - t).square().mean()
        names, params = zip(*[(n, p) for n, p in m.named_parameters() if p.requires_grad])
        return energy, forces, dict(zip(names, torch.autograd.grad(loss, params, allow_unused=True)))

    dev = cuda_device
    e, f, g = run(model, pos.float().to(dev), species.to(dev), src.to(dev), dst.to(dev), shift.float().to(dev),
                  target.float().to(dev))
    re, rf, rg = run(twin, pos, species, src, dst, shift, target)
    # as the tests of the model without block norms
    assert_close(e.detach().cpu(), re.detach(), 1e-5, None, "energy")
    assert_close(f.detach().cpu(), rf.detach(), 1e-4, 1e-3, "forces")
    for name, want in rg.items():
        if want is None:
            assert g[name] is None or float(g[name].abs().max()) == 0.0, name
        else:
            assert_close(g[name].cpu(), want, 1e-4, None, name)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(bits, cuda_device):
    """Each step moves every weight as the optimizer's formula says for the gradients of that step, the loss is
    finite, and the model computes with the new weights."""
    import copy
    from mace_ictc.runtime import configure_model, energy_and_forces
    from mace_ictc.training import create_optimizer, force_loss, train_step
    model, _ = build(16, 2, 2)
    model = model.to(cuda_device)
    configure_model(model)
    args = batch_of([20, 31], cuda_device, torch.float32)
    gen = torch.Generator(device=cuda_device).manual_seed(3)
    targets = (torch.randn(2, device=cuda_device, generator=gen), torch.randn(51, 3, device=cuda_device, generator=gen))
    opt = create_optimizer(model, lr=2e-3, state_bits=bits, max_norm=5.0, skip_nonfinite=True, ema_decay=0.9, seed=11)
    assert [len(g["params"]) for g in opt.param_groups][1] == 6 and opt.param_groups[1]["weight_decay"] == 0.0
    for step in range(3):
        starts = dict(zip([p for g in opt.param_groups for p in g["params"]], opt._table.starts))
        m, v = (x.double() for x in opt.moments())
        old = {p: (p.detach().double(), m[s:s + p.numel()].view(p.shape), v[s:s + p.numel()].view(p.shape))
               for p, s in starts.items()}
        loss = train_step(model, opt, *args, *targets)
        assert torch.isfinite(loss)
        norm = torch.cat([p.grad.double().reshape(-1) for p in old]).norm()
        clip = min(1.0, 5.0 / (float(norm) + 1e-6))
        for group in opt.param_groups:
            hyper = {k: group[k] for k in ("lr", "betas", "eps", "weight_decay")}
            for p in group["params"]:
                w0, m0, v0 = old[p]
                each = (w0, p.grad.double(), m0, v0, step + 1)
                want = adamw_oracle.step(*each, **hyper, clip=clip)[0]
                bound = adamw_oracle.step_bounds(*each, **hyper, clip=clip, clipped=True, approximate=bits == 8)[0]
                assert int(opt.state[p]["step"]) == step + 1
                assert bool(((p.detach().double() - want).abs() <= bound).all())
        with torch.no_grad():
            now = energy_and_forces(model, *args)
            again = energy_and_forces(copy.deepcopy(model), *args)
        # (sums over graphs and edges outside these operators add in any order)
        assert torch.equal(now["atomic_energy"], again["atomic_energy"])
    result = energy_and_forces(model, *args, training=True)
    assert torch.isfinite(force_loss(result, args[2], *targets))
