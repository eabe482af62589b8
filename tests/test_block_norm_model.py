"""Block norms inside the model and the training step around it (CPU, FP64 oracle operators)."""
import pytest
import torch


def _model(seed=0, layers=3, **kwargs):
    from mace_ictc.models import MACEICTC
    from oracle.model_ops import OracleOps
    torch.manual_seed(seed)
    model = MACEICTC(channels=4, lmax=2, num_interactions=layers, r_max=3.0, avg_num_neighbors=5.0, ops=OracleOps(),
                     **kwargs)
    return model.double()


def _system():
    from test_checkpoint import _system as system
    return system()


def test_models_without_block_norms_are_what_they_were():
    plain, again = _model(3), _model(3, block_norm=False)
    assert list(plain.state_dict()) == list(again.state_dict())
    normed = _model(3, block_norm=True)
    own = [n for n in normed.state_dict() if n not in plain.state_dict()]
    assert own and all(n.split(".")[0] in ("input_norm", "block_norms", "block_gates") for n in own)
    assert all(torch.equal(v, normed.state_dict()[n]) for n, v in plain.state_dict().items())


def test_energy_is_invariant_and_its_forces_match_differences():
    model = _model(1, block_norm=True, block_scale=0.5)
    pos, species, src, dst, shift = _system()
    energy, forces = model.energy_and_forces(pos, species, src, dst, shift)
    turn, _ = torch.linalg.qr(torch.randn(3, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(2)))
    e2, f2 = model.energy_and_forces(pos @ turn, species, src, dst, shift @ turn)
    # Without norms the model turns with its system to 2e-10 of its forces (the coupling tables' own
    # precision); each of three norms divides a branch by its size, here 0.01 to 0.1 for the first ones, so that
    # up to 1e3 times as much is left: 2e-7.  A form that did not turn would be off by the forces themselves.
    assert float((e2 - energy).detach().abs()) <= 2e-7 * float(energy.detach().abs().max() + forces.detach().norm())
    assert float((f2 - forces @ turn).detach().norm()) <= 2e-7 * float(forces.detach().norm())
    h = 1e-5
    for atom, axis in ((0, 0), (7, 2)):
        step = torch.zeros_like(pos)
        step[atom, axis] = h
        slope = (model.energy(pos + step, species, src, dst, shift)
                 - model.energy(pos - step, species, src, dst, shift)) / (2 * h)
        assert abs(float(-slope.detach() - forces[atom, axis].detach())) <= 1e-6 * max(1.0, float(forces.detach().abs().max()))


def test_normed_inputs_do_not_depend_on_the_embedding_scale():
    """What the norms are for: the first block's input keeps its size whatever the embedding's."""
    model = _model(2, block_norm=True)
    x = torch.randn(5, 4, dtype=torch.float64)
    torch.testing.assert_close(model._block_start(1000 * x), model._block_start(x), rtol=1e-6, atol=1e-6)


def test_refusals():
    from mace_ictc.checkpoint import check_reference_metadata, from_reference_state_dict, to_reference_state_dict
    with pytest.raises(ValueError, match="first_layer_self_connection"):
        _model(block_norm=True, first_layer_self_connection=False)
    model = _model(block_norm=True)
    for call in (lambda: to_reference_state_dict(model), lambda: from_reference_state_dict(model, {}),
                 lambda: check_reference_metadata(model, {})):
        with pytest.raises(ValueError, match="block norms"):
            call()


def test_loss_and_its_checks():
    from mace_ictc.training import force_loss
    energy, forces = torch.tensor([6.0, -2.0]), torch.zeros(5, 3)
    batch = torch.tensor([0, 0, 0, 1, 1])
    result = {"energy": energy, "forces": forces}
    loss = force_loss(result, batch, torch.tensor([1.0, 0.0]), torch.ones(5, 3))
    assert float(loss) == pytest.approx((1.0 + 1.0) / 2 + 100.0)
    assert float(force_loss(result, batch, torch.tensor([1.0, 0.0]), forces, energy_weight=2.0)) == pytest.approx(2.0)
    with pytest.raises(ValueError):
        force_loss(result, batch, torch.zeros(3), forces)


def test_optimizer_requires_the_device():
    from mace_ictc.training import create_optimizer
    with pytest.raises(ValueError):
        create_optimizer(_model(block_norm=True))


def _normed_model():
    from mace_ictc.models import MACEICTC
    from oracle.model_ops import OracleOps
    torch.manual_seed(12)
    return MACEICTC(channels=8, lmax=2, num_interactions=3, r_max=3.0, avg_num_neighbors=5.0, ops=OracleOps(),
                    block_norm=True, block_scale=0.5).double()


def _rank(rank, world, port, out_dir, case):
    import os
    import test_parallel_cpu
    test_parallel_cpu._model = _normed_model
    if rank < world:
        test_parallel_cpu._worker(rank, world, port, out_dir, case)
    else:       # the single process, beside the ranks and with as many threads (coupling tables depend on them)
        torch.set_num_threads(1)
        torch.save(test_parallel_cpu._single(*test_parallel_cpu._system(**case["system"])),
                   os.path.join(out_dir, "single.pt"))


def test_slab_decomposition_with_block_norms(tmp_path):
    """Norms act row by row, so ranks with halos give the single process's energy and forces."""
    import torch.multiprocessing as mp
    from test_parallel_cpu import _free_port
    case = {"system": {"n_atoms": 60, "seed": 4}}
    mp.start_processes(_rank, args=(2, _free_port(), str(tmp_path), case), nprocs=3, join=True, start_method="spawn")
    outs = [torch.load(tmp_path / f"rank{r}.pt") for r in range(2)]
    energy, forces, virial = torch.load(tmp_path / "single.pt")
    joined = torch.empty_like(forces)
    for out in outs:
        joined[out["ids"]] = out["forces"]
        # FP64 sums in another order (1e-15 each, some 1e3 terms) through three norms (1e3 times)
        torch.testing.assert_close(out["energy"], energy, rtol=1e-9, atol=1e-9)
        torch.testing.assert_close(out["virial"], virial, rtol=1e-8, atol=1e-8)
    torch.testing.assert_close(joined, forces, rtol=1e-8, atol=1e-8)


def test_training_step_refuses_a_capture(monkeypatch):
    from mace_ictc.training import train_step
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        train_step(*[None] * 11)
