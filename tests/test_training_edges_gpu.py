"""Training where a call is out of the ordinary."""
import pytest
import torch

from test_training_gpu import batch_of

pytestmark = pytest.mark.gpu


def test_the_factory_builds_block_norms(cuda_device):
    """``create_model(block_norm=True)`` trains like any other model of this package."""
    from mace_ictc.runtime import check_model, configure_model, create_model, energy_and_forces
    from mace_ictc.training import create_optimizer, train_step
    torch.manual_seed(2)
    model = create_model(channels=16, lmax=2, num_interactions=3, block_norm=True, block_scale=0.25, device=cuda_device)
    assert model.block_norm and all(bool((n.scale == 0.25).all()) for n in model.block_norms)
    assert not create_model(channels=16, lmax=2, device=cuda_device).block_norm
    assert check_model(model)["supported"]
    configure_model(model)
    args = batch_of([20, 17], cuda_device, torch.float32)
    before = energy_and_forces(model, *args)
    optimizer = create_optimizer(model, lr=1e-3)
    loss = train_step(model, optimizer, *args, torch.zeros(2, device=cuda_device), torch.zeros(37, 3, device=cuda_device))
    after = energy_and_forces(model, *args)
    assert torch.isfinite(loss) and not torch.equal(before["energy"], after["energy"])
    with pytest.raises(TypeError):
        create_model(block_norm=1)
