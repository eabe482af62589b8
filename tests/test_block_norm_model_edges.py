"""Models from before there were block norms (CPU, FP64 oracle operators)."""
import pickle

import torch

from test_block_norm_model import _model, _system


def test_models_without_the_option_still_run():
    """A pickled model has no attribute of that name, and an interaction block of a user's own takes no stream."""
    model = _model(4, layers=2)
    system = _system()
    want = model.energy_and_forces(*system)
    old = pickle.loads(pickle.dumps(model))
    del old.__dict__["block_norm"]

    def forward(ops, node_feats, edge_harmonics, edge_feats, src, dst, mask, groups, owned=None, species=None,
                exchange=None):
        return block(ops, node_feats, edge_harmonics, edge_feats, src, dst, mask, groups, owned, species, exchange)

    block = type(old.interactions[1]).forward.__get__(old.interactions[1])
    old.interactions[1].forward = forward
    for a, b in zip(old.energy_and_forces(*system), want):
        assert torch.equal(a, b)
