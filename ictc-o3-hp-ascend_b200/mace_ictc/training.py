"""Force-loss training step of a MACE-ICTC model on the CUDA backend.

The loss is the reference trainer's kind (``mace_ictc/training/train_loop.py:1204``): squared
errors of the energy per atom and of the force components.  A step runs the energy, the forces
with their graph, the backward through the mixed second derivatives, and AdamW.
"""
from __future__ import annotations

import torch

from ictc_o3.optim import AdamW

from .runtime import energy_and_forces

__all__ = ["create_optimizer", "force_loss", "train_step"]

# Weights that scale channels one by one: decaying them would pull the blocks towards zero.
_NO_DECAY = (".post_weight", ".scale", ".pre_weight", "input_norm.weight")


def create_optimizer(model, lr=1e-3, *, weight_decay=1e-2, **options):
    """``ictc_o3.optim.AdamW`` over the model's trainable weights; norm weights and residual scales
    do not decay.  ``options`` go to the optimizer (``state_bits``, ``max_norm``, ``ema_decay``, ...)."""
    decay, keep = [], []
    for name, p in model.named_parameters():
        if p.requires_grad:
            (keep if name.endswith(_NO_DECAY) else decay).append(p)
    groups = [{"params": decay}] + ([{"params": keep, "weight_decay": 0.0}] if keep else [])
    return AdamW(groups, lr=lr, weight_decay=weight_decay, **options)


def force_loss(result, batch, energy_target, force_target, *, energy_weight=1.0, force_weight=100.0):
    """energy_weight * mean (E / atoms - target)^2 + force_weight * mean (F - target)^2 of an
    ``energy_and_forces(..., training=True)`` result; ``energy_target`` is per atom [B]."""
    energy, forces = result["energy"], result["forces"]
    if energy_target.shape != energy.shape or force_target.shape != forces.shape:
        raise ValueError("Targets must have the shapes of energies [B] and forces [N,3]")
    atoms = torch.zeros_like(energy).index_add(0, batch, torch.ones_like(batch, dtype=energy.dtype))
    per_atom = energy / atoms.clamp_min(1.0)
    return (energy_weight * (per_atom - energy_target).square().mean()
            + force_weight * (forces - force_target).square().mean())


def train_step(model, optimizer, positions, atomic_numbers, batch, edge_src, edge_dst, edge_shifts, cell, energy_target,
               force_target, *, energy_weight=1.0, force_weight=100.0):
    """One step on a prebuilt batch of graphs (arguments of ``energy_and_forces``): the loss before
    it, as a device scalar that was not waited for.  Not to be captured: what the model derives from its weights
    (packed radial weights, folded tables) is renewed by the host, so replays would use old ones."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a training step cannot be captured into a CUDA graph")
    optimizer.zero_grad(set_to_none=True)
    result = energy_and_forces(model, positions, atomic_numbers, batch, edge_src, edge_dst, edge_shifts, cell,
                               training=True)
    loss = force_loss(result, batch, energy_target, force_target, energy_weight=energy_weight,
                      force_weight=force_weight)
    loss.backward()
    optimizer.step()
    return loss.detach()
