"""AdamW kernels on the CUDA backend: static tables and launches of one optimizer.

``TensorTable`` is what does not change while an optimizer lives: how its tensors are
cut into chunks, and where each one's state lies (starts are multiples of
``BLOCK`` values).  The addresses of weights and gradients are gathered for every step.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native
from ._native import launch

BLOCK = 256   # values that share a scale of the 8-bit moments (csrc/adamw.cu)
WAVE = 740    # blocks of the 8-bit kernel that a B200 holds at once (five per multiprocessor; four of the 32-bit one)


def blocks_of(numel: int) -> int:
    return -(-numel // BLOCK)


def turns_of(total: int) -> int:
    """Turns of 1,024 values per block: as many as leave one wave of blocks, 8 at most.

    Microseconds of a step with 32 / 8-bit states and 1, 2, 4, 8, 16 turns:
    30,000 values 8.3 8.6 10.4 12.5 18.6 / 6.3 8.4 10.3 12.4 18.6;  1 M 12.4 10.4 11.5 14.5 20.6 / 11.1
    10.4 10.4 14.5 20.6;  4 M 24.6 20.0 20.2 18.4 22.7 / 24.7 20.6 20.6 21.2 24.7;  16 M 94 77 76 76 78 / 90
    74 67 67 75;  160 M 859 684 663 673 678 / 828 655 584 542 532."""
    turns = 1
    while turns < 8 and total > turns * 1024 * WAVE:
        turns *= 2
    return turns


class TensorTable:
    """Chunks and state places of tensors of the given sizes."""

    def __init__(self, sizes, device, turns=None):
        sizes = list(sizes)
        if turns is None:
            turns = turns_of(sum(sizes))
        chunk = turns * int(_native.library().ictc_adamw_turn_values())
        sizes = torch.tensor(sizes, dtype=torch.int64)
        blocks = (sizes + BLOCK - 1) // BLOCK
        counts = (sizes + chunk - 1) // chunk
        first = torch.zeros(sizes.numel() + 1, dtype=torch.int64)
        torch.cumsum(counts, 0, out=first[1:])
        starts = torch.cumsum(blocks, 0) - blocks
        tensor = torch.repeat_interleave(torch.arange(sizes.numel()), counts)
        number = torch.arange(int(first[-1])) - first[tensor]
        if int(blocks.sum()) > 0x7fffffff:
            raise ValueError("the optimizer holds too many values")
        values = torch.clamp(sizes[tensor] - number * chunk, max=chunk)
        block = starts[tensor] + number * (chunk // BLOCK)
        table = torch.stack((tensor, values, block, number), 1).to(torch.int32)
        self.count, self.chunk = sizes.numel(), chunk
        self.starts = (starts * BLOCK).tolist()
        self.blocks = int(blocks.sum())
        self.values = self.blocks * BLOCK
        self.chunks = table.contiguous().to(device)
        self.first_chunk = (ctypes.c_int64 * (self.count + 1))(*first.tolist())
        self.workspace = torch.zeros(int(_native.library().ictc_adamw_workspace_bytes()), dtype=torch.uint8,
                                     device=device)
        self.device, self.chunks_at, self.workspace_at = (self.workspace.device, self.chunks.data_ptr(),
                                                          self.workspace.data_ptr())
        # word 2 of the workspace: gradient norm of the last step that computed one
        self.norm = self.workspace[8:12].view(torch.float32)[0]

    def grad_norm(self, grads, max_norm, skip_nonfinite):
        """``grads``: address of a host array of ``count`` device pointers (0: no gradient)."""
        launch(self.device, "ictc_adamw_grad_norm", grads, self.count, self.chunks_at, self.first_chunk, self.chunk,
               1.0 if max_norm is None else max_norm, max_norm is not None, skip_nonfinite, self.workspace_at)

    def step(self, weights, grads, first, count, bits, state, *, lr, betas, eps, weight_decay, ema_decay, seed,
             use_norm):
        """``state``: addresses of m, v, their scales, the average, steps and rates (this optimizer's own)."""
        launch(self.device, "ictc_adamw_step", weights, grads, first, count, self.chunks_at, self.first_chunk, self.chunk,
               bits, *state, lr, *betas, eps, weight_decay, ema_decay, seed, use_norm, self.workspace_at)

    def decode(self, state):
        """BF16 values of the 8-bit moments."""
        device = self.workspace.device
        m = torch.empty(self.values, dtype=torch.bfloat16, device=device)
        v = torch.empty(self.values, dtype=torch.bfloat16, device=device)
        if self.values:
            launch(device, "ictc_adamw_decode", state["m"], state["v"], state["m_scale"], state["v_scale"],
                   self.values, m, v)
        return m, v
