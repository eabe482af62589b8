"""Norms before and after a block, fused with the block's gate and residual scale.

A stack of interaction and product blocks keeps a stream of node rows
``[N, C (L+1)^2]`` (degrees 0..L, inside a degree ``mul_ir`` = [C][2l+1] or
``ir_mul`` = [2l+1][C]).  With r(x) = (mean over a degree of x^2 + eps)^(-1/2), the end of one block and the
start of the next are

    stream' = stream + scale * sigmoid(gate) * post_weight * r(branch) * branch
    normed  = pre_weight * r(stream') * stream'

with weights and gates per degree and channel.  r depends on a degree's length only, so the
operator commutes with rotations.  For lmax = 0 a row is a plain vector of C channels.
Forward, first and second derivatives are one kernel each (forces and force-loss training
need both); higher ones go through torch operations.  ``torch.jit.trace`` and forward-mode
derivatives are refused.  All of it can be
captured into a CUDA graph; a backward pass is refused there while a graph of the same leaves recorded on the default stream lives.
"""
from __future__ import annotations

import functools

import torch

from ictc_o3.backends.cuda import _native
from ictc_o3.backends.cuda.block_norm import LAYOUTS, Form, block, dense, read_status
from ictc_o3.backends.cuda.runtime import require_cuda_fp32

__all__ = ["degree_norm", "residual_block_norm", "DegreeNorm", "ResidualBlockNorm",
           "block_norm_status"]


_is_tracing = getattr(torch._C, "_is_tracing", torch.jit.is_tracing)


@functools.lru_cache(maxsize=256, typed=True)
def _form(channels, lmax, layout, eps, norm):
    if not isinstance(channels, int) or isinstance(channels, bool) or channels < 1:
        raise ValueError("channels must be a positive integer")
    if not isinstance(lmax, int) or isinstance(lmax, bool) or not 0 <= lmax <= 3:
        raise ValueError("lmax must be 0, 1, 2 or 3")
    if layout not in LAYOUTS:
        raise ValueError("layout must be ir_mul or mul_ir")
    if isinstance(eps, bool) or not isinstance(eps, (int, float)) or not 1.2e-38 <= eps < float("inf"):
        raise ValueError("eps must be a positive FP32 number")
    if not _native.library().ictc_block_supported(channels, lmax):
        raise ValueError("rows of this width do not fit the kernels' shared memory")
    return Form(channels, lmax, layout, float(eps), norm)


def _check(form, rows, weights, gate=None):
    if _is_tracing():      # sizes are tensors there, and a trace would hold the outputs' allocation alone
        raise ValueError("block norms cannot be traced; the CUDA backend requires ordinary eager autograd")
    c, degrees = form.channels, form.lmax + 1
    n = rows[0].shape[0] if rows[0].ndim else 0
    tensors = [*rows, *weights] if gate is None else [*rows, *weights, gate]
    index = rows[0].get_device()
    if index < 0 or any([t.dtype is not torch.float32 or t.get_device() != index for t in tensors]):
        require_cuda_fp32(*tensors)
    require_cuda_fp32(rows[0])      # and the modes that forbid it
    width, shape = (n, c * degrees * degrees), (degrees, c)
    if any([x.shape != width for x in rows]):
        raise ValueError("Rows must have shape [N,C*(L+1)^2]")
    if any([w.shape != shape for w in weights]):
        raise ValueError("Weights must have shape [L+1,C]")
    if gate is not None and gate.shape != (n, degrees * c) and gate.shape != (n, degrees, c):
        raise ValueError("Gates must have shape [N,(L+1)*C] or [N,L+1,C]")


def block_norm_status(device="cuda", reset=False):
    """0, or what a kernel of this module left after a copy into shared memory did not land within two
    seconds; the results that it could not compute are NaN then.  Launches of replayed graphs count.  Waits
    for the current stream, and with ``reset`` clears the word: for tests, or to tell the cause of NaN."""
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("block norms run on CUDA devices")
    if device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    if not isinstance(reset, bool):
        raise TypeError("reset must be a boolean")
    return read_status(device, reset)


def degree_norm(features, weight=None, *, channels, lmax, layout="mul_ir", eps=1e-6):
    """weight * r(features) * features: the norm before the first block."""
    form = _form(channels, lmax, layout, eps, True)
    _check(form, (features,), () if weight is None else (weight,))
    return block(form, dense(features), None, None, None, None, dense(weight))[1]


def residual_block_norm(stream, branch, *, channels, lmax, post_weight=None, scale=None, gate=None, pre_weight=None,
                        norm=None, layout="mul_ir", eps=1e-6):
    """(stream', normed): the block's branch normed, gated, scaled and added, and the next block's norm.

    Weights [L+1, C] (None: ones), gate [N, (L+1) C] before its sigmoid (None: no gate).  ``norm``:
    whether the normed rows are wanted (default: when ``pre_weight`` is given); normed is None without."""
    if norm is None:
        norm = pre_weight is not None
    if not isinstance(norm, bool) or (pre_weight is not None and not norm):
        raise ValueError("norm must be a boolean, and true where pre_weight is given")
    form = _form(channels, lmax, layout, eps, norm)
    _check(form, (stream, branch), tuple(w for w in (post_weight, scale, pre_weight) if w is not None), gate)
    if gate is not None and gate.ndim == 3:
        gate = gate.reshape(gate.shape[0], (lmax + 1) * channels)
    return block(form, dense(stream), dense(branch), dense(gate), dense(post_weight),
                 dense(scale), dense(pre_weight))


class DegreeNorm(torch.nn.Module):
    """``degree_norm`` with a weight per degree and channel."""

    def __init__(self, channels, lmax, *, layout="mul_ir", eps=1e-6):
        super().__init__()
        self.channels, self.lmax, self.layout, self.eps = channels, lmax, layout, eps
        self.form = _form(channels, lmax, layout, eps, True)
        self.weight = torch.nn.Parameter(torch.ones(lmax + 1, channels))

    def forward(self, features):
        return degree_norm(features, self.weight, channels=self.channels, lmax=self.lmax, layout=self.layout,
                           eps=self.eps)


class ResidualBlockNorm(torch.nn.Module):
    """``residual_block_norm`` with its weights; ``next_norm`` False at the end of a stack.

    ``scale_init`` is the branch's share at the start of training."""

    def __init__(self, channels, lmax, *, next_norm=True, scale_init=1.0, layout="mul_ir", eps=1e-6):
        super().__init__()
        self.channels, self.lmax, self.layout, self.eps = channels, lmax, layout, eps
        self.form = _form(channels, lmax, layout, eps, bool(next_norm))
        self.post_weight = torch.nn.Parameter(torch.ones(lmax + 1, channels))
        self.scale = torch.nn.Parameter(torch.full((lmax + 1, channels), float(scale_init)))
        self.pre_weight = torch.nn.Parameter(torch.ones(lmax + 1, channels)) if next_norm else None

    def forward(self, stream, branch, gate=None):
        return residual_block_norm(stream, branch, post_weight=self.post_weight, scale=self.scale, gate=gate,
                                   pre_weight=self.pre_weight, channels=self.channels, lmax=self.lmax,
                                   layout=self.layout, eps=self.eps)
