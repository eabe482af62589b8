"""Norms before and after a block with its gate and residual scale, on the CUDA backend.

``_Block`` is the operator, ``_BlockGrad`` its gradients as an operator of its own, so that
both the first derivatives (training, forces) and the second ones (force-loss training) are
single kernels; anything beyond those goes through the torch formula.  The norm without
a block (``branch`` None) is the same pair.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ictc_o3.autograd.adjoint_requirements import required_gradients
from . import _native
from ._native import ptr, stream_of

LAYOUTS = {"ir_mul": 0, "mul_ir": 1}


class Form(NamedTuple):
    """What does not depend on the values."""
    channels: int
    lmax: int
    layout: str
    eps: float
    norm: bool          # normed rows are produced

    @property
    def shape(self):
        return self.channels, self.lmax, LAYOUTS[self.layout]


def formula(form: Form, stream, branch, gate, post, scale, pre):
    """The operator in torch operations (any dtype and device): (stream, normed or None)."""
    c, n = form.channels, stream.shape[0]

    def degrees(x):
        for l in range(form.lmax + 1):
            block = x[:, c * l * l:c * (l + 1) ** 2]
            yield block.reshape(n, 2 * l + 1, c).transpose(1, 2) if form.layout == "ir_mul" else block.reshape(
                n, c, 2 * l + 1)

    def normed(x, factors):
        out = []
        for l, b in enumerate(degrees(x)):
            b = b * (b.square().mean((1, 2), keepdim=True) + form.eps).rsqrt()
            for f in factors:
                b = b * f[..., l * c:(l + 1) * c].unsqueeze(-1)
            out.append((b.transpose(1, 2) if form.layout == "ir_mul" else b).reshape(n, (2 * l + 1) * c))
        return torch.cat(out, 1)

    if branch is not None:
        factors = [w.reshape(-1) for w in (post, scale) if w is not None]
        if gate is not None:
            factors.append(torch.sigmoid(gate))
        stream = stream + normed(branch, factors)
    return stream, normed(stream, [] if pre is None else [pre.reshape(-1)]) if form.norm else None


def _formula_gradients(form, stream, branch, gate, post, scale, pre, p, q):
    """First gradients (stream, branch, gate, post, scale, pre) through ``formula``, where ``stream``
    is the stream behind the block; differentiable in every argument."""
    tensors = [stream, branch, gate, post, scale, pre]
    with torch.enable_grad():
        # the norm acts on the stream behind the block, the rest on the block's branch
        grads = [None] * 6
        total = p
        if q is not None:
            _, u = formula(form._replace(norm=True), stream, None, None, None, None, pre)
            wanted = [stream] + ([pre] if pre is not None else [])
            got = torch.autograd.grad(u, wanted, q, create_graph=True)
            total = got[0] if p is None else p + got[0]
            if pre is not None:
                grads[5] = got[1]
        if branch is not None:
            delta, _ = formula(form._replace(norm=False), torch.zeros_like(branch), branch, gate, post, scale, None)
            names = [k for k in (1, 2, 3, 4) if tensors[k] is not None]
            for k, v in zip(names, torch.autograd.grad(delta, [tensors[k] for k in names], total, create_graph=True)):
                grads[k] = v
        grads[0] = total
    return grads


def _like(x, wanted=True):
    return torch.empty_like(x) if wanted and x is not None else None


def _partial(form, x, wanted):
    if not wanted:
        return None
    count = int(_native.library().ictc_block_partial_floats(form.channels, form.lmax))
    return torch.empty(count, device=x.device, dtype=torch.float32)


_status = {}


def status_word(device):
    """The device word (int32) that the kernels set when a copy did not land in time."""
    word = _status.get(device)
    if word is None:
        word = torch.zeros(1, dtype=torch.int32, device=device)
        if not torch.cuda.is_current_stream_capturing():      # a capture's memory is its graph's own
            _status[device] = word
    return word


def _dense(x):
    return None if x is None else x.contiguous()


class _Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, form, stream, branch, gate, post, scale, pre):
        n = stream.shape[0]
        keep = any(ctx.needs_input_grad)
        out = _like(stream, branch is not None)
        u = _like(stream, form.norm)
        r1 = torch.empty(n, 4, device=stream.device, dtype=torch.float32) if keep and branch is not None else None
        r2 = torch.empty(n, 4, device=stream.device, dtype=torch.float32) if keep and form.norm else None
        with torch.cuda.device(stream.device):
            _native.call("ictc_block_forward", ptr(stream), ptr(branch), ptr(gate), ptr(post), ptr(scale), ptr(pre),
                         int(form.norm), n, *form.shape, form.eps, ptr(out), ptr(u), ptr(r1), ptr(r2),
                         ptr(status_word(stream.device)), stream_of(stream))
        ctx.form, ctx.rates = form, (r1, r2)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(stream if out is None else out, branch, gate, post, scale, pre)
        return (u,) if out is None else (out,) if u is None else (out, u)

    @staticmethod
    def backward(ctx, *cotangents):
        form = ctx.form
        stream, branch, gate, post, scale, pre = ctx.saved_tensors
        p = cotangents[0] if branch is not None else None
        q = cotangents[-1] if form.norm else None
        if p is None and q is None:
            return (None,) * 7
        need = required_gradients((None, stream, branch, gate, post, scale, pre),
                                  (False, *ctx.needs_input_grad[1:]))
        # the saved stream is this operator's output: whether the input's gradient runs is declared
        need = (False, ctx.needs_input_grad[1], *need[2:])
        grads = _BlockGrad.apply(form, ctx.rates, need[1:], stream, branch, gate, post, scale, pre, _dense(p),
                                 _dense(q))
        dx = p if q is None else grads[0]
        return (None, dx if need[1] else None, *grads[1:])


class _BlockGrad(torch.autograd.Function):
    """(stream, branch, gate, post, scale, pre) gradients; ``stream`` is the one behind the block."""

    @staticmethod
    def forward(ctx, form, rates, need, stream, branch, gate, post, scale, pre, p, q):
        ctx.form, ctx.rates = form, rates
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(stream, branch, gate, post, scale, pre, p, q)
        r1, r2 = rates
        out = [_like(t, w) for t, w in zip((stream, branch, gate, post, scale, pre), need)]
        if q is None:
            out[0] = out[5] = None
        if branch is not None or out[0] is not None or out[5] is not None:
            partial = _partial(form, stream, any(w is not None for w in out[3:]))
            with torch.cuda.device(stream.device):
                _native.call("ictc_block_backward", ptr(stream), ptr(branch), ptr(gate), ptr(post), ptr(scale),
                             ptr(pre), ptr(r1), ptr(r2), ptr(p), ptr(q), stream.shape[0], *form.shape,
                             *(ptr(t) for t in out), ptr(partial), ptr(status_word(stream.device)), stream_of(stream))
        return tuple(out)

    @staticmethod
    def backward(ctx, dot_stream, dot_branch, dot_gate, *dot_weights):
        form, (r1, r2) = ctx.form, ctx.rates
        saved = ctx.saved_tensors
        stream, branch, gate, post, scale, pre, p, q = saved
        need = ctx.needs_input_grad[3:]
        dots = (dot_stream, dot_branch, dot_gate, *dot_weights)
        if all(d is None for d in dots):
            return (None,) * 11
        if torch.is_grad_enabled() or any(d is not None for d in dot_weights):
            # third derivatives, or derivatives of the weights' gradients
            with torch.enable_grad():
                # views, so that each argument's derivative is the partial one (the stream's history
                # holds the branch)
                values = [t if t is None else t.view_as(t) if t.requires_grad else t.detach().requires_grad_()
                          for t in saved]
                grads = _formula_gradients(form, *values)
                pairs = [(g, d) for g, d in zip(grads, dots) if d is not None and g is not None]
                wanted = [k for k in range(8) if need[k]]
                got = torch.autograd.grad([g for g, _ in pairs], [values[k] for k in wanted], [d for _, d in pairs],
                                          create_graph=torch.is_grad_enabled(), allow_unused=True)
            result = [None] * 8
            for k, v in zip(wanted, got):
                result[k] = v
            return (None, None, None, *result)
        out = [_like(t, w) for t, w in zip(saved, need)]
        if q is None:
            out[0] = out[5] = out[7] = None
        partial = _partial(form, stream, any(w is not None for w in out[3:6]))
        dots = [_dense(d) for d in dots[:3]]
        with torch.cuda.device(stream.device):
            _native.call("ictc_block_second", ptr(stream), ptr(branch), ptr(gate), ptr(post), ptr(scale), ptr(pre),
                         ptr(r1), ptr(r2), ptr(p), ptr(q), *(ptr(d) for d in dots), stream.shape[0], *form.shape,
                         *(ptr(t) for t in out), ptr(partial), ptr(status_word(stream.device)), stream_of(stream))
        return (None, None, None, *out)
