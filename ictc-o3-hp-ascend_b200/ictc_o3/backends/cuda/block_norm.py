"""Norms before and after a block with its gate and residual scale, on the CUDA backend.

``_Block`` is the operator, ``_BlockGrad`` its gradients as an operator of its own, so that
both the first derivatives (training, forces) and the second ones (force-loss training) are
single kernels; anything beyond those goes through the torch formula.  The norm without
a block (``branch`` None) is the same pair.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import _native
from ._native import launch

LAYOUTS = {"ir_mul": 0, "mul_ir": 1}


class Form(NamedTuple):
    """What does not depend on the values."""
    channels: int
    lmax: int
    layout: str
    eps: float
    norm: bool          # normed rows are produced


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


_partial_floats = {}


def _partial(form, x, wanted):
    """Scratch of the weight gradients' sums."""
    if not wanted:
        return None
    key = (x.device, form.channels, form.lmax)
    count = _partial_floats.get(key)
    if count is None:
        with torch.cuda.device(x.device):
            count = _partial_floats[key] = int(_native.library().ictc_block_partial_floats(form.channels, form.lmax))
    return torch.empty(count, device=x.device, dtype=torch.float32)


_status = {}


def status_word(device):
    """Address of the device word (int32) that the kernels set when a copy did not land in time: the
    library's own, so captured launches set it too."""
    word = _status.get(device)
    if word is None:
        found = ctypes.c_void_p()
        with torch.cuda.device(device):
            _native.call("ictc_block_status_word", ctypes.byref(found))
        word = _status[device] = found.value
    return word


def read_status(device, reset):
    value = ctypes.c_int()
    launch(device, "ictc_block_status", reset, ctypes.addressof(value))
    return value.value


def dense(x):
    """``x`` with its values one after another at its address: contiguous, and no lazily negated view."""
    if x is None or (x.is_contiguous() and not x.is_neg()):
        return x
    return x.resolve_neg().contiguous()


def _refuse_tangents(*tensors):
    """Forward-mode derivatives have no kernel: outputs written by address would drop their tangents."""
    if getattr(forward_ad, "_current_level", 0) < 0:      # no dual level is open
        return
    if any([t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors]):
        raise ValueError("block norms have no forward-mode derivatives; the CUDA backend requires ordinary eager "
                         "autograd")


def _forward(form, keep, stream, branch, gate, post, scale, pre):
    """(stream', normed, r1, r2): what is not produced, or without ``keep`` not kept, is None."""
    n, device = stream.shape[0], stream.device
    out = None if branch is None else torch.empty_like(stream)
    u = torch.empty_like(stream) if form.norm else None
    r1 = torch.empty(n, 4, device=device, dtype=torch.float32) if keep and branch is not None else None
    r2 = torch.empty(n, 4, device=device, dtype=torch.float32) if keep and form.norm else None
    launch(device, "ictc_block_forward", stream, branch, gate, post, scale, pre, form.norm, n, form.channels, form.lmax,
           LAYOUTS[form.layout], form.eps, out, u, r1, r2, status_word(device))
    return out, u, r1, r2


def _first(form, rates, need, stream, branch, gate, post, scale, pre, p, q):
    """Gradients of (stream, branch, gate, post, scale, pre), None where ``need`` is false."""
    out = [_like(t, w) for t, w in zip((stream, branch, gate, post, scale, pre), need)]
    if q is None:
        out[0] = out[5] = None
    if any(t is not None for t in out):
        partial = _partial(form, stream, any(t is not None for t in out[3:]))
        launch(stream.device, "ictc_block_backward", stream, branch, gate, post, scale, pre, *rates, p, q,
               stream.shape[0], form.channels, form.lmax, LAYOUTS[form.layout], *out, partial,
               status_word(stream.device))
    return tuple(out)


_probe = getattr(torch._C, "_will_engine_execute_node", None)


def _runs(node):
    """Whether the running backward pass executes an input's gradient node (true where it cannot tell)."""
    if _probe is None or node is None or hasattr(node, "variable"):      # a leaf: the engine does not say
        return True
    try:
        return _probe(node)
    except RuntimeError:
        return True


def _check_capture(ctx):
    """A captured backward pass hands each leaf's gradient to the stream of the oldest living graph with this
    leaf.  If that is the default stream, which cannot take part in a capture, the process would end: refused here."""
    if not torch.cuda.is_current_stream_capturing():
        return
    for node, _ in ctx.next_functions:
        leaf = getattr(node, "variable", None)
        if leaf is not None and _native.host_tensors().accumulates_on_default_stream(leaf):
            raise RuntimeError("a backward pass cannot be captured while a graph of the same leaves, recorded on the "
                               "default stream, lives: drop its outputs first")


class _Block(torch.autograd.Function):
    @staticmethod
    def forward(ctx, form, stream, branch, gate, post, scale, pre):
        out, u, *ctx.rates = _forward(form, True, stream, branch, gate, post, scale, pre)
        ctx.form = form
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(stream if out is None else out, branch, gate, post, scale, pre)
        return (u,) if out is None else (out,) if u is None else (out, u)

    @staticmethod
    def backward(ctx, *cotangents):
        form = ctx.form
        _check_capture(ctx)
        _refuse_tangents(*cotangents)
        stream, branch, gate, post, scale, pre = saved = ctx.saved_tensors      # once: checkpoints recompute per access
        p = cotangents[0] if branch is not None else None
        q = cotangents[-1] if form.norm else None
        if p is None and q is None:
            return (None,) * 7
        # asked of the engine: whether the branch's gradient runs (a row written or not) and whether any
        # weight's does; the weights share their sums, and a gate's gradient is small.  autograd.grad does not tell
        # for leaves, so a pass for forces sums the weights' gradients too (6 us at 8,192 rows of C128/lmax 3;
        # views that could be asked cost 25 us of host time)
        _, need_stream, need_branch, need_gate, *need_weights = ctx.needs_input_grad
        nodes = iter([node for node, _ in ctx.next_functions])      # of the tensors among the arguments
        _, at_branch, _, *at_weights = [None if t is None else next(nodes) for t in saved]
        need_branch = need_branch and _runs(at_branch)
        runs = any(n and _runs(node) for n, node in zip(need_weights, at_weights))
        need = (need_stream, need_branch, need_gate, *[n and runs for n in need_weights])
        args = (form, ctx.rates, need, stream, branch, gate, post, scale, pre, dense(p), dense(q))
        grads = _BlockGrad.apply(*args) if torch.is_grad_enabled() else _first(*args)
        dx = p if q is None else grads[0]
        return (None, dx if need[0] else None, *grads[1:])


class _BlockGrad(torch.autograd.Function):
    """(stream, branch, gate, post, scale, pre) gradients; ``stream`` is the one behind the block."""

    @staticmethod
    def forward(ctx, form, rates, need, stream, branch, gate, post, scale, pre, p, q):
        ctx.form, ctx.rates = form, rates
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(stream, branch, gate, post, scale, pre, p, q)
        return _first(form, rates, need, stream, branch, gate, post, scale, pre, p, q)

    @staticmethod
    def backward(ctx, dot_stream, dot_branch, dot_gate, *dot_weights):
        form = ctx.form
        _check_capture(ctx)
        saved = ctx.saved_tensors
        stream, branch, gate, post, scale, pre, p, q = saved
        need = ctx.needs_input_grad[3:]
        dots = (dot_stream, dot_branch, dot_gate, *dot_weights)
        _refuse_tangents(*dots)
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
        partial = _partial(form, stream, any(t is not None for t in out[3:6]))
        launch(stream.device, "ictc_block_second", stream, branch, gate, post, scale, pre, *ctx.rates, p, q,
               *[dense(d) for d in dots[:3]], stream.shape[0], form.channels, form.lmax, LAYOUTS[form.layout], *out,
               partial, status_word(stream.device))
        return (None, None, None, *out)


def block(form, stream, branch, gate, post, scale, pre):
    """(stream', normed) of arguments that went through ``dense``; without anything to differentiate no graph is made."""
    args = (stream, branch, gate, post, scale, pre)
    _refuse_tangents(*args)
    if torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in args]):
        out = _Block.apply(form, *args)
        return (None, out[0]) if branch is None else out if form.norm else (out[0], None)
    return _forward(form, False, *args)[:2]
