"""Block norms with tensors and calls out of the ordinary."""
import contextlib

import pytest
import torch

from test_block_norm_gpu import inputs

pytestmark = pytest.mark.gpu
NAMES = ("stream", "branch", "gate", "post_weight", "scale", "pre_weight")
FORM = {"channels": 12, "lmax": 2}


def call(t):
    from ictc_o3.ops.block_norm import residual_block_norm
    return residual_block_norm(t["stream"], t["branch"], **{k: t[k] for k in NAMES[2:]}, **FORM)


def all_of(t):
    """Outputs, first gradients and their adjoints."""
    leaves = [t[k] for k in NAMES]
    out = call(t)
    first = torch.autograd.grad(out, leaves, [t["p"], t["q"]], create_graph=True)
    second = torch.autograd.grad(first[:3], [*leaves, t["p"], t["q"]], [t["d_stream"], t["d_branch"], t["d_gate"]])
    return [x.detach() for x in (*out, *first, *second)]


@pytest.mark.parametrize("name", [*NAMES, "p", "q", "d_stream", "d_branch", "d_gate"])
def test_negated_views(name, cuda_device):
    """A lazily negated tensor is contiguous and stores the other sign."""
    from ictc_o3.ops.block_norm import degree_norm
    t = inputs(23, 12, 2, seed=3)
    want = all_of(t)
    t[name] = torch._neg_view(t[name].detach().neg()).requires_grad_()
    assert t[name].is_neg() and t[name].is_contiguous()
    assert all(torch.equal(a, b) for a, b in zip(all_of(t), want))
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(call(t), want))
        if name in ("stream", "pre_weight"):
            plain = degree_norm(t["stream"].resolve_neg(), t["pre_weight"].resolve_neg(), **FORM)
            assert torch.equal(degree_norm(t["stream"], t["pre_weight"], **FORM), plain)


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, cuda_device):
    """No kernel computes tangents, with or without a graph; other tensors may be dual meanwhile."""
    from torch.autograd import forward_ad
    t = inputs(7, 12, 2)
    want = [x.detach() for x in call(t)]
    for grad in (False, True):
        u = {k: v.detach().requires_grad_(grad) for k, v in t.items()}
        with forward_ad.dual_level():
            assert all(torch.equal(a, b) for a, b in zip(call(u), want))
            u[name] = forward_ad.make_dual(u[name], torch.ones_like(u[name]))
            with pytest.raises(ValueError, match="forward-mode"):
                call(u)


@pytest.mark.parametrize("second", [False, True])
def test_forward_mode_over_a_backward_pass_is_refused(second, cuda_device):
    from torch.autograd import forward_ad
    t = inputs(7, 12, 2)
    out = call(t)
    cotangents = [t["p"], t["q"]]
    if second:
        out = torch.autograd.grad(out, [t["branch"]], cotangents, create_graph=True)
        cotangents = [t["d_branch"]]
    with forward_ad.dual_level():
        cotangents[0] = forward_ad.make_dual(cotangents[0].detach(), torch.ones_like(cotangents[0]))
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(out, [t["branch"], t["scale"]], cotangents)


@contextlib.contextmanager
def no_patience():
    """Every wait of the block norms for a copy runs out at once (the kernels then drain their copies)."""
    from ictc_o3.backends.cuda import _native
    try:
        _native.call("ictc_block_wait_limit", 0)
        yield
    finally:
        torch.cuda.synchronize()
        _native.call("ictc_block_wait_limit", 2_000_000_000)


@pytest.mark.parametrize("n, channels, lmax", [(1, 64, 2), (37, 4, 0), (301, 8, 3), (20_011, 8, 1), (900, 128, 3), (2003, 132, 1)])
def test_given_up_copies_leave_nan(n, channels, lmax, cuda_device):
    """A kernel whose rows did not arrive reports it, leaves NaN in what it did not compute, and the next
    one works again."""
    from ictc_o3.ops.block_norm import block_norm_status, residual_block_norm
    t = inputs(n, channels, lmax)
    leaves = [t[k] for k in NAMES]

    def forward():
        return residual_block_norm(t["stream"], t["branch"], **{k: t[k] for k in NAMES[2:]}, channels=channels, lmax=lmax)

    def first(out):
        return torch.autograd.grad(out, leaves, [t["p"], t["q"]], create_graph=True)

    def second(grads):
        return torch.autograd.grad(grads[:3], [*leaves, t["p"], t["q"]], [t["d_stream"], t["d_branch"], t["d_gate"]],
                                   retain_graph=True)

    def spoilt(results):
        code = block_norm_status(reset=True)
        return code == 1 and all(bool(x.isnan().all()) for x in results)

    out = forward()
    grads = first(out)
    want = [x.detach().clone() for x in (*out, *grads, *second(grads))]
    assert block_norm_status() == 0
    with no_patience():
        assert spoilt(forward())
        assert spoilt(first(out))
        assert spoilt(second(grads))
    again = forward()
    grads = first(again)
    assert all(torch.equal(a, b) for a, b in zip((*again, *grads, *second(grads)), want))
    assert block_norm_status() == 0


def test_status_of_a_first_call_inside_a_capture(cuda_device, monkeypatch):
    """Replays report to the word that block_norm_status reads, whether or not a call came before the capture."""
    from ictc_o3.backends.cuda import block_norm
    from ictc_o3.ops.block_norm import block_norm_status
    t = {k: v.detach() for k, v in inputs(50, 12, 2).items()}
    want = call(t)
    assert block_norm_status() == 0
    monkeypatch.setattr(block_norm, "_status", {})
    graph = torch.cuda.CUDAGraph()
    with no_patience(), torch.cuda.graph(graph):
        held = call(t)
    assert block_norm_status() == 0
    for _ in range(2):
        graph.replay()
        assert block_norm_status(reset=True) == 1 and all(bool(x.isnan().all()) for x in held)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(call(t), want)) and block_norm_status(reset=True) == 1
    assert block_norm_status() == 0
    with pytest.raises(TypeError):
        block_norm_status(reset=1)


def test_first_use_of_the_library_inside_a_capture(cuda_device):
    """In a process of its own: not even the library's code is on the device before the capture."""
    import os
    import subprocess
    import sys
    from conftest import PACKAGE_ROOT
    program = """
import torch
from ictc_o3.ops.block_norm import block_norm_status, residual_block_norm
x = torch.randn(50, 72, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = residual_block_norm(x, x, channels=8, lmax=2, norm=True)
graph.replay()
assert all(torch.equal(a, b) for a, b in zip(held, residual_block_norm(x, x, channels=8, lmax=2, norm=True)))
assert block_norm_status() == 0
print("same")
"""
    run = subprocess.run([sys.executable, "-c", program], env={**os.environ, "PYTHONPATH": PACKAGE_ROOT},
                         capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "same" in run.stdout, run.stderr[-2000:]


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_blocks(reentrant, cuda_device):
    """Recomputed in the backward pass: the same gradients, and the same adjoints of theirs."""
    from torch.utils.checkpoint import checkpoint
    t = inputs(23, 12, 2, seed=3)
    leaves = [t[k] for k in NAMES]

    def whole(*args):
        return call(dict(zip(NAMES, args)))

    if reentrant:       # this form has first gradients alone, into .grad
        want = torch.autograd.grad(call(t), leaves, [t["p"], t["q"]])
        torch.autograd.backward(checkpoint(whole, *leaves, use_reentrant=True), [t["p"], t["q"]])
        assert all(torch.equal(x.grad, w) for x, w in zip(leaves, want))
        return
    want = all_of(t)
    out = checkpoint(whole, *leaves, use_reentrant=False)
    first = torch.autograd.grad(out, leaves, [t["p"], t["q"]], create_graph=True)
    second = torch.autograd.grad(first[:3], [*leaves, t["p"], t["q"]], [t["d_stream"], t["d_branch"], t["d_gate"]])
    assert all(torch.equal(a, b) for a, b in zip((*out, *first, *second), want))
