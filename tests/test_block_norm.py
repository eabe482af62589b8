"""Block norms: refusals, entry points and the torch formula's derivatives (CPU only)."""
import ctypes

import pytest
import torch


def test_host_tensors_are_refused():
    from ictc_o3.ops.block_norm import DegreeNorm, ResidualBlockNorm, degree_norm, residual_block_norm
    x = torch.zeros(4, 8 * 9)
    with pytest.raises(ValueError):
        degree_norm(x, torch.ones(3, 8), channels=8, lmax=2)
    with pytest.raises(ValueError):
        residual_block_norm(x, x, channels=8, lmax=2)
    with pytest.raises(ValueError):
        DegreeNorm(8, 2)(x)
    with pytest.raises(ValueError):
        ResidualBlockNorm(8, 2)(x, x)


@pytest.mark.parametrize("change", [{"channels": 0}, {"channels": 8.0}, {"lmax": 4}, {"lmax": -1}, {"lmax": True},
                                    {"layout": "irmul"}, {"eps": 0.0}, {"eps": float("inf")}, {"eps": 1e-42},
                                    {"channels": 100_000}])
def test_forms_are_checked_before_tensors(change):
    from ictc_o3.ops.block_norm import residual_block_norm
    form = {"channels": 8, "lmax": 2, **change}
    with pytest.raises(ValueError, match="channels|lmax|layout|eps|width"):
        residual_block_norm(None, None, **form)
    with pytest.raises(ValueError, match="norm"):
        residual_block_norm(None, None, channels=8, lmax=2, pre_weight=torch.ones(3, 8), norm=False)


def test_native_entry_points_validate_before_launching():
    from ictc_o3.backends.cuda import _native
    lib = _native.library()
    some = ctypes.c_void_p(16)
    no = None

    def forward(stream=some, branch=some, norm=1, rows=4, c=8, l=2, layout=1, eps=1e-6, out=some, normed=some,
                status=some):
        return lib.ictc_block_forward(stream, branch, no, no, no, no, norm, rows, c, l, layout, eps, out, normed, no,
                                      no, status, no)

    for bad in ({"stream": no}, {"out": no}, {"normed": no}, {"rows": -1}, {"c": 0}, {"l": 4}, {"layout": 2},
                {"eps": 0.0}, {"branch": no, "norm": 0}, {"status": no}):
        assert forward(**bad) == -1, bad
        assert "invalid" in lib.ictc_last_error().decode()
    assert forward(rows=0, stream=no, out=no, normed=no) == 0
    assert forward(c=100_000) == -2
    nothing = [no] * 6
    back = lambda p, q, grads, r=some, partial=some: lib.ictc_block_backward(  # noqa: E731
        some, some, no, no, no, no, r, r, p, q, 4, 8, 2, 1, *grads, partial, some, no)
    assert back(no, no, nothing) == -1
    assert back(some, no, [some] + [no] * 5) == -1                # the stream's gradient is p itself
    assert back(some, some, [no] * 3 + [some, no, no], partial=no) == -1
    assert back(some, some, [no, no, some, no, no, no]) == -1     # a gate gradient without a gate
    assert back(some, some, nothing, r=no) == -1
    second = lambda q, dots, grads: lib.ictc_block_second(  # noqa: E731
        some, some, no, no, no, no, some, some, some, q, *dots, 4, 8, 2, 1, *grads, some, some, no)
    assert second(some, [some, some, some], [no] * 8) == -1
    assert second(no, [some, some, no], [no] * 7 + [some]) == -1
    assert lib.ictc_block_partial_floats(8, 4) == -1
    assert [lib.ictc_block_supported(*s) for s in ((1, 0), (450, 3), (7200, 0), (0, 1), (8, 4), (4000, 3))] == [
        1, 1, 1, 0, 0, 0]


@pytest.mark.parametrize("gated, norm", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("layout", ["mul_ir", "ir_mul"])
def test_formula_gradients(layout, gated, norm):
    """The torch formula (used past the second order) and its gradients against differences in FP64, and
    against autograd of the whole operator."""
    from ictc_o3.backends.cuda.block_norm import Form, _formula_gradients, formula
    torch.manual_seed(0)
    form = Form(3, 2, layout, 1e-3, norm)
    make = lambda *shape: torch.randn(*shape, dtype=torch.float64, requires_grad=True)  # noqa: E731
    stream, branch, gate = make(2, 27), make(2, 27), make(2, 9) if gated else None
    post, scale, pre = make(3, 3), make(3, 3), make(3, 3) if norm else None
    tensors = [t for t in (stream, branch, gate, post, scale, pre) if t is not None]

    def run(*values):
        it = iter(values)
        out = formula(form, next(it), next(it), next(it) if gated else None, next(it), next(it),
                      next(it) if norm else None)
        return out if norm else out[0]

    assert torch.autograd.gradcheck(run, tensors)
    out, u = formula(form, stream, branch, gate, post, scale, pre)
    p, q = torch.randn_like(out), torch.randn_like(out) if norm else None
    want = torch.autograd.grad([out] + ([u] if norm else []), tensors, [p] + ([q] if norm else []))
    args = [t if t is None else t.detach().requires_grad_() for t in (out, branch, gate, post, scale, pre)]
    got = [g for g, t in zip(_formula_gradients(form, *args, p, q), args) if t is not None]
    for a, b in zip(got, want):
        torch.testing.assert_close(a.detach(), b, rtol=1e-12, atol=1e-12)


def test_norm_commutes_with_rotations():
    from ictc_o3.backends.cuda.block_norm import Form, formula
    torch.manual_seed(1)
    q, _ = torch.linalg.qr(torch.randn(3, 3, dtype=torch.float64))
    x, y = (torch.randn(5, 4, 4, dtype=torch.float64) for _ in range(2))
    gate, w = torch.randn(5, 8, dtype=torch.float64), torch.randn(2, 4, dtype=torch.float64)

    def flat(t, turn):        # degree 0: column 0, degree 1: the three others
        return torch.cat([t[:, :, 0], (t[:, :, 1:] @ turn).reshape(5, -1)], 1)

    eye = torch.eye(3, dtype=torch.float64)
    form = Form(4, 1, "mul_ir", 1e-6, True)
    plain = formula(form, flat(x, eye), flat(y, eye), gate, w, None, w)
    turned = formula(form, flat(x, q), flat(y, q), gate, w, None, w)
    for a, b in zip(plain, turned):
        a = torch.cat([a[:, :4], (a[:, 4:].reshape(5, 4, 3) @ q).reshape(5, -1)], 1)
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)
