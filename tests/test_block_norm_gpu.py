"""Block norms, their gradients and their second derivatives on the GPU against FP64.

Every value is checked against its own bound: k u M, u = 2^-24 and M the value's formula with
all terms taken by magnitude (``magnitudes``; a gradient may cancel down to nothing, its rounding errors do
not).  k counts roundings along the longest chain, first order.  A degree's sum: at most
28 + 7 terms in one lane, 5 steps over lanes, 8 over warps: 48 (products included).  r(y): half of that and
4: 28; sigmoid 4.  stream': 28 + 4 + 6 = 38, below 50.  r(stream') carries 28 + 38 K, K = r^2 <|h'|, M(h')> / D
(what stream' cancelled): below 38 rho, rho = 1 + K.  normed: 38 + 38 rho + 4, with M(h') for h'.
T: r^3 h' <h', b q>: 3 x 38 rho + 38 + 38 + 48 + 6 < 250 rho.  dbranch, dgate: 250 rho + 3 x 28 + 48 + 10 <
400 rho.  Second derivatives take T, tau (400 rho + 28 + 10) or both times r^5 (5 x 38 rho)
and two sums (96): below 400 + 440 + 190 + 96 + 20 < 1200 rho.  A sum over N rows adds N.
"""
import gc
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ROUNDINGS = {"out": 100, "d": 400, "dd": 1200}


def magnitudes(form, t, wanted):
    """Upper magnitudes of all results (the names of ``results``), the factor rho included."""
    c, degrees, n = form.channels, range(form.lmax + 1), t["stream"].shape[0]

    def cut(x):
        x = [x[:, c * l * l:c * (l + 1) ** 2] for l in degrees]
        if form.layout == "ir_mul":
            return [b.reshape(n, 2 * l + 1, c).transpose(1, 2) for l, b in zip(degrees, x)]
        return [b.reshape(n, c, 2 * l + 1) for l, b in zip(degrees, x)]

    def join(x):
        if form.layout == "ir_mul":
            x = [b.transpose(1, 2) for b in x]
        return torch.cat([b.reshape(n, c * (2 * l + 1)) for l, b in zip(degrees, x)], 1)

    d = {k: None if v is None else v.detach().double().cpu() for k, v in t.items()}
    zero = torch.zeros_like(d["stream"])
    rows = lambda k: cut((d[k] if k in wanted and d[k] is not None else zero).abs())  # noqa: E731
    weight = lambda k: [torch.ones(1, c, 1).double() if d[k] is None else d[k][l].abs()[None, :, None]  # noqa: E731
                        for l in degrees]
    rate = lambda x: [(b.square().mean((1, 2), keepdim=True) + form.eps) ** -0.5 for b in x]  # noqa: E731
    mean = lambda a, b: (a * b).mean((1, 2), keepdim=True)  # noqa: E731
    over = lambda f: [f(l) for l in degrees]  # noqa: E731
    flat = lambda x: torch.cat([b.expand(n, c, 1)[:, :, 0] for b in x], 1)  # noqa: E731
    total = lambda x: torch.stack([b.sum((0, 2)) for b in x]) if n else torch.zeros(form.lmax + 1, c).double()  # noqa: E731
    out = {}
    x = cut(d["stream"])
    if d["branch"] is not None:
        ys = cut(d["branch"])
        r1, y = rate(ys), [b.abs() for b in ys]
        post, scale = weight("post_weight"), weight("scale")
        sig = over(lambda l: torch.ones(n, c, 1).double()) if d["gate"] is None else over(
            lambda l: torch.sigmoid(d["gate"].view(n, form.lmax + 1, c, 1)[:, l]))
        w = over(lambda l: post[l] * scale[l])
        a = over(lambda l: w[l] * sig[l])
        sign = over(lambda l: (1 if d["post_weight"] is None else d["post_weight"][l][None, :, None])
                    * (1 if d["scale"] is None else d["scale"][l][None, :, None]) * sig[l])
        true = over(lambda l: x[l] + sign[l] * r1[l] * ys[l])
        h = over(lambda l: x[l].abs() + a[l] * r1[l] * y[l])
        out["out0"] = join(h)
    else:
        true, h = x, [b.abs() for b in x]
    rho = over(lambda l: torch.ones(n, 1, 1).double())
    if form.norm:
        b, r2 = weight("pre_weight"), rate(true)
        rho = over(lambda l: 1 + r2[l] ** 2 * mean(true[l].abs(), h[l]))
        out["out1"] = join(over(lambda l: rho[l] * b[l] * r2[l] * h[l]))
    T = rows("p") if d["branch"] is not None else cut(zero)
    if form.norm:
        q = rows("q")
        t2 = over(lambda l: b[l] * q[l])
        T = over(lambda l: T[l] + r2[l] * t2[l] + r2[l] ** 3 * h[l] * mean(h[l], t2[l]))
    out["d stream"] = join(over(lambda l: rho[l] * T[l]))
    if d["branch"] is not None:
        t1 = over(lambda l: a[l] * T[l])
        out["d branch"] = join(over(lambda l: rho[l] * (r1[l] * t1[l] + r1[l] ** 3 * y[l] * mean(y[l], t1[l]))))
        S = over(lambda l: (r1[l] * y[l] * T[l]).sum(2, keepdim=True))
        out["d gate"] = flat(over(lambda l: rho[l] * w[l] * sig[l] * S[l]))
        sums = total(over(lambda l: rho[l] * sig[l] * S[l]))
        out["d post_weight"] = sums * torch.stack(scale)[:, 0, :, 0]
        out["d scale"] = sums * torch.stack(post)[:, 0, :, 0]
    if form.norm:
        out["d pre_weight"] = total(over(lambda l: rho[l] * r2[l] * h[l] * q[l]))
    tau, gh = rows("d_stream"), cut(zero)
    if d["branch"] is not None:
        be = rows("d_branch")
        de = torch.zeros(n, form.lmax + 1, c, 1).double() if d["gate"] is None or "d_gate" not in wanted else \
            d["d_gate"].abs().view(n, form.lmax + 1, c, 1)
        z = over(lambda l: de[:, l] * w[l] * sig[l])
        inner = over(lambda l: r1[l] * be[l] + r1[l] ** 3 * y[l] * mean(y[l], be[l]))
        tau = over(lambda l: tau[l] + a[l] * inner[l] + z[l] * r1[l] * y[l])
        gy = over(lambda l: r1[l] ** 3 * (y[l] * (mean(t1[l], be[l]) + mean(y[l], z[l] * T[l])) + t1[l] * mean(y[l], be[l])
                                          + be[l] * mean(y[l], t1[l]))
                  + 3 * r1[l] ** 5 * y[l] * mean(y[l], t1[l]) * mean(y[l], be[l]) + r1[l] * z[l] * T[l])
        ga = over(lambda l: (T[l] * inner[l]).sum(2, keepdim=True))
        gw = over(lambda l: sig[l] * (ga[l] + de[:, l] * S[l]))
        gg = over(lambda l: w[l] * sig[l] * (ga[l] + 3 * de[:, l] * S[l]))
    if form.norm:
        down = over(lambda l: r2[l] * tau[l] + r2[l] ** 3 * h[l] * mean(h[l], tau[l]))
        gh = over(lambda l: r2[l] ** 3 * (h[l] * mean(t2[l], tau[l]) + t2[l] * mean(h[l], tau[l])
                                          + tau[l] * mean(h[l], t2[l]))
                  + 3 * r2[l] ** 5 * h[l] * mean(h[l], t2[l]) * mean(h[l], tau[l]))
        out["dd q"] = join(over(lambda l: rho[l] * b[l] * down[l]))
        out["dd pre_weight"] = total(over(lambda l: rho[l] * q[l] * down[l]))
    out["dd stream"], out["dd p"] = join(over(lambda l: rho[l] * gh[l])), join(over(lambda l: rho[l] * tau[l]))
    if d["branch"] is not None:      # stream' = stream + a r(branch) branch carries gh on
        t3 = over(lambda l: a[l] * gh[l])
        S3 = over(lambda l: (r1[l] * y[l] * gh[l]).sum(2, keepdim=True))
        out["dd branch"] = join(over(lambda l: rho[l] * (gy[l] + r1[l] * t3[l] + r1[l] ** 3 * y[l] * mean(y[l], t3[l]))))
        out["dd gate"] = flat(over(lambda l: rho[l] * (gg[l] + w[l] * sig[l] * S3[l])))
        sums = total(over(lambda l: rho[l] * (gw[l] + sig[l] * S3[l])))
        out["dd post_weight"] = sums * torch.stack(scale)[:, 0, :, 0]
        out["dd scale"] = sums * torch.stack(post)[:, 0, :, 0]
    return out


def close(got, want, bound, k, what):
    got, want = got.detach().double().cpu(), want.detach().cpu()
    assert got.shape == want.shape == bound.shape, what
    assert torch.isfinite(got).all(), what
    # 2^-126: products of tiny factors may fall below FP32's normal range
    worst = ((got - want).abs() / (bound + 2.0 ** -126)).max() if got.numel() else 0.0
    assert worst <= 1, f"{what}: {float(worst):.2f} of the bound"
    if got.numel() >= 100:      # independent roundings add by their squares: sqrt(k) of k, four times over
        off, most = float((got - want).norm()), 4 * k ** -0.5 * float(bound.norm())
        assert off <= most, f"{what}: {off / most:.2f} of the bound of the norm"


def inputs(n, channels, lmax, seed=0, device="cuda", gate=True, offset=0):
    """FP32 leaves on the device (views `offset` values into their buffers) by name."""
    gen = torch.Generator().manual_seed(seed)
    width, deg = channels * (lmax + 1) ** 2, lmax + 1

    def make(*shape, shift=0.0, size=1.0):
        x = (shift + size * torch.randn(*shape, generator=gen)).float()
        buf = torch.empty(x.numel() + offset, device=device)
        buf[offset:] = x.reshape(-1).to(device)
        return buf[offset:].view(shape).requires_grad_()

    out = {"stream": make(n, width), "branch": make(n, width, size=0.4),
           "gate": make(n, deg * channels) if gate else None, "post_weight": make(deg, channels, shift=1.0, size=0.2),
           "scale": make(deg, channels, shift=0.5, size=0.2), "pre_weight": make(deg, channels, shift=1.0, size=0.2),
           "p": make(n, width), "q": make(n, width), "d_stream": make(n, width), "d_branch": make(n, width),
           "d_gate": make(n, deg * channels) if gate else None}
    return out


def reference(form, t, order, wanted):
    """Outputs, first and second derivatives in FP64 through autograd of the torch formula."""
    from ictc_o3.backends.cuda.block_norm import formula
    d = {k: v if v is None else v.detach().double().cpu().requires_grad_() for k, v in t.items()}
    stream, u = formula(form, d["stream"], d["branch"], d["gate"], d["post_weight"], d["scale"], d["pre_weight"])
    return results([stream, u] if d["branch"] is not None else [None, u], d, order, wanted)


def results(out, d, order, wanted):
    first_names = [k for k in ("stream", "branch", "gate") if d[k] is not None]
    weights = [k for k in ("post_weight", "scale", "pre_weight") if d[k] is not None]
    pairs = [(o, d[c]) for o, c in zip(out, ("p", "q")) if o is not None and c in wanted]
    found = {"out%d" % k: o for k, o in enumerate(out) if o is not None}
    if order == 0:
        return found
    outs, cots = [o for o, _ in pairs], [c for _, c in pairs]
    if order == 1:
        names = first_names + weights
        got = torch.autograd.grad(outs, [d[k] for k in names], cots, allow_unused=True, materialize_grads=True)
        return found | dict(zip(("d " + k for k in names), got))
    first = torch.autograd.grad(outs, [d[k] for k in first_names], cots, create_graph=True)
    found |= dict(zip(("d " + k for k in first_names), first))
    dots = [(g, d["d_" + k]) for g, k in zip(first, first_names) if "d_" + k in wanted]
    names = first_names + weights + [c for c in ("p", "q") if c in wanted]
    got = torch.autograd.grad([g for g, _ in dots], [d[k] for k in names], [c for _, c in dots], allow_unused=True,
                              materialize_grads=True)
    return found | dict(zip(("dd " + k for k in names), got))


def compare(n, channels, lmax, layout, *, gate=True, norm=True, branch=True, order=2, offset=0, seed=0, device,
            wanted=("p", "q", "d_stream", "d_branch", "d_gate"), weights=True, eps=1e-6, change=None):
    from ictc_o3.backends.cuda.block_norm import Form
    from ictc_o3.ops.block_norm import degree_norm, residual_block_norm
    t = inputs(n, channels, lmax, seed, device, gate and branch, offset)
    if change is not None:
        with torch.no_grad():
            change(t)
    if not branch:
        t["branch"] = t["post_weight"] = t["scale"] = None
    if not norm:
        t["pre_weight"] = None
        wanted = [k for k in wanted if k != "q"]
    if not weights:
        t["post_weight"] = t["scale"] = t["pre_weight"] = None
    form = {"channels": channels, "lmax": lmax, "layout": layout, "eps": eps}
    if branch:
        out = residual_block_norm(t["stream"], t["branch"], post_weight=t["post_weight"], scale=t["scale"],
                                  gate=t["gate"], pre_weight=t["pre_weight"], norm=norm, **form)
    else:
        out = [None, degree_norm(t["stream"], t["pre_weight"], **form)]
    got = results(list(out), t, order, wanted)
    want = reference(Form(channels, lmax, layout, eps, norm), t, order, wanted)
    assert got.keys() == want.keys()
    sizes = magnitudes(Form(channels, lmax, layout, eps, norm), t, wanted)
    for key in want:
        weight = key.split()[-1] in ("post_weight", "scale", "pre_weight")
        k = ROUNDINGS[key.split()[0].rstrip("01")] + (n if weight else 0)
        close(got[key], want[key], k * U * sizes[key], k, f"{key} of {n} rows C{channels} lmax {lmax} {layout}")
    return got


@pytest.mark.parametrize("layout", ["mul_ir", "ir_mul"])
@pytest.mark.parametrize("lmax", [0, 1, 2, 3])
@pytest.mark.parametrize("channels", [1, 2, 4, 7, 8, 32, 50, 64, 100, 128, 132])
def test_all_derivatives(channels, lmax, layout, cuda_device):
    for n in (1, 3, 70):
        compare(n, channels, lmax, layout, device=cuda_device, seed=n)


@pytest.mark.parametrize("channels, lmax", [(257, 1), (512, 2), (450, 3), (1028, 0), (7200, 0), (2000, 0), (1001, 1)])
def test_wide_rows(channels, lmax, cuda_device):
    for layout in ("mul_ir", "ir_mul"):
        compare(5, channels, lmax, layout, device=cuda_device)


@pytest.mark.parametrize("n, channels, lmax", [(20_011, 8, 2), (5003, 64, 2), (4099, 128, 3), (9001, 50, 1)])
def test_many_rows(n, channels, lmax, cuda_device):
    compare(n, channels, lmax, "mul_ir", device=cuda_device)
    compare(n, channels, lmax, "ir_mul", device=cuda_device, order=1)


@pytest.mark.parametrize("gate, norm, branch, weights", [c for c in itertools.product([True, False], repeat=4)
                                                         if c[2] or (c[1] and not c[0])])
@pytest.mark.parametrize("channels", [16, 50])
def test_parts(channels, gate, norm, branch, weights, cuda_device):
    for order in (0, 1, 2):
        compare(37, channels, 2, "mul_ir", gate=gate, norm=norm, branch=branch, weights=weights, order=order,
                device=cuda_device)


@pytest.mark.parametrize("wanted", [("p", "d_branch"), ("q", "d_stream"), ("p", "q", "d_gate"), ("q", "d_branch"),
                                    ("p", "q", "d_stream")])
def test_absent_cotangents(wanted, cuda_device):
    compare(29, 24, 2, "mul_ir", wanted=wanted, device=cuda_device)


@pytest.mark.parametrize("frozen", [("stream",), ("branch", "gate"), ("stream", "branch", "gate"),
                                    ("post_weight", "scale", "pre_weight"), ("stream", "branch", "scale", "pre_weight"),
                                    ("gate", "post_weight", "pre_weight"), ("branch", "post_weight", "scale")])
def test_frozen_arguments(frozen, cuda_device):
    """Whatever does not require a gradient, the others receive the same ones."""
    from ictc_o3.ops.block_norm import residual_block_norm
    t = inputs(41, 24, 2, seed=9)
    names = ["stream", "branch", "gate", "post_weight", "scale", "pre_weight"]

    def run(values):
        out = residual_block_norm(values["stream"], values["branch"], channels=24, lmax=2,
                                  **{k: values[k] for k in names[2:]})
        live = [k for k in names if values[k].requires_grad]
        first = torch.autograd.grad(out, [values[k] for k in live], [t["p"], t["q"]], create_graph=True)
        rows = [g for g, k in zip(first, live) if k in names[:3]]
        found = dict(zip(live, first))
        if rows:
            dots = [t["d_" + k] for k in live if k in names[:3]]
            second = torch.autograd.grad(rows, [values[k] for k in live], dots, allow_unused=True)
            found |= {"dd " + k: g for k, g in zip(live, second)}
        return found

    some = {k: t[k].detach().requires_grad_(k not in frozen) for k in names}
    got, full = run(some), run({k: t[k] for k in names})
    for k, g in got.items():
        if not k.startswith("dd ") and g is not None:
            assert torch.equal(g, full[k]), k
    zero = dict(t, **{"d_" + k: torch.zeros_like(t["d_" + k]) for k in names[:3] if k in frozen})
    t.update(zero)                       # frozen rows have no cotangent of their gradient
    full = run({k: t[k].detach().requires_grad_() for k in names})
    for k, g in got.items():
        if k.startswith("dd ") and g is not None:
            assert torch.allclose(g, full[k], rtol=1e-5, atol=1e-5 * float(full[k].abs().max())), k


@pytest.mark.parametrize("offset", [1, 2])
@pytest.mark.parametrize("channels, lmax", [(64, 2), (50, 1), (7, 3)])
def test_unaligned_views(channels, lmax, offset, cuda_device):
    a = compare(45, channels, lmax, "mul_ir", offset=offset, device=cuda_device)
    b = compare(45, channels, lmax, "mul_ir", device=cuda_device)
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_zero_rows_and_extreme_values(cuda_device):
    def zero(t):
        t["branch"][2] = 0.0
        t["stream"][3] = 0.0
        t["branch"][3] = 0.0
        t["gate"][4] = 200.0
        t["gate"][5] = -200.0
        t["branch"][6] *= 1e15
        t["stream"][7] *= 1e-12

    compare(11, 32, 2, "mul_ir", device=cuda_device, order=0, change=zero)
    compare(11, 32, 2, "mul_ir", device=cuda_device, order=1, change=zero, eps=1e-2)
    compare(11, 32, 2, "mul_ir", device=cuda_device, order=2, change=zero, eps=1e-2)
    compare(0, 32, 2, "mul_ir", device=cuda_device, order=0)
    got = compare(0, 32, 2, "mul_ir", device=cuda_device, order=1)
    assert not got["d scale"].any()


def test_rows_do_not_mix(cuda_device):
    """A row with NaN or infinity spoils itself alone, and results do not depend on the rows around."""
    from ictc_o3.ops.block_norm import residual_block_norm
    for channels in (8, 64, 50):
        t = inputs(33, channels, 2)
        form = {"channels": channels, "lmax": 2}
        call = lambda s, b, g: residual_block_norm(s, b, gate=g, norm=True, **form)  # noqa: E731
        with torch.no_grad():
            clean = call(t["stream"], t["branch"], t["gate"])
            bad = t["branch"].clone()
            bad[5, 3], bad[17, 0] = float("nan"), float("inf")
            dirty = call(t["stream"], bad, t["gate"])
            keep = torch.ones(33, dtype=torch.bool, device=cuda_device)
            keep[5] = keep[17] = False
            part = call(t["stream"][9:14], t["branch"][9:14], t["gate"][9:14])
        for a, b, c in zip(clean, dirty, part):
            assert torch.equal(a[keep], b[keep]) and not torch.isfinite(b[~keep]).all()
            assert torch.equal(a[9:14], c)


def test_repeated_runs_and_shared_inputs(cuda_device):
    """Same bits every time (no atomics); one tensor given as stream and branch receives both gradients."""
    from ictc_o3.ops.block_norm import residual_block_norm
    t = inputs(3001, 64, 2)
    form = {"channels": 64, "lmax": 2}

    def grads():
        out = residual_block_norm(t["stream"], t["branch"], post_weight=t["post_weight"], scale=t["scale"],
                                  gate=t["gate"], pre_weight=t["pre_weight"], **form)
        return torch.autograd.grad(out, [t[k] for k in ("stream", "branch", "gate", "post_weight", "scale",
                                                        "pre_weight")], [t["p"], t["q"]])

    assert all(torch.equal(a, b) for a, b in zip(grads(), grads()))
    x = t["stream"]
    both = residual_block_norm(x, x, norm=True, **form)
    (whole,) = torch.autograd.grad(both, [x], [t["p"], t["q"]])
    y = x.detach().clone().requires_grad_()
    split = torch.autograd.grad(residual_block_norm(x, y, norm=True, **form), [x, y], [t["p"], t["q"]])
    assert torch.equal(whole, split[0] + split[1])
    shared = torch.ones(64, device=cuda_device, requires_grad=True)      # one weight broadcast to every degree
    out, _ = residual_block_norm(x, y, scale=shared.expand(3, 64), **form)
    (g,) = torch.autograd.grad(out, [shared], [t["p"]])
    full = torch.ones(3, 64, device=cuda_device, requires_grad=True)
    out, _ = residual_block_norm(x, y, scale=full, **form)
    assert torch.allclose(g, torch.autograd.grad(out, [full], [t["p"]])[0].sum(0), rtol=1e-6)


def test_gradient_against_differences(cuda_device):
    """Directional derivative of the FP32 kernels by central differences."""
    from ictc_o3.ops.block_norm import residual_block_norm
    t = inputs(40, 16, 2, seed=4)
    names = ("stream", "branch", "gate", "post_weight", "scale", "pre_weight")

    def value(**v):
        out, u = residual_block_norm(v.pop("stream"), v.pop("branch"), channels=16, lmax=2, **v)
        return (out.double() * t["p"].double()).sum() + (u.double() * t["q"].double()).sum()

    grads = torch.autograd.grad(value(**{k: t[k] for k in names}), [t[k] for k in names])
    h = 2.0 ** -7
    for name, g in zip(names, grads):
        step = torch.randn_like(t[name])
        at = {k: t[k].detach() for k in names}
        up, down = (float(value(**{**at, name: at[name] + s * h * step})) for s in (1, -1))
        slope = float((g.double() * step.double()).sum())
        # O(h^2) of the third derivative, and FP32 rounding of the value over 2 h
        scale = float(g.double().norm() * step.double().norm())
        assert abs((up - down) / (2 * h) - slope) <= 2e-3 * scale, name


def test_third_derivatives_and_weight_gradient_adjoints(cuda_device):
    """Past the kernels: d/dx of second derivatives, and derivatives of a weight gradient, against FP64."""
    from ictc_o3.backends.cuda.block_norm import Form, formula
    from ictc_o3.ops.block_norm import residual_block_norm
    t = inputs(6, 8, 1, seed=2)

    def third(d, op):
        out, u = op(d)
        (g,) = torch.autograd.grad([out, u], [d["branch"]], [d["p"], d["q"]], create_graph=True)
        (h,) = torch.autograd.grad(g, [d["branch"]], [d["d_branch"]], create_graph=True)
        return torch.autograd.grad(h.square().sum(), [d["stream"], d["branch"], d["gate"], d["scale"]])

    def weight(d, op):
        out, u = op(d)
        g = torch.autograd.grad([out, u], [d["scale"], d["pre_weight"]], [d["p"], d["q"]], create_graph=True)
        return torch.autograd.grad(sum(x.square().sum() for x in g), [d["stream"], d["branch"], d["p"], d["scale"]])

    def cuda(d):
        return residual_block_norm(d["stream"], d["branch"], post_weight=d["post_weight"], scale=d["scale"],
                                   gate=d["gate"], pre_weight=d["pre_weight"], channels=8, lmax=1)

    def plain(d):
        return formula(Form(8, 1, "mul_ir", 1e-6, True), d["stream"], d["branch"], d["gate"], d["post_weight"],
                       d["scale"], d["pre_weight"])

    d = {k: v.detach().double().cpu().requires_grad_() for k, v in t.items()}
    for f in (third, weight):
        for a, b in zip(f(t, cuda), f(d, plain)):
            # torch's own FP32 operations past the second order: far from a wrong term, which is O(1)
            assert float((a.double().cpu() - b).norm()) <= 1e-4 * float(b.norm()), f.__name__


def test_streams_and_capture(cuda_device):
    from ictc_o3.ops.block_norm import residual_block_norm
    t = inputs(300, 64, 2)
    form = {"channels": 64, "lmax": 2}

    def step():
        out = residual_block_norm(t["stream"], t["branch"], post_weight=t["post_weight"], scale=t["scale"],
                                  gate=t["gate"], pre_weight=t["pre_weight"], **form)
        first = torch.autograd.grad(out, [t["stream"], t["branch"], t["gate"]], [t["p"], t["q"]], create_graph=True)
        second = torch.autograd.grad(first, [t["branch"], t["scale"], t["pre_weight"]],
                                     [t["d_stream"], t["d_branch"], t["d_gate"]])
        return [x.detach() for x in (*out, *first, *second)]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        t["stream"].mul_(0.5)
        t["branch"].add_(0.1)
    graph.replay()
    fresh = step()
    assert all(torch.equal(a, b) for a, b in zip(held, fresh))


def test_first_call_inside_a_capture(cuda_device, monkeypatch):
    """Nothing that a first call sets up (status word, scratch size) needs to be there before a capture."""
    from ictc_o3.backends.cuda import block_norm
    from ictc_o3.ops.block_norm import block_norm_status, residual_block_norm
    monkeypatch.setattr(block_norm, "_status", {})
    monkeypatch.setattr(block_norm, "_partial_floats", {})
    t = inputs(50, 20, 1)

    def step():
        out = residual_block_norm(t["stream"], t["branch"], scale=t["scale"], norm=True, channels=20, lmax=1)
        return [x.detach() for x in (*out, *torch.autograd.grad(out, [t["branch"], t["scale"]], [t["p"], t["q"]]))]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))
    assert block_norm_status() == 0


def test_backward_inside_a_capture(cuda_device):
    """A captured backward pass gives the eager gradients, and is refused while a graph of the same leaves lives."""
    from ictc_o3.ops.block_norm import residual_block_norm
    t = inputs(50, 20, 1)
    leaves = [t[k].detach().requires_grad_() for k in ("stream", "branch", "scale")]

    def step():
        out = residual_block_norm(leaves[0], leaves[1], scale=leaves[2], norm=True, channels=20, lmax=1)
        return out, lambda: torch.autograd.backward(out, [t["p"], t["q"]])

    out, backward = step()
    backward()
    want = [x.grad.clone() for x in leaves]
    for x in leaves:
        x.grad = None
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            step()[1]()
    del out, backward, graph
    gc.collect()
    for x in leaves:
        x.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()[1]()
    graph.replay()
    assert all(torch.equal(x.grad, w) for x, w in zip(leaves, want))


def test_refusals(cuda_device):
    from ictc_o3.ops.block_norm import ResidualBlockNorm, degree_norm, residual_block_norm
    x = torch.zeros(4, 72, device=cuda_device)
    w = torch.ones(3, 8, device=cuda_device)
    form = {"channels": 8, "lmax": 2}
    for bad in ({"branch": x[:3]}, {"branch": x[:, :71]}, {"scale": w[:2]}, {"gate": x[:, :23]}, {"gate": x[:3, :24]},
                {"branch": x.double()}, {"branch": x.cpu()}, {"scale": w.cpu()}, {"gate": x[:, :24].half()}):
        with pytest.raises(ValueError):
            residual_block_norm(x, bad.pop("branch", x), **form, **bad)
    with pytest.raises(ValueError):
        degree_norm(x[0], w, **form)
    from ictc_o3.ops.block_norm import block_norm_status
    assert block_norm_status() == 0
    with pytest.raises(ValueError):
        block_norm_status("cpu")
    module = ResidualBlockNorm(8, 2, next_norm=False).to(cuda_device)
    out, none = module(x, x, torch.zeros(4, 3, 8, device=cuda_device))
    assert none is None and out.shape == x.shape
