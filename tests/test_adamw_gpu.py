"""AdamW over many tensors against FP64 (32-bit moments) and code by code (8-bit moments)."""
import copy

import pytest
import torch

from oracle import adamw_oracle

pytestmark = pytest.mark.gpu

HYPER = {"lr": 3e-3, "betas": (0.9, 0.99), "eps": 1e-8, "weight_decay": 0.02}
SIZES = {"one": [1], "edges": [3, 4, 5, 255, 256, 257, 2047, 2048, 2049, 1], "empty": [0, 7, 0, 1025],
         "many": [1 + 37 * k % 911 for k in range(500)], "large": [1_300_003], "turns": [3_100_001, 9000, 40_000, 255, 3_000_000]}


def make(sizes, device, seed=0, offset=0):
    """Parameters (views `offset` values into their buffers) with gradients of varied size."""
    gen = torch.Generator(device=device).manual_seed(seed)
    params = []
    for k, n in enumerate(sizes):
        p = torch.nn.Parameter(torch.randn(n + offset, device=device, generator=gen)[offset:])
        p.grad = (torch.randn(n + offset, device=device, generator=gen) * 10.0 ** -(k % 6))[offset:]
        params.append(p)
    return params


def random_state(opt, seed, steps=7):
    """Load plausible moments and step counts; returns the FP64 moments per parameter."""
    saved = opt.state_dict()
    out, i = [], 0
    for group in opt.param_groups:
        for p in group["params"]:
            gen = torch.Generator(device=p.device).manual_seed(seed * 1000 + i)
            g = p.grad if p.grad is not None else torch.randn_like(p)
            m = torch.randn(p.shape, device=p.device, generator=gen) * g.abs().mean() if p.numel() else p.detach()
            v = (torch.rand(p.shape, device=p.device, generator=gen) + 0.1) * g.square()
            entry = {"step": steps + i % 3}
            start = opt._table.starts[i]
            if opt.state_bits == 32:
                entry |= {"exp_avg": m, "exp_avg_sq": v}
                out.append((entry["step"], start, m.detach().double(), v.double()))
            else:
                r1 = torch.randint(0, 65536, (p.numel(),), generator=torch.Generator().manual_seed(i))
                for key, x, signed in (("exp_avg", m, True), ("exp_avg_sq", v, False)):
                    codes, byte = adamw_oracle.encode(x.detach(), r1, signed)
                    entry[key] = codes.view(p.shape)
                    entry[key + "_exponent"] = byte
                out.append((entry["step"], start,
                            adamw_oracle.decode(entry["exp_avg"], entry["exp_avg_exponent"], True),
                            adamw_oracle.decode(entry["exp_avg_sq"], entry["exp_avg_sq_exponent"], False)))
            if opt.ema_decay is not None:
                entry["ema"] = p.detach() * 1.5
            saved["state"][i] = entry
            i += 1
    opt.load_state_dict(saved)
    return out


def within(actual, expected, bound, what):
    """|actual - expected| <= bound, and where the bound passes below FP32's range one smallest step."""
    err = (actual.double().cpu() - expected.double().cpu()).abs()
    worst = float((err - bound.cpu() - 1.5e-45).max()) if err.numel() else 0.0
    assert worst <= 0, f"{what}: error exceeds its bound by {worst:.3e}"


@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("ema", [None, 0.9])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("name", list(SIZES))
def test_32_bit_step_against_fp64(name, offset, ema, clip, cuda_device):
    from ictc_o3.optim import AdamW
    params = make(SIZES[name], cuda_device, offset=offset)
    total = torch.cat([p.grad.double().reshape(-1) for p in params]).norm()
    opt = AdamW(params, **HYPER, max_norm=0.25 * float(total) if clip else None, ema_decay=ema)
    before = random_state(opt, 1)
    old = [p.detach().double() for p in params]
    opt.step()
    factor = 1.0
    if clip:
        assert abs(float(opt.grad_norm) - float(total)) <= 2.0 ** -23 * float(total)
        factor = min(1.0, opt.max_norm / (float(total) + 1e-6))
    for p, w, (steps, _, m, v) in zip(params, old, before):
        args = (w, p.grad.double(), m, v, steps + 1)
        new = adamw_oracle.step(*args, **HYPER, clip=factor)
        bounds = adamw_oracle.step_bounds(*args, **HYPER, clip=factor, clipped=clip)
        state = opt.state[p]
        assert int(state["step"]) == steps + 1
        for what, got, want, bound in zip(("weight", "exp_avg", "exp_avg_sq"),
                                          (p.detach(), state["exp_avg"], state["exp_avg_sq"]), new, bounds):
            within(got, want, bound, f"{name} {what}")
        if ema is not None:
            # both products: constant 1, product 1; the sum 1; plus the weight's error
            want = ema * 1.5 * w + (1 - ema) * new[0]
            slack = adamw_oracle.U * 3.1 * (ema * 1.5 * w.abs() + (1 - ema) * new[0].abs()) + (1 - ema) * bounds[0]
            # the old average 1.5 w was itself rounded once
            within(state["ema"], want, slack + adamw_oracle.U * 1.6 * w.abs(), f"{name} ema")


@pytest.mark.parametrize("name", list(SIZES))
def test_8_bit_codes_are_exact(name, cuda_device, monkeypatch):
    """Without clipping every operation before the rounding is a single FP32 operation, so the codes
    equal those of the FP32 restatement; weights meet the FP32 bounds."""
    from ictc_o3.optim import AdamW
    sizes = {"large": [200_003], "turns": [9001, 70_000]}.get(name, SIZES[name])
    params = make(sizes, cuda_device, seed=3, offset=1 if name == "edges" else 0)
    if name == "turns":      # blocks of several turns, as many values have them
        from ictc_o3.backends.cuda import adamw
        monkeypatch.setattr(adamw, "turns_of", lambda total: 8)
    opt = AdamW(params, **HYPER, state_bits=8, seed=0x0123456789ABCDEF)
    before = random_state(opt, 2)
    old = [p.detach().double() for p in params]
    opt.step()
    b1, b2 = (torch.tensor(b, dtype=torch.float32) for b in HYPER["betas"])
    c1, c2 = (torch.tensor(1 - b, dtype=torch.float32) for b in HYPER["betas"])
    values = [x.cpu() for x in opt.moments()]
    for p, w, (steps, start, m, v) in zip(params, old, before):
        g = p.grad.cpu()
        new_m = (m.float() * b1 + g * c1).reshape(-1)
        new_v = (v.float() * b2 + (g * g) * c2).reshape(-1)
        r_m, r_v = adamw_oracle.random_bits(start, p.numel(), steps + 1, opt.seed)
        state = opt.state[p]
        for k, (key, x, r, signed) in enumerate((("exp_avg", new_m, r_m, True), ("exp_avg_sq", new_v, r_v, False))):
            codes, byte = adamw_oracle.encode(x, r, signed)
            assert torch.equal(state[key].cpu().view(-1), codes) and torch.equal(state[key + "_exponent"].cpu(), byte)
            want = adamw_oracle.decode(codes, byte, signed)
            assert torch.equal(values[k][start:start + p.numel()].double(), want.bfloat16().double())
        args = (w.cpu(), g.double(), m, v, steps + 1)
        within(p.detach(), adamw_oracle.step(*args, **HYPER)[0], adamw_oracle.step_bounds(*args, **HYPER, approximate=True)[0],
               name)


def test_matches_library_over_several_steps(cuda_device):
    """Five steps from zero next to torch.optim.AdamW in FP64, gradients changing, two groups."""
    from ictc_o3.optim import AdamW
    sizes = [129, 4000, 17]
    params = make(sizes, cuda_device, seed=5)
    twins = [torch.nn.Parameter(p.detach().double()) for p in params]
    groups = [{"params": params[:2]}, {"params": params[2:], "lr": 1e-2, "weight_decay": 0.0, "betas": (0.8, 0.95)}]
    opt = AdamW(groups, **HYPER)
    ref = torch.optim.AdamW([{"params": twins[:2]}, {**groups[1], "params": twins[2:]}], **HYPER)
    for k in range(5):
        for p, q, fresh in zip(params, twins, make(sizes, cuda_device, seed=50 + k)):
            p.grad, q.grad = fresh.grad, fresh.grad.double()
        opt.param_groups[0]["lr"] = ref.param_groups[0]["lr"] = HYPER["lr"] / (k + 1)
        opt.step()
        ref.step()
    for p, q in zip(params, twins):
        # each of five steps is off by at most some 25 half steps of max(|w|, lr)
        within(p.detach(), q.detach(), 5 * 25 * adamw_oracle.U * (q.detach().abs() + 3e-2), "weights")


def test_steps_and_betas_may_change_between_steps(cuda_device):
    """Bias corrections follow the step counters and betas of the moment, whatever the last step left."""
    from ictc_o3.optim import AdamW
    for change in (lambda o: o.state[o.param_groups[0]["params"][0]]["step"].fill_(400),
                   lambda o: o.param_groups[0].update(betas=(0.5, 0.75)),
                   lambda o: o.state[o.param_groups[0]["params"][1]]["step"].zero_()):
        params = make([700, 33], cuda_device)
        opt = AdamW(params, **HYPER)
        for _ in range(3):
            opt.step()
        change(opt)
        hyper = {**HYPER, "betas": opt.param_groups[0]["betas"]}
        before = [(p.detach().double(), p.grad.double(), opt.state[p]["exp_avg"].double(),
                   opt.state[p]["exp_avg_sq"].double(), int(opt.state[p]["step"]) + 1) for p in params]
        opt.step()
        for p, args in zip(params, before):
            within(p.detach(), adamw_oracle.step(*args, **hyper)[0], adamw_oracle.step_bounds(*args, **hyper)[0], "weight")


def test_absent_gradients_leave_tensors_alone(cuda_device):
    from ictc_o3.optim import AdamW
    for bits in (32, 8):
        params = make([300, 300, 5], cuda_device)
        params[1].grad = None
        opt = AdamW(params, state_bits=bits, ema_decay=0.9)
        w = params[1].detach().clone()
        opt.step()
        opt.step()
        assert [int(opt.state[p]["step"]) for p in params] == [2, 0, 2]
        assert torch.equal(params[1].detach(), w) and not opt.state[params[1]]["exp_avg"].any()
        assert torch.equal(opt.state[params[1]]["ema"], w)
        for p in params:
            p.grad = None
        opt.step()
        assert [int(opt.state[p]["step"]) for p in params] == [2, 0, 2]


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("bits", [32, 8])
def test_nonfinite_gradients(bits, bad, cuda_device):
    from ictc_o3.optim import AdamW

    def snapshot(opt, params):
        return [x.detach().clone() for p in params for x in (p, *opt.state[p].values())]

    params = make([4000, 700], cuda_device)
    opt = AdamW(params, state_bits=bits, skip_nonfinite=True, ema_decay=0.5)
    opt.step()
    params[0].grad[1234] = bad
    kept = snapshot(opt, params)
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(kept, snapshot(opt, params)))
    assert not torch.isfinite(opt.grad_norm)
    params[0].grad[1234] = 0.0
    opt.step()
    assert int(opt.state[params[0]]["step"]) == 2 and torch.isfinite(opt.grad_norm)
    # without skipping: FP32 moments take it in at that value, 8-bit ones keep its block
    params = make([4000, 700], cuda_device)
    params[0].grad[1234] = bad
    opt = AdamW(params, state_bits=bits)
    w = params[0].detach().clone()
    opt.step()
    changed = (params[0].detach() != w) | params[0].detach().isnan()
    if bits == 32:
        assert torch.isnan(params[0][1234]) and int(params[0].isnan().sum()) == 1
    else:
        block = torch.arange(4000, device=cuda_device) // 256 == 1234 // 256
        assert not changed[block].any() and changed[~block].all()
        assert not opt.state[params[0]]["exp_avg"][block].any()


def test_clipping_spans_launches_and_groups(cuda_device):
    """600 tensors need three launches; the norm is that of all of them, and zero gradients do not divide by zero."""
    from ictc_o3.optim import AdamW
    params = make([1 + 13 * k % 700 for k in range(600)], cuda_device, seed=8)
    total = float(torch.cat([p.grad.double() for p in params]).norm())
    opt = AdamW([{"params": params[:100]}, {"params": params[100:], "lr": 1e-2}], max_norm=1.0)
    opt.step()
    assert abs(float(opt.grad_norm) - total) <= 2.0 ** -23 * total
    for p in params:
        p.grad.zero_()
    before = [p.detach().clone() for p in params]
    opt.step()
    assert float(opt.grad_norm) == 0.0 and all(torch.isfinite(p).all() for p in params)
    assert any(not torch.equal(a, b) for a, b in zip(before, params))      # moments carry on


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(bits, cuda_device):
    from ictc_o3.optim import AdamW
    sets = [make([5000, 33], cuda_device, seed=4) for _ in range(2)]
    opts = [AdamW(p, state_bits=bits, max_norm=1.0, ema_decay=0.9, seed=5) for p in sets]
    for opt in opts:
        opt.step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        opts[0].step()
    for k in range(3):
        for p, q in zip(*sets):
            p.grad.mul_(0.5 + k)
            q.grad.mul_(0.5 + k)
        graph.replay()
        version = sets[0][0]._version
        opts[0].mark_updated()
        assert sets[0][0]._version > version
        opts[1].step()
    for p, q in zip(*sets):
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opts[0].state[p].values(),
                                                                            opts[1].state[q].values()))


def test_other_stream_and_strided_gradient(cuda_device):
    from ictc_o3.optim import AdamW
    a, b = (torch.nn.Parameter(torch.ones(48, 80, device=cuda_device)) for _ in range(2))
    a.grad = torch.randn(80, 48, device=cuda_device).t()
    b.grad = a.grad.contiguous()
    x, y = AdamW([a]), AdamW([b])
    y.step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x.step()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(a, b)


def test_negated_view_as_gradient(cuda_device):
    """An imaginary part of a lazily conjugated tensor stores the values with the other sign."""
    from ictc_o3.optim import AdamW
    a, b = (torch.nn.Parameter(torch.zeros(1, device=cuda_device)) for _ in range(2))
    a.grad = torch.full((1,), 1 + 2j, device=cuda_device).conj().imag
    assert a.grad.is_neg() and a.grad.is_contiguous()
    b.grad = a.grad.resolve_neg()
    for p in (a, b):
        AdamW([p], **HYPER).step()
    assert float(a) == float(b) > 0


def test_tiny_gradients_and_epsilon(cuda_device):
    """Second moments below FP32's normal range still divide (no flush to zero), in both forms."""
    from ictc_o3.optim import AdamW
    hyper = {**HYPER, "eps": 1e-24}
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.randn(700, device=cuda_device))
        p.grad = torch.randn(700, device=cuda_device) * 3e-20
        w, g, zero = p.detach().double(), p.grad.double(), torch.zeros(700, dtype=torch.float64, device=cuda_device)
        opt = AdamW([p], **hyper, state_bits=bits)
        opt.step()
        # v = (1 - b2) g^2 is some 1e-41, a multiple of 2^-149: its root is off by up to 2^-149 / (2 root), and the
        # quotient, of size 1, by that over the root
        v = 0.01 * g * g
        want = adamw_oracle.step(w, g, zero, zero, 1, **hyper)[0]
        loose = hyper["lr"] * 2.0 ** -149 / v.clamp_min(2.0 ** -149) * 2
        fine = v > 64 * 2.0 ** -149
        bound = adamw_oracle.step_bounds(w, g, zero, zero, 1, **hyper, approximate=bits == 8)[0] + loose
        assert fine.sum() > 300 and bool(((p.detach().double() - want).abs() <= bound)[fine].all())


def test_results_are_reproducible_and_seeded(cuda_device):
    from ictc_o3.optim import AdamW

    def states(seed):
        params = make([40_000, 999], cuda_device, seed=6)
        opt = AdamW(params, state_bits=8, max_norm=0.5, seed=seed)
        for _ in range(4):
            opt.step()
        return [x.clone() for x in opt.moments()] + [p.detach().clone() for p in params]

    a, b, c = states(1), states(1), states(2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert not torch.equal(a[0], c[0]) and not torch.equal(a[1], c[1])


def test_8_bit_moments_follow_their_averages(cuda_device):
    """Rounding is unbiased: after many steps with one gradient the stored moments, averaged over
    equal values, approach g and g^2 although a step moves the second by a fiftieth of a code step."""
    from ictc_o3.optim import AdamW
    n = 65536
    p = torch.nn.Parameter(torch.zeros(n, device=cuda_device))
    p.grad = torch.full((n,), 0.02, device=cuda_device)
    p.grad[::256] = 0.05                                   # sets the blocks' scales
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.99), state_bits=8, seed=9)
    steps = 600
    for _ in range(steps):
        opt.step()
    m, v = (x.double() for x in opt.moments())
    keep = torch.arange(n, device=cuda_device) % 256 != 0
    # a stored value differs from the average by at most some code steps (1/8); the mean of 65,000 independent ones
    # by a 250th of that; 2% leaves room for both
    assert abs(float(m[keep].mean()) / 0.02 - 1) < 0.02
    assert abs(float(v[keep].mean()) / 0.0004 / (1 - 0.99 ** steps) - 1) < 0.02
    p.grad.zero_()
    for _ in range(100):
        opt.step()
    later = opt.moments()[1].double()
    assert abs(float(later[keep].mean()) / (float(v[keep].mean()) * 0.99 ** 100) - 1) < 0.05


def test_state_dicts(cuda_device):
    from ictc_o3.optim import AdamW
    for bits in (32, 8):
        params = make([700, 3], cuda_device)
        opt = AdamW(params, **HYPER, state_bits=bits, ema_decay=0.9, seed=3)
        opt.step()
        twins = make([700, 3], cuda_device)
        for q, p in zip(twins, params):
            q.data.copy_(p.data)
        other = AdamW(twins, state_bits=bits, ema_decay=0.9, seed=3)
        other.load_state_dict(copy.deepcopy(opt.state_dict()))
        opt.step()
        other.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opt.state[p].values(),
                                                                                other.state[q].values()))
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(make([700, 3], cuda_device), state_bits=8).load_state_dict(AdamW(make([700, 3], cuda_device)).state_dict())
    bad = copy.deepcopy(opt.state_dict())
    bad["state"][0]["exp_avg_exponent"][0] = 255
    with pytest.raises(ValueError, match="1..253"):
        opt.load_state_dict(bad)
    # a scheduler continues where it was
    first = AdamW(make([5], cuda_device), lr=1e-2)
    schedule = torch.optim.lr_scheduler.StepLR(first, 1, 0.5)
    first.step()
    schedule.step()
    second = AdamW(make([5], cuda_device), lr=1.0)
    second.load_state_dict(first.state_dict())
    assert second.param_groups[0]["initial_lr"] == 1e-2
    torch.optim.lr_scheduler.StepLR(second, 1, 0.5, last_epoch=schedule.last_epoch).step()
    assert second.param_groups[0]["lr"] < 5e-3 + 1e-9
    with pytest.raises(ValueError, match="parameter groups"):
        AdamW(make([700], cuda_device)).load_state_dict(opt.state_dict())
    # the library's own state continues here
    params = make([900], cuda_device)
    ref = torch.optim.AdamW(params, **HYPER)
    ref.step()
    mine = AdamW(make([900], cuda_device), **HYPER)
    mine.load_state_dict(ref.state_dict())
    p = mine.param_groups[0]["params"][0]
    assert torch.equal(mine.state[p]["exp_avg"], ref.state[params[0]]["exp_avg"]) and int(mine.state[p]["step"]) == 1


def test_refusals(cuda_device):
    from ictc_o3.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(64, device=cuda_device))
    with pytest.raises(ValueError):
        AdamW([{"params": [p]}, {"params": [p]}])
    whole = torch.zeros(64, device=cuda_device)
    with pytest.raises(ValueError, match="share memory"):
        AdamW([torch.nn.Parameter(whole[:40]), torch.nn.Parameter(whole[39:])])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.nn.Parameter(torch.zeros(4, 8, device=cuda_device).t())])
    opt = AdamW([p])
    with pytest.raises(ValueError, match="fixed"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2, device=cuda_device))]})
    with pytest.raises(TypeError):
        copy.deepcopy(opt)
    p.grad = torch.zeros(64, device=cuda_device)
    opt.param_groups[0]["lr"] = torch.tensor(1e-3)
    with pytest.raises(TypeError):
        opt.step()
    opt.param_groups[0]["lr"] = 1e-3
    q = torch.nn.Parameter(torch.zeros(64, device=cuda_device))
    q.grad = torch.zeros(64, device=cuda_device).to_sparse()
    with pytest.raises(ValueError, match="dense"):
        AdamW([q]).step()
    p.grad = None
    p.data = torch.zeros(32, device=cuda_device)
    p.grad = torch.zeros(32, device=cuda_device)
    with pytest.raises(ValueError, match="has changed"):
        opt.step()


def test_a_step_renews_what_a_model_derives_from_its_weights(cuda_device):
    """Packed radial weights and folded contraction tables are kept per weight version: after a step the model
    computes with the new weights."""
    from ictc_o3.optim import AdamW
    from test_model_gpu import brute_neighbors, build_models, random_system
    pos, species, side = random_system(30, seed=11)
    args = [t.to(cuda_device) for t in (pos.float(), species, *brute_neighbors(pos, side, 5.0))]
    args[-1] = args[-1].float()
    model, _ = build_models(lmax=2)
    model = model.to(cuda_device)
    weights = [p for p in model.parameters() if p.requires_grad]
    opt = AdamW(weights, lr=1e-2)
    energy, _ = model.energy_and_forces(*args, training=True)
    for p, g in zip(weights, torch.autograd.grad(energy.sum(), weights, allow_unused=True)):
        p.grad = g
    opt.step()
    after, forces = model.energy_and_forces(*args)
    fresh = copy.deepcopy(model)                 # rebuilds all derived state
    e2, f2 = fresh.energy_and_forces(*args)
    assert torch.equal(after, e2) and torch.equal(forces, f2)
    assert abs(float(after - energy)) > 1e-3 * abs(float(energy))
