"""AdamW where a step or a state dict is out of the ordinary."""
import pytest
import torch

from oracle import adamw_oracle
from test_adamw_gpu import HYPER, make, within

pytestmark = pytest.mark.gpu


def snapshot(opt, params):
    return [x.detach().clone() for p in params for k, x in (("", p), *opt.state[p].items()) if k != "step"]


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_with_a_nonfinite_norm(bits, bad, cuda_device):
    """The factor min(1, max_norm / (|g| + 1e-6)) of a NaN norm is NaN and that of an infinite one 0: a NaN
    spoils the whole step (8-bit blocks then stay as they were), an infinity its own value, and the rest takes a
    step with zero gradients."""
    from ictc_o3.optim import AdamW
    sizes = [4000, 700, 3]
    params, twins = make(sizes, cuda_device, seed=21), make(sizes, cuda_device, seed=21)
    opts = [AdamW(x, **HYPER, state_bits=bits, max_norm=1.0, ema_decay=0.5, seed=4) for x in (params, twins)]
    for opt in opts:
        opt.step()
    params[0].grad[1234] = bad
    for q in twins:
        q.grad.zero_()
    kept = snapshot(opts[0], params)
    for opt in opts:
        opt.step()
    assert not torch.isfinite(opts[0].grad_norm)
    assert all(int(opts[0].state[p]["step"]) == 2 for p in params)
    if bad != bad:
        if bits == 32:
            assert all(bool(x.isnan().all()) for x in snapshot(opts[0], params))
        else:
            assert all(torch.equal(a, b) for a, b in zip(kept, snapshot(opts[0], params)))
        return
    spoilt = torch.zeros(4000, dtype=torch.bool, device=cuda_device)
    if bits == 32:
        spoilt[1234] = True
        assert torch.isnan(params[0][1234]) and torch.isnan(opts[0].state[params[0]]["ema"][1234])
    else:
        spoilt[1234 // 256 * 256:1234 // 256 * 256 + 256] = True
        assert torch.equal(params[0][spoilt], kept[0][spoilt])
    for p, q in zip(params, twins):
        good = ~spoilt if p is params[0] else slice(None)
        assert torch.equal(p[good], q[good])
        for key in ("exp_avg", "exp_avg_sq", "ema"):
            assert torch.equal(opts[0].state[p][key][good], opts[1].state[q][key][good])


@pytest.mark.parametrize("decay", [0.0, 0.3, 0.5, 0.9, 0.999, 0.9999, 0.99999])
@pytest.mark.parametrize("bits", [32, 8])
def test_weight_average(bits, decay, cuda_device):
    """d average + (1 - d) weight: two half steps for the rounded factor times the distance, one for the
    difference and one for the sum, and an average equal to its weights stays there."""
    from ictc_o3.optim import AdamW
    params = make([3000, 5], cuda_device, seed=31)
    opt = AdamW(params, **HYPER, state_bits=bits, ema_decay=decay)
    saved = opt.state_dict()
    old = [p.detach() * 1.5 - 0.25 for p in params]
    for i, e in enumerate(old):
        saved["state"][i] = {**saved["state"][i], "ema": e}
    opt.load_state_dict(saved)
    opt.step()
    share = min(decay, 1 - decay)
    for p, e in zip(params, old):
        w, e = p.detach().double(), e.double()
        want = decay * e + (1 - decay) * w
        within(opt.state[p]["ema"], want, 1.01 * adamw_oracle.U * (2 * share * (w - e).abs() + want.abs()), "average")
    still = make([700, 5], cuda_device, seed=32)
    opt = AdamW(still, lr=0.0, weight_decay=0.0, state_bits=bits, ema_decay=decay)
    start = [p.detach().clone() for p in still]
    for _ in range(300):
        opt.step()
    for p, w in zip(still, start):
        assert torch.equal(p, w) and torch.equal(opt.state[p]["ema"], w)


@pytest.mark.parametrize("ema", [None, 0.9])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dicts_with_missing_entries(bits, ema, cuda_device):
    """Parameters without an entry start anew, all of them or some."""
    from ictc_o3.optim import AdamW
    params = make([700, 0, 300], cuda_device, seed=41)
    opt = AdamW(params, **HYPER, state_bits=bits, ema_decay=ema)
    for kept in ((), (0,), (1,), (0, 2)):
        opt.step()
        opt.step()
        saved = opt.state_dict()
        saved = {"state": {i: {k: v.clone() for k, v in saved["state"][i].items()} for i in kept},
                 "param_groups": saved["param_groups"]}
        opt.load_state_dict(saved)
        for i, p in enumerate(params):
            state = opt.state[p]
            if i in kept:
                assert int(state["step"]) == 2
                assert all(torch.equal(state[k], v) for k, v in saved["state"][i].items())
            else:
                assert int(state["step"]) == 0 and not state["exp_avg"].any() and not state["exp_avg_sq"].any()
                assert ema is None or torch.equal(state["ema"], p.detach())
                assert bits == 32 or bool((state["exp_avg_exponent"] == 1).all())
        for p in params:
            opt.state[p]["step"].zero_()
    if bits == 32:      # the library's, before its first step
        opt.load_state_dict(torch.optim.AdamW(make([700, 0, 300], cuda_device), lr=0.125).state_dict())
        assert opt.param_groups[0]["lr"] == 0.125 and not opt.state[params[0]]["exp_avg"].any()


def test_hooks_of_loading_run(cuda_device):
    from ictc_o3.optim import AdamW
    opt, calls = AdamW(make([300], cuda_device), lr=0.5), []

    def before(optimizer, state_dict):
        calls.append(("before", optimizer is opt, optimizer.param_groups[0]["lr"]))
        groups = [{**g, "lr": 2 * g["lr"]} for g in state_dict["param_groups"]]
        return {**state_dict, "param_groups": groups}

    removed = opt.register_load_state_dict_pre_hook(lambda optimizer, state_dict: calls.append("removed"))
    opt.register_load_state_dict_pre_hook(before)
    opt.register_load_state_dict_post_hook(lambda optimizer: calls.append(("after", optimizer.param_groups[0]["lr"])))
    removed.remove()
    other = AdamW(make([300], cuda_device), lr=0.125)
    other.step()
    saved = other.state_dict()
    opt.load_state_dict(saved)
    assert calls == [("before", True, 0.5), ("after", 0.25)]
    assert saved["param_groups"][0]["lr"] == 0.125          # the caller's dict is what it was
    (p,), (q,) = opt.param_groups[0]["params"], other.param_groups[0]["params"]
    assert torch.equal(opt.state[p]["exp_avg"], other.state[q]["exp_avg"]) and int(opt.state[p]["step"]) == 1


def test_seed_travels_with_8_bit_states(cuda_device):
    """A resumed optimizer rounds as the saved one would have, whatever seed it was built with."""
    from ictc_o3.optim import AdamW
    params, twins = make([5000, 33], cuda_device, seed=51), make([5000, 33], cuda_device, seed=51)
    opt, other = AdamW(params, state_bits=8, seed=(1 << 64) - 3), AdamW(twins, state_bits=8, seed=8)
    opt.step()
    for p, q in zip(params, twins):
        q.data.copy_(p.data)
    saved = opt.state_dict()
    other.load_state_dict(saved)
    assert other.seed == (1 << 64) - 3
    opt.step()
    other.step()
    assert all(torch.equal(a, b) for a, b in zip(snapshot(opt, params), snapshot(other, twins)))
    del saved["seed"]                 # one of an earlier release keeps the optimizer's own
    third = AdamW(make([5000, 33], cuda_device), state_bits=8, seed=8)
    third.load_state_dict(saved)
    assert third.seed == 8
    for bad in (-1, 1 << 64, 0.5, True, None):
        kept = snapshot(other, twins)
        with pytest.raises(ValueError, match="seed"):
            other.load_state_dict({**saved, "state": {}, "seed": bad})
        assert all(torch.equal(a, b) for a, b in zip(kept, snapshot(other, twins)))
    assert "seed" not in AdamW(make([3], cuda_device)).state_dict()


def test_edited_state_dicts_load(cuda_device):
    """Values replaced in a state dict change the optimizer when it is loaded, and not before."""
    from ictc_o3.optim import AdamW
    (p,) = params = make([700], cuda_device, seed=61)
    opt = AdamW(params, **HYPER, ema_decay=0.9)
    opt.step()
    saved, m = opt.state_dict(), opt.state[p]["exp_avg"].clone()
    saved["state"][0]["ema"] = torch.full((700,), 2.0, device=cuda_device)
    saved["state"][0]["exp_avg"] = 3 * m
    assert torch.equal(opt.state[p]["exp_avg"], m)
    opt.load_state_dict(saved)
    assert torch.equal(opt.state[p]["exp_avg"], 3 * m) and torch.equal(opt.moments()[0][:700], 3 * m)
    assert bool((opt.averages()[:700] == 2.0).all())
    opt.step()
    assert torch.equal(opt.state[p]["ema"], opt.averages()[:700]) and bool((opt.averages()[:700] != 2.0).any())


@pytest.mark.parametrize("before, after", [((0.9, 0.9999999), (0.9, 0.99999991)), ((0.99999991, 0.99), (0.9999999, 0.99)),
                                           ((0.0, 0.99), (0.9, 0.0))])
def test_betas_that_fp32_cannot_tell_apart(before, after, cuda_device):
    """Bias corrections left behind by a step hold for its own betas only."""
    from ictc_o3.optim import AdamW
    params, twins = make([700, 33], cuda_device, seed=71), make([700, 33], cuda_device, seed=71)
    opt = AdamW(params, lr=0.1, betas=before)
    opt.step()
    for p, q in zip(params, twins):
        q.data.copy_(p.data)
    fresh = AdamW(twins, lr=0.1, betas=before)
    fresh.load_state_dict(opt.state_dict())              # copies no bias corrections
    for o in (opt, fresh):
        o.param_groups[0]["betas"] = after
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    for p, q in zip(params, twins):
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.state[p][k], fresh.state[q][k])


@pytest.mark.parametrize("bits", [32, 8])
def test_without_the_extension_module(bits, cuda_device, monkeypatch):
    """Where it was not built, addresses and checks go through Python, with the same results and refusals."""
    from ictc_o3.backends.cuda import _native
    from ictc_o3.optim import AdamW
    sets = [make([5000, 0, 33, 7], cuda_device, seed=81) for _ in range(2)]
    opts = [AdamW(sets[0], state_bits=bits, max_norm=1.0, ema_decay=0.9)]

    def missing():
        raise _native.NativeError("not built")

    monkeypatch.setattr(_native, "host_tensors", missing)
    opts.append(AdamW(sets[1], state_bits=bits, max_norm=1.0, ema_decay=0.9))
    for params in sets:
        params[3].grad = None
    versions = [p._version for p in sets[1]]
    for _ in range(2):
        for opt in opts:
            opt.step()
    assert all(torch.equal(a, b) for a, b in zip(*(snapshot(o, p) for o, p in zip(opts, sets))))
    assert [p._version > v for p, v in zip(sets[1], versions)] == [True, True, True, False]
    sets[1][0].data = torch.zeros(5, device=cuda_device)
    sets[1][0].grad = torch.zeros(5, device=cuda_device)
    with pytest.raises(ValueError, match="has changed"):
        opts[1].step()


def test_negated_parameters_are_refused(cuda_device):
    """A lazily negated view stores the other sign: steps would go uphill."""
    from ictc_o3.optim import AdamW
    negated = torch._neg_view(torch.ones(5, device=cuda_device))
    with pytest.raises(ValueError, match="negated"):
        AdamW([torch.nn.Parameter(negated)])
    p = torch.nn.Parameter(torch.ones(5, device=cuda_device))
    opt = AdamW([p])
    p.data = negated
    p.grad = torch.ones(5, device=cuda_device)
    with pytest.raises(ValueError, match="has changed"):
        opt.step()


@pytest.mark.parametrize("native", [True, False])
def test_changed_groups_are_refused(native, cuda_device, monkeypatch):
    """Addresses lie in arrays of the parameters at construction: other lists must not be read from them."""
    from ictc_o3.backends.cuda import _native
    from ictc_o3.optim import AdamW

    def missing():
        raise _native.NativeError("not built")

    if not native:
        monkeypatch.setattr(_native, "host_tensors", missing)
    a, b, c, d = make([30, 5, 7, 5], cuda_device)
    opt = AdamW([{"params": [a, b]}, {"params": [c], "lr": 1e-2}])
    opt.step()
    kept = snapshot(opt, [a, b, c])
    first, second = opt.param_groups
    for groups in ([{**first, "params": [a, b, d]}, second], [{**first, "params": [a]}, second], [first], [second, first],
                   [{**first, "params": [a, d]}, second], [first, second, {**second, "params": [d]}],
                   [first, {**second, "params": []}], [first, {**second, "params": [c, d, d, d]}], []):
        opt.param_groups = groups
        with pytest.raises(ValueError, match="fixed"):
            opt.step()
        assert all(torch.equal(x, y) for x, y in zip(kept, snapshot(opt, [a, b, c])))
    opt.param_groups = [{**first, "params": (a, b)}, second]      # the same ones in another container
    opt.step()
    assert int(opt.state[c]["step"]) == 2


def test_8_bit_codes_with_clipping_are_exact(cuda_device):
    """The clip factor that the first kernel left is one more FP32 product: codes equal the restatement's."""
    from ictc_o3.optim import AdamW
    from test_adamw_gpu import random_state
    params = make([1, 255, 257, 9001], cuda_device, seed=91)
    total = float(torch.cat([p.grad.double() for p in params]).norm())
    opt = AdamW(params, **HYPER, state_bits=8, max_norm=0.3 * total, seed=77)
    before = random_state(opt, 3)
    opt.step()
    clip = opt._table.workspace[12:16].view(torch.float32).cpu()
    assert abs(float(clip) - 0.3 * total / (total + 1e-6)) <= 4 * adamw_oracle.U
    b1, b2 = (torch.tensor(b, dtype=torch.float32) for b in HYPER["betas"])
    c1, c2 = (torch.tensor(1 - b, dtype=torch.float32) for b in HYPER["betas"])
    for p, (steps, start, m, v) in zip(params, before):
        g = p.grad.cpu() * clip
        r_m, r_v = adamw_oracle.random_bits(start, p.numel(), steps + 1, opt.seed)
        for key, x, r, signed in (("exp_avg", m.float() * b1 + g * c1, r_m, True),
                                  ("exp_avg_sq", v.float() * b2 + (g * g) * c2, r_v, False)):
            codes, byte = adamw_oracle.encode(x.reshape(-1), r, signed)
            assert torch.equal(opt.state[p][key].cpu().view(-1), codes)
            assert torch.equal(opt.state[p][key + "_exponent"].cpu(), byte)


def test_state_of_a_users_own(cuda_device):
    """What a user keeps in the optimizer's state beside the tensors' entries travels with the state dict."""
    from ictc_o3.optim import AdamW
    opt = AdamW(make([30], cuda_device))
    opt.state["epoch"] = 3
    opt.step()
    saved = opt.state_dict()
    assert saved["state"]["epoch"] == 3 and set(saved["state"][0]) == {"step", "exp_avg", "exp_avg_sq"}
    opt.load_state_dict(saved)
    opt.step()
    assert int(opt.state[opt.param_groups[0]["params"][0]]["step"]) == 2
