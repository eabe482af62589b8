"""AdamW on the CUDA backend: tables, refusals and the 8-bit format (CPU only)."""
import ctypes

import pytest
import torch

from oracle import adamw_oracle


@pytest.mark.parametrize("turns", [1, 4])
def test_chunk_table_covers_every_value_once(turns):
    from ictc_o3.backends.cuda import _native
    from ictc_o3.backends.cuda.adamw import TensorTable
    chunk = turns * int(_native.library().ictc_adamw_turn_values())
    sizes = [1, chunk, chunk + 1, 0, 255, 256, 257, 5 * chunk - 3, 3]
    table = TensorTable(sizes, "cpu", turns)
    rows = table.chunks.tolist()
    assert table.chunk == chunk
    assert list(table.first_chunk) == [0, 1, 2, 4, 4, 5, 6, 7, 12, 13]
    assert table.starts == [0, 256, 256 + chunk, 2 * chunk + 512] + [
        2 * chunk + 512 + d for d in (0, 256, 512, 1024, 1024 + 5 * chunk)]
    for t, n in enumerate(sizes):
        mine = [r for r in rows if r[0] == t]
        assert sum(r[1] for r in mine) == n and all(0 < r[1] <= chunk for r in mine)
        assert [r[3] for r in mine] == list(range(len(mine)))
        assert [256 * r[2] for r in mine] == [table.starts[t] + k * chunk for k in range(len(mine))]
    assert table.values == table.starts[-1] + 256 and table.values == 256 * table.blocks


def test_turns_grow_with_the_total():
    from ictc_o3.backends.cuda.adamw import turns_of
    assert [turns_of(n) for n in (1, 700_000, 1_000_000, 3_000_000, 20_000_000, 10 ** 10)] == [1, 1, 2, 4, 8, 8]


def test_state_format_is_monotone_and_round_trips():
    for signed, least in ((True, 1.125 * 2.0 ** -15), (False, 1.125 * 2.0 ** -31)):
        grid = adamw_oracle.table(signed)[:128 if signed else 256]
        assert grid[0] == 0 and grid[1] == least and bool((grid[1:] > grid[:-1]).all())
        x = torch.cat([grid[grid <= 1.0].float(), torch.ones(256)])[:256]
        for r in (0, 65535):
            codes, byte = adamw_oracle.encode(x, torch.full((x.numel(),), r), signed)
            assert int(byte[0]) == 128                     # scale 2: the largest value 1 is half of it
            back = adamw_oracle.decode(codes, byte, signed)
            # the scale is twice the largest value, so the two lowest grid values lie below its least
            inside = x >= 2 * least
            assert torch.equal(back[inside].float(), x[inside])


@pytest.mark.parametrize("kwargs, error", [
    ({"state_bits": 16}, ValueError), ({"max_norm": 0.0}, ValueError), ({"max_norm": "1"}, TypeError),
    ({"ema_decay": 1.0}, ValueError), ({"seed": -1}, ValueError), ({"seed": 1 << 64}, ValueError),
    ({"skip_nonfinite": 1}, TypeError), ({"max_norm": float("nan")}, ValueError)])
def test_constructor_refuses(kwargs, error):
    from ictc_o3.optim import AdamW
    with pytest.raises(error):
        AdamW([torch.nn.Parameter(torch.zeros(3))], **kwargs)


@pytest.mark.parametrize("kwargs", [{"lr": -1.0}, {"lr": float("nan")}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)},
                                    {"eps": 0.0}, {"eps": 1e-42}, {"weight_decay": -1.0}])
def test_hyperparameters_are_checked(kwargs):
    from ictc_o3.optim import _hyperparameters
    with pytest.raises(ValueError):
        _hyperparameters({"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.0, **kwargs})


def test_host_and_non_fp32_parameters_are_refused():
    from ictc_o3.optim import AdamW
    for p in (torch.zeros(3), torch.zeros(3, dtype=torch.float64)):
        with pytest.raises(ValueError):
            AdamW([torch.nn.Parameter(p)])


def test_native_entry_points_validate_before_launching():
    from ictc_o3.backends.cuda import _native
    lib = _native.library()
    first = (ctypes.c_int64 * 2)(0, 1)
    ones = (ctypes.c_void_p * 1)(1)
    some = ctypes.c_void_p(1)
    common = [first, 1024, 32, some, some, None, None, None, some, some, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0.0, 0, 0]

    def step(**change):
        names = ["first_chunk", "chunk", "bits", "m", "v", "m_scale", "v_scale", "average", "steps", "rates", "lr", "b1", "b2", "eps",
                 "wd", "avg", "seed", "use_norm"]
        values = dict(zip(names, common), **change)
        return lib.ictc_adamw_step(change.pop("weights", ones), ones, 0, 1, some, *[values[n] for n in names], some,
                                   None)

    for change in ({"bits": 16}, {"bits": 8}, {"m": None}, {"steps": None}, {"rates": None}, {"b1": 1.0}, {"b2": -0.1}, {"eps": 0.0},
                   {"eps": 1e-50}, {"first_chunk": None},
                   {"chunk": 0}, {"chunk": 1000}, {"chunk": 1536}, {"chunk": 1 << 20}):
        assert step(**change) == -1, change
        assert "invalid" in lib.ictc_last_error().decode()
    assert lib.ictc_adamw_step(ones, ones, 0, -1, some, *common, some, None) == -1
    assert lib.ictc_adamw_step(ones, ones, 0, 1, some, *common, None, None) == -1
    assert lib.ictc_adamw_grad_norm(ones, 1, some, first, 1024, 0.0, 1, 0, some, None) == -1
    assert lib.ictc_adamw_grad_norm(None, 1, some, first, 1024, 1.0, 1, 0, some, None) == -1
    assert lib.ictc_adamw_decode(some, some, some, some, 255, some, some, None) == -1
    assert lib.ictc_adamw_decode(None, None, None, None, 256, None, None, None) == -1
    assert lib.ictc_adamw_decode(None, None, None, None, 0, None, None, None) == 0


def test_host_addresses():
    """The extension module refuses what is not a list of tensors and finds CPU tensors unfit (no GPU needed)."""
    from array import array
    from ictc_o3.backends.cuda._native import host_tensors
    host = host_tensors()
    params = [torch.nn.Parameter(torch.zeros(n)) for n in (3, 5)]
    sizes, weights, grads = array("q", [3, 5]), array("Q", [9, 9]), array("Q", [9, 9])
    args = (sizes.buffer_info()[0], 0, weights.buffer_info()[0], grads.buffer_info()[0], 1)
    assert host.gather(params, *args) == 0 and list(weights) == list(grads) == [0, 0]
    params[1].grad = torch.zeros(5)
    assert host.gather(params, *args) == -2                 # the second is not on the device
    version = [p._version for p in params]
    present = array("Q", [0, 7])
    host.changed(params, present.buffer_info()[0])
    assert [p._version - v for p, v in zip(params, version)] == [0, 1]
    for bad in (lambda: host.gather(tuple(params), *args), lambda: host.gather([1], *args),
                lambda: host.gather(params, *args[:3]), lambda: host.changed(params), lambda: host.gather(params, "x", *args[1:])):
        with pytest.raises(TypeError):
            bad()


def test_where_gradients_are_added_up():
    from ictc_o3.backends.cuda._native import host_tensors
    leaf = torch.zeros(2, requires_grad=True)
    for graph in (None, leaf * 2):      # on the CPU there is no stream
        assert host_tensors().accumulates_on_default_stream(leaf) is False
    with pytest.raises(TypeError):
        host_tensors().accumulates_on_default_stream(None)
