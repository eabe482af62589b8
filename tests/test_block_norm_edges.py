"""Block norms in calls that they refuse (CPU only)."""
import pytest
import torch


def test_tracing_is_refused():
    """While torch.jit.trace runs, a tensor's sizes are host tensors: their addresses must not reach a kernel as row
    counts."""
    from ictc_o3.ops.block_norm import degree_norm, residual_block_norm
    x, w = torch.zeros(4, 72), torch.ones(3, 8)
    for weight in (w, w.clone().requires_grad_()):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(lambda t: degree_norm(t, weight, channels=8, lmax=2), (x,))
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(lambda t: residual_block_norm(t, t, scale=weight, channels=8, lmax=2)[0], (x,))


def test_launches_take_no_host_tensors(monkeypatch):
    from ictc_o3.backends.cuda import _native
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(_native, "_raw_stream", lambda index: 0)
    lib = _native.library()
    called = []
    monkeypatch.setattr(_native, "_lib", type("Recorder", (), {"__getattr__": lambda self, name: lambda *a: called.append(
        (name, a)) or 0})())
    assert lib is not None
    _native.launch(torch.device("cuda", 0), "ictc_block_forward", None, 3)
    assert called == [("ictc_block_forward", (None, 3, 0))]
    with pytest.raises(TypeError, match="CUDA tensors"):
        _native.launch(torch.device("cuda", 0), "ictc_block_forward", torch.tensor(3))
    assert len(called) == 1


def test_status_and_wait_limit_are_checked():
    from ictc_o3.backends.cuda import _native
    lib = _native.library()
    assert lib.ictc_block_wait_limit(2_000_000_001) == -1 and "two seconds" in lib.ictc_last_error().decode()
    assert lib.ictc_block_wait_limit(2_000_000_000) == 0
    assert lib.ictc_block_status_word(None) == -1 and lib.ictc_block_status(0, None, None) == -1
