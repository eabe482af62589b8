"""The optimizer's host helpers (CPU only)."""
import pytest
import torch


def test_lists_of_the_same_items():
    from ictc_o3.backends.cuda._native import host_tensors
    holds = host_tensors().holds
    a, b, c = (torch.zeros(2) for _ in range(3))
    whole = [a, b, c]
    assert holds(whole, 0, [a, b]) and holds(whole, 1, [b, c]) and holds(whole, 3, []) and holds(whole, 0, whole)
    for start, part in ((0, [b]), (2, [c, a]), (3, [c]), (-1, [a]), (4, []), (0, [a, b, c, a]), (1, [torch.zeros(2)])):
        assert holds(whole, start, part) is False
    for bad in (lambda: holds(whole, 0, (a,)), lambda: holds(whole, "0", []), lambda: holds(whole, 0),
                lambda: holds((a,), 0, [])):
        with pytest.raises(TypeError):
            bad()
