"""What the stand-alone operators owe to autograd and to their caller's tensors, as far as it shows without a GPU: launches
are replaced where a call would reach one."""
import pytest
import torch

from bidiff import ops

BF = torch.bfloat16
TABLE = torch.zeros(8, 4, 2)


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def test_rotary_in_place_counts_as_a_change(monkeypatch):
    monkeypatch.setattr(ops._lib, "require_device", lambda *a: None)
    monkeypatch.setattr(ops, "_rotary_launch", lambda pairs, *a: None)
    q, k = z(1, 3, 2, 8), z(1, 3, 1, 8)
    before = q._version, k._version
    ops.rotary_(q, k, TABLE)
    assert q._version > before[0] and k._version > before[1]
    w = torch.ones(8, requires_grad=True)
    x = torch.ones(1, 3, 2, 8)
    loss = (x * w).sum()
    ops.rotary_(x[:, 1:], None, TABLE)                # a view: the whole tensor counts
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():                      # tensors without a version
        ops.rotary_(z(1, 3, 2, 8), None, TABLE)
