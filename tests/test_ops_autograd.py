"""What the stand-alone operators owe to autograd and to their caller's tensors, as far as it shows without a GPU: launches
are replaced where a call would reach one."""
import pytest
import torch
from torch.autograd import forward_ad

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


@pytest.mark.parametrize("at", range(4))
@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_is_refused(at, grad):
    """No operator here has a forward-mode derivative: a dual operand is refused, its tangent is not dropped."""
    with forward_ad.dual_level():
        def dual(i, t):
            return forward_ad.make_dual(t, torch.ones_like(t)) if i == at else t.requires_grad_(grad)
        calls = [lambda: ops.differential_attention(dual(0, z(2, 3, 4, 32)), dual(1, z(2, 5, 4, 32)), dual(2, z(2, 5, 2, 64)), dual(3, z(2)))]
        if at < 2:
            calls.append(lambda: ops.rotary(dual(0, z(1, 3, 2, 8)), dual(1, z(1, 3, 2, 8)), TABLE))
            calls.append(lambda: ops.linear_cross_entropy(dual(0, z(3, 64)), dual(1, z(7, 64)), torch.zeros(3, dtype=torch.long)))
            if not grad:
                calls.append(lambda: ops.rotary_(dual(0, z(1, 3, 2, 8)), dual(1, z(1, 3, 2, 8)), TABLE))
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError):             # an open level alone refuses nothing (here: a CPU operand)
            ops.linear_cross_entropy(z(3, 64), z(7, 64), torch.zeros(3, dtype=torch.long))


def test_forward_mode_of_the_rotary_table_is_refused():
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.rotary(z(1, 3, 2, 8), None, forward_ad.make_dual(TABLE.clone(), TABLE + 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, BF, torch.float64, torch.complex64])
def test_weights_of_rows_that_are_not_whole_numbers_are_refused(dtype):
    """``attention_mask`` holds whole numbers: 0.5 would count as 0 and 1.9 as 1."""
    with pytest.raises(TypeError, match="attention_mask"):
        ops.linear_cross_entropy(z(3, 64), z(7, 64), torch.zeros(3, dtype=torch.long), None, torch.ones(3, dtype=dtype))
