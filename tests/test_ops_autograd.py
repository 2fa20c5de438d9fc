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
