"""The stand-alone operators and the training step that uses them under autograd: gradients that others hold, gradients
that a hook inside the backward pass reads, tensors written in place, operands without a gradient."""
import pytest
import torch

from bidiff import ops
from bidiff.model.backbone import DiffusionBackbone
from bidiff.model.diffusion import DiscreteMaskingDiffusion
from bidiff.training import autograd as AG
from bidiff.training.optimizer import FlatAdamW
from tests.golden import replay_inputs as RI

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def small_model(dev, heads=3, attention="softmax", dropout=0.0):
    cfg = dict(RI.SMALL_CFG, vocab_size=39, num_layers=4, dropout=dropout, num_heads=heads)
    torch.manual_seed(7)
    bb = DiffusionBackbone(**cfg, attention=attention)
    model = DiscreteMaskingDiffusion(bb, num_steps=cfg["num_diffusion_steps"], mask_token_id=1, pad_token_id=0, bos_token_id=2,
                                     eos_token_id=3).to(dev).train()
    ids, attn, t = (torch.from_numpy(x).to(dev) for x in RI.backbone_inputs(cfg, 33, B=64, L=128))
    return bb, model, ids, attn, t


def test_gradient_of_the_heads_rows_is_left_alone(gpu_device):
    """The backward pass of the backbone reads the gradient of the rows it returned and writes none of it: whoever keeps
    that tensor (a hook, ``torch.autograd.grad`` on the rows, another consumer of the same gradient) keeps its values."""
    dev = gpu_device
    bb, model, ids, attn, t = small_model(dev)
    hidden = AG.backbone_forward_train(bb, ids, t, attn, hidden_states="bf16")
    leaf = hidden.detach().clone().requires_grad_(True)
    (want,) = torch.autograd.grad(ops.linear_cross_entropy(leaf, bb.output_proj.weight.detach(), ids, None, attn), (leaf,))
    kept = []
    hidden.register_hook(kept.append)
    loss = ops.linear_cross_entropy(hidden, bb.output_proj.weight.detach(), ids, None, attn)
    got = torch.autograd.grad(loss, (hidden, bb.final_norm.weight))[0]
    assert torch.equal(got, want) and torch.equal(kept[0], want)
