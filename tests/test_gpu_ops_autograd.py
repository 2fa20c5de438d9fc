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


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("heads,attention", [(3, "softmax"), (8, "softmax"), (6, "differential")])
def test_tail_hook_of_the_fused_head_loss(gpu_device, heads, attention, packed):
    """The hook inside the backward pass (data-parallel training starts the all-reduce of ``flat_grad[split:]`` there) sees
    the final gradients of the upper layers, the final norm and the vocabulary head, whose gradient the fused loss makes."""
    from bidiff.parallel import tail_split_offset
    bb, model, ids, attn, _ = small_model(gpu_device, heads, attention, dropout=0.1)
    model.fused_head_loss, model.skip_padded_rows = True, packed
    opt = FlatAdamW(model.parameters(), lr=1e-3)
    off = tail_split_offset(opt, bb, 2)
    seen = []
    AG.set_tail_ready_hook(lambda: seen.append((opt.flat_grad[off:].clone(), opt.flat_grad[:off].clone())), 2, model=bb)
    try:
        for _ in range(3):
            opt.zero_grad()
            seen.clear()
            model(ids, attn)["loss"].backward()
            torch.cuda.synchronize()
            assert len(seen) == 1
            assert float(bb.output_proj.weight.grad.abs().max()) > 0
            assert torch.equal(seen[0][0], opt.flat_grad[off:]), "tail complete when the hook fires"
            assert not torch.equal(seen[0][1], opt.flat_grad[:off]), "head still in progress"
        bb.dropout = 0.0               # no dropout decisions: the passes differ in nothing but the hook
        grads = []
        for hook in (lambda: None, None):
            AG.set_tail_ready_hook(hook, 2, model=bb)
            opt.zero_grad()
            torch.manual_seed(5)       # same timesteps and corruption
            (model(ids, attn)["loss"] / 2).backward()
            (model(ids, attn)["loss"] / 2).backward()      # a second micro-batch adds to the first's gradients
            grads.append(opt.flat_grad.clone())
        assert float((grads[0] - grads[1]).norm() / grads[1].norm()) < 1e-4      # (atomic sums: another order each time)
    finally:
        AG.set_tail_ready_hook(None, model=bb)


def test_tail_hook_waits_for_a_head_outside_the_backbone(gpu_device):
    """Rows of ``backbone_forward_train(hidden_states="bf16")`` under a loss of the caller's own: the head's gradient does not
    pass through the backbone's backward pass, which therefore cannot report the tail as complete."""
    from bidiff.parallel import tail_split_offset
    bb, model, ids, attn, t = small_model(gpu_device)
    opt = FlatAdamW(model.parameters(), lr=1e-3)
    off = tail_split_offset(opt, bb, 2)
    seen = []
    AG.set_tail_ready_hook(lambda: seen.append(opt.flat_grad[off:].clone()), 2, model=bb)
    try:
        for frozen in (False, True):
            opt.zero_grad()
            seen.clear()
            hidden = AG.backbone_forward_train(bb, ids, t, attn, hidden_states="bf16")
            w = bb.output_proj.weight
            ops.linear_cross_entropy(hidden, w.detach() if frozen else w, ids, None, attn).backward()
            torch.cuda.synchronize()
            assert all(torch.equal(s, opt.flat_grad[off:]) for s in seen)
    finally:
        AG.set_tail_ready_hook(None, model=bb)


def test_rotary_in_place_is_seen_by_autograd(gpu_device):
    """A tensor that a living graph saved and ``rotary_`` then turned: the backward pass raises, as after any in-place operation."""
    dev = gpu_device
    table = ops.rotary_table(32, 8, device=dev)
    x, y = (torch.randn(2, 8, 3, 32, device=dev) for _ in range(2))
    w = torch.randn(32, device=dev, requires_grad=True)
    for a, b in ((x, None), (y, x)):
        loss = ((a * w).sum() if b is None else (b * w).sum())
        ops.rotary_(a, b, table)
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    loss = (x * w).sum()
    with torch.no_grad():
        ops.rotary_(x.detach()[:, 2:5], None, table)           # through a detached view
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():
        z = torch.randn(2, 8, 3, 32, device=dev, dtype=BF)      # no version to count
        before = z.clone()
        ops.rotary_(z, None, table)
        ops.rotary_(z, None, table, inverse=True)
        # two roundings of values that turn twice: half a step of a pair's length each
        assert float((z.float() - before.float()).abs().max()) <= 4 * 2.0 ** -8 * float(before.abs().max())


@pytest.mark.parametrize("packed", [False, True])
def test_fused_head_loss_under_a_mask_in_floating_point(gpu_device, packed):
    """The diffusion step takes its 0 / 1 mask in any type, with the fused loss as with logits."""
    _, model, ids, attn, t = small_model(gpu_device)
    model.fused_head_loss, model.skip_padded_rows = True, packed
    losses = []
    for mask in (attn, attn.float(), attn.bool()):
        torch.manual_seed(4)
        losses.append(model(ids, mask, t)["loss"])
        with torch.no_grad():
            torch.manual_seed(4)
            losses.append(model(ids, mask, t)["loss"])
    assert all(torch.equal(a, b) for a, b in zip(losses, losses[2:]))


FORMS = {"kept maps": (2, 70, 300, 4, 2, 32, False), "keys walked twice": (2, 70, 150, 4, 2, 64, False), "two key tiles": (3, 40, 100, 2, 2, 64, False),
         "wide heads": (1, 33, 90, 2, 1, 128, False), "packed": (3, 60, 60, 4, 2, 32, True)}


@pytest.mark.parametrize("form", FORMS)
def test_frozen_operands_of_differential_attention(gpu_device, monkeypatch, form):
    """Any subset of q, k, v and lam may need a gradient. Theirs have the bits of the full backward; for the others nothing is
    computed into memory: no dq where q is frozen, no launch for the keys' side where k and v are."""
    dev = gpu_device
    B, Lq, Lk, H, Hkv, D, packed = FORMS[form]
    g = torch.Generator(device=dev).manual_seed(21)
    lead_q, lead_k = ((B * Lq,), (B * Lk,)) if packed else ((B, Lq), (B, Lk))
    base = {n: torch.randn(*s, generator=g, device=dev).to(BF) for n, s in
            (("q", (*lead_q, 2 * H, D)), ("k", (*lead_k, 2 * Hkv, D)), ("v", (*lead_k, Hkv, 2 * D)))}
    base["lam"] = torch.rand(H, generator=g, device=dev)
    dout = torch.randn(*lead_q, H, 2 * D, generator=g, device=dev).to(BF)
    # (packed: rows before the first and behind the last sequence, too)
    kw = dict(cu_seqlens=torch.tensor([2, 60, 61, B * Lq - 3], dtype=torch.int32, device=dev), max_seqlen=115) if packed else {}
    written = []
    call = ops._attention_call

    def spy(entry, *args, **kwargs):
        if kwargs.get("grads") or entry == "bd_diff_attention_bwd":
            grads = kwargs.get("grads") or next(a for a in args if isinstance(a, tuple) and len(a) == 6)
            written.append(tuple(t is not None for t in grads[1:4]))
        return call(entry, *args, **kwargs)
    monkeypatch.setattr(ops, "_attention_call", spy)

    def run(names):
        x = {n: t.clone().requires_grad_(n in names) for n, t in base.items()}
        out = ops.differential_attention(*x.values(), **kw)
        return dict(zip(names, torch.autograd.grad(out, [x[n] for n in names], dout)))

    def same(a, b):                # (one packed sequence is longer than announced: NaN there)
        return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    full = run(("q", "k", "v", "lam"))
    assert written.pop() == (True, True, True)
    for names in (("q",), ("k",), ("v",), ("lam",), ("q", "lam"), ("k", "v"), ("q", "v"), ("k", "lam")):
        got = run(names)
        assert all(same(got[n], full[n]) for n in names), names
        keys = "k" in names or "v" in names
        assert written.pop() == ("q" in names, keys, keys), names


@pytest.mark.parametrize("M,d,V", [(33000, 64, 39), (20000, 256, 803), (700, 128, 300), (3000, 64, 65000)])
@pytest.mark.parametrize("wdt", [BF, torch.float32])
def test_either_gradient_of_the_head_loss_alone(gpu_device, M, d, V, wdt):
    """The rows' gradient alone and the head's alone, each in the scratch it asks for (with and without slabs, in one piece of
    the vocabulary and in two), have the bits that they have together."""
    dev = gpu_device
    g = torch.Generator(device=dev).manual_seed(31)
    h, w = torch.randn(M, d, generator=g, device=dev).to(BF), (torch.randn(V, d, generator=g, device=dev) / d ** 0.5).to(wdt)
    t, ind = torch.randint(0, V, (M,), generator=g, device=dev), torch.rand(M, generator=g, device=dev) < 0.6

    def run(*need):
        leaves = [x.clone().requires_grad_(n) for x, n in zip((h, w), need)]
        return torch.autograd.grad(ops.linear_cross_entropy(*leaves, t, ind), [x for x in leaves if x.requires_grad])
    dh, dw = run(True, True)
    assert torch.equal(run(True, False)[0], dh) and torch.equal(run(False, True)[0], dw)


@pytest.mark.parametrize("M,d,live", [(40000, 576, 0.5), (40000, 64, 0.02), (9000, 1024, 0.9)])
def test_rows_gathered_by_the_head_loss(gpu_device, M, d, live):
    """The weighted rows reach the compact matrix whole and in order, whatever the timing of the waves that copy them: the loss
    has the bits of the call that gets these rows alone, time after time."""
    dev = gpu_device
    g = torch.Generator(device=dev).manual_seed(41)
    h, w = torch.randn(M, d, generator=g, device=dev).to(BF), (torch.randn(300, d, generator=g, device=dev) / d ** 0.5).to(BF)
    t, ind = torch.randint(0, 300, (M,), generator=g, device=dev), torch.rand(M, generator=g, device=dev) < live
    alone = ops.linear_cross_entropy(h[ind], w, t[ind])
    assert all(torch.equal(ops.linear_cross_entropy(h, w, t, ind), alone) for _ in range(5))
