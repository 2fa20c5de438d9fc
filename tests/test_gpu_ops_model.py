"""The operators where the package's own paths call them: a denoiser with differential attention and rotary positions
(training on padded and packed rows, inference, sampling), the fused head loss of the diffusion training step, and a run
of all three together against one 64-bit statement."""
import math

import numpy as np
import pytest
import torch

from bidiff import ops
from bidiff.model.backbone import DiffusionBackbone, MultiHeadAttention, TransformerBlock
from bidiff.model.diffusion import DiscreteMaskingDiffusion
from bidiff.training.optimizer import FlatAdamW
from oracle import backbone_ref as BR
from oracle import ops_ref as R
from tests.golden import replay_inputs as RI

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rel(a, b):
    return float((a - b).norm() / b.norm().clamp(min=1e-12))


def build(dev, heads, attention, rotary_base, dropout=0.0, d=128, V=39, L=48):
    cfg = dict(vocab_size=V, hidden_size=d, num_layers=2, num_heads=heads, ffn_hidden_size=256, max_position_embeddings=64,
               num_diffusion_steps=20, dropout=dropout, pad_token_id=0)
    torch.manual_seed(3)
    bb = DiffusionBackbone(**cfg, attention=attention, rotary_base=rotary_base)
    RI.perturb_state_dict({k: v for k, v in bb.state_dict().items() if "lambda" not in k}, 11)
    model = DiscreteMaskingDiffusion(bb, num_steps=20, mask_token_id=1, pad_token_id=0, bos_token_id=2, eos_token_id=3)
    sd = {k: v.clone() for k, v in bb.state_dict().items()}
    rs = np.random.RandomState(5)
    B = 6
    lens = rs.randint(3, L + 1, size=B)
    lens[0], lens[1] = L, 0
    ids = rs.randint(5, V, size=(B, L)).astype(np.int64)
    attn = (np.arange(L)[None] < lens[:, None]).astype(np.int64)
    attn[2, 1] = 0
    ids[attn == 0] = 0
    t = rs.randint(1, 21, size=B).astype(np.int64)
    return cfg, model.to(dev), sd, *(torch.from_numpy(x) for x in (ids, attn, t))


VARIANTS = [(4, "differential", None), (2, "softmax", 10000.0), (4, "differential", 500.0), (8, "differential", 10000.0)]   # heads of 32, 64, 32, 16 -> 32


@pytest.mark.parametrize("heads,attention,rotary_base", VARIANTS)
@pytest.mark.parametrize("packed", [False, True])
def test_training_gradients_against_fp32_autograd(gpu_device, monkeypatch, heads, attention, rotary_base, packed):
    """Loss and every parameter gradient of the training path against fp32 autograd of the statement, within what bf16
    products leave (the same bounds as the plain model's tests)."""
    dev = gpu_device
    cfg, model, sd, ids, attn, t = build(dev, heads, attention, rotary_base)
    model.train()
    model.skip_padded_rows = packed
    u = torch.rand(ids.shape, generator=torch.Generator().manual_seed(9))
    noisy, ind = model.forward_process(ids.to(dev), t.to(dev), attn.to(dev), uniforms=u.to(dev))
    from bidiff.training import autograd as AG
    if packed:
        loss, _ = AG.packed_training_loss(model, noisy, t.to(dev), attn.to(dev), ids.to(dev), ind)
    else:
        loss = model._compute_loss(model.backbone(noisy, t.to(dev), attn.to(dev)), ids.to(dev), ind, attn.to(dev))
    loss.backward()
    monkeypatch.setattr(BR, "attention", R.block_attention(rotary_base))
    ref = {k: v.clone().requires_grad_(True) for k, v in sd.items()}
    want = BR.masked_ce(BR.logits(ref, cfg, noisy.cpu(), t, attn), ids, ind.cpu(), attn)
    want.backward()
    assert abs(loss.item() - want.item()) < 2e-2 * abs(want.item())
    norms = sorted(float(p.grad.norm()) for p in ref.values() if p.grad is not None)
    for k, p in model.backbone.named_parameters():
        g = ref[k].grad
        if float(g.norm()) < 1e-2 * norms[len(norms) // 2]:      # (the k bias: its exact gradient is zero)
            assert float(p.grad.norm()) < 1e-1 * norms[len(norms) // 2], k
            continue
        cos = float((p.grad.cpu() * g).sum() / (p.grad.cpu().norm() * g.norm()))
        assert rel(p.grad.cpu(), g) < 1e-1 and cos > 0.995, (k, rel(p.grad.cpu(), g), cos)
    if attention == "differential":
        assert any("lambda_weight" in k for k, _ in model.backbone.named_parameters())


@pytest.mark.parametrize("heads,attention,rotary_base", VARIANTS)
def test_inference_forward_and_modules(gpu_device, monkeypatch, heads, attention, rotary_base):
    dev = gpu_device
    cfg, model, sd, ids, attn, t = build(dev, heads, attention, rotary_base)
    bb = model.backbone.eval()
    monkeypatch.setattr(BR, "attention", R.block_attention(rotary_base))
    with torch.no_grad():
        got = bb(ids.to(dev), t.to(dev), attn.to(dev)).cpu()
        want = BR.logits(sd, cfg, ids, t, attn)
        assert float((got - want).abs().max()) < 2e-2 * float(want.abs().max())
        for layer in (0, 1, -1):
            h = bb.get_hidden_states(ids.to(dev), t.to(dev), attn.to(dev), layer_idx=layer).cpu()
            hw = BR.hidden_states(sd, cfg, ids, t, attn, layer_idx=layer)
            keep = attn.bool() if layer >= 0 else torch.ones_like(attn, dtype=torch.bool)
            assert float((h - hw)[keep].abs().max()) < 3e-2 * float(hw.abs().max())
        pooled = bb.get_pooled_output(ids.to(dev), t.to(dev), attn.to(dev))
        assert bool(torch.isfinite(pooled).all())
    train = bb(ids.to(dev), t.to(dev), attn.to(dev))             # autograd on: the training path, the same kernels
    assert float((train.detach().cpu() - got).abs().max()) < 1e-2 * float(want.abs().max())
    assert not bb.plain_attention and bb.rows_forward_mode(6, 48) is None and bb.wave_table_for_mask(attn.to(dev)) is None
    bb.compute_dtype = "fp32"
    with pytest.raises(NotImplementedError), torch.no_grad():
        bb(ids.to(dev), t.to(dev), attn.to(dev))


def test_modules_on_their_own(gpu_device):
    """The block-level modules with both options against the statement; head sizes the attention kernels have."""
    dev = gpu_device
    torch.manual_seed(1)
    blk = TransformerBlock(256, 4, 512, 0.0, differential=True, rotary_base=10000.0, depth=2).to(dev).eval()
    assert math.isclose(float(blk.attn.lambda_weight[0]), 0.8 - 0.6 * math.exp(-0.6), rel_tol=1e-6)
    x = torch.randn(3, 37, 256, device=dev)
    m = torch.ones(3, 37, device=dev)
    m[1, 20:] = 0
    m[2] = 0
    with torch.no_grad():
        got = blk.attn(x, m).cpu()
        out = blk(x, m)
    sd = {f"attn.{k}": v.cpu() for k, v in blk.attn.state_dict().items()}
    want = R.block_attention(10000.0)(x.cpu(), sd, "attn", 4, m.cpu())
    assert float((got - want).abs().max()) < 2e-2 * float(want.abs().max()) and bool(torch.isfinite(out).all())


def test_options_are_checked_and_absent_by_default():
    assert not any("lambda" in k for k in DiffusionBackbone(39, 128, 1, 2, 256, 64, 20).state_dict())
    assert set(DiffusionBackbone(39, 128, 1, 2, 256, 64, 20).config_dict()) == {
        "vocab_size", "hidden_size", "num_layers", "num_heads", "ffn_hidden_size", "max_position_embeddings", "num_diffusion_steps", "dropout",
        "pad_token_id"}
    bb = DiffusionBackbone(39, 128, 1, 2, 256, 64, 20, attention="differential", rotary_base=100.0)
    assert bb.config_dict()["attention"] == "differential" and bb.config_dict()["rotary_base"] == 100.0
    for bad in (dict(attention="linear"), dict(attention="differential", num_heads=1), dict(rotary_base=-1.0)):
        with pytest.raises(ValueError):
            DiffusionBackbone(**{**dict(vocab_size=39, hidden_size=128, num_layers=1, num_heads=2, ffn_hidden_size=256), **bad})
    with pytest.raises(ValueError):
        MultiHeadAttention(126, 42, 0.0, rotary_base=10.0)


def test_save_and_load_of_a_differential_model(gpu_device, tmp_path):
    dev = gpu_device
    _, model, _, ids, attn, t = build(dev, 4, "differential", 10000.0)
    path = str(tmp_path / "bb.pt")
    model.backbone.save_pretrained(path)
    again = DiffusionBackbone.load_pretrained(path).to(dev).eval()
    with torch.no_grad():
        assert torch.equal(again(ids.to(dev), t.to(dev), attn.to(dev)), model.backbone.eval()(ids.to(dev), t.to(dev), attn.to(dev)))


def test_sampling_with_a_differential_model(gpu_device):
    from bidiff.sampling.sampler import ConstrainedSampler
    from bidiff.utils import synthetic
    tok = synthetic.smiles_tokenizer()
    torch.manual_seed(0)
    bb = DiffusionBackbone(tok.vocab_size, 128, 2, 4, 256, 64, 6, 0.0, tok.pad_token_id, attention="differential", rotary_base=10000.0)
    model = DiscreteMaskingDiffusion(bb, num_steps=6, mask_token_id=tok.mask_token_id, pad_token_id=tok.pad_token_id,
                                     bos_token_id=tok.bos_token_id, eos_token_id=tok.eos_token_id).to(gpu_device).eval()
    smp = ConstrainedSampler(model, tok, num_steps=6, temperature=1.0, use_constraints=True, device="cuda:0")
    smp._core.seed = 7
    out, strings = smp.sample(8, 32, show_progress=False)
    again, _ = smp.sample(8, 32, show_progress=False)
    assert (out != tok.mask_token_id).all() and len(strings) == 8 and torch.equal(out, again)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("V", [39, 803])
def test_fused_head_loss_of_the_training_step(gpu_device, packed, V):
    """DiscreteMaskingDiffusion.fused_head_loss: the loss of the logits form and its gradients, the logits on request."""
    dev = gpu_device
    _, model, _, ids, attn, t = build(dev, 2, "softmax", None, V=V)
    model.train()
    model.skip_padded_rows = packed
    u = torch.rand(ids.shape, generator=torch.Generator().manual_seed(9)).to(dev)
    process = model.forward_process
    model.forward_process = lambda i, tt, am=None: process(i, tt, am, uniforms=u)
    res = {}
    for fused in (False, True):
        model.fused_head_loss = fused
        for p in model.parameters():
            p.grad = None
        out = model(ids.to(dev), attn.to(dev), t.to(dev))
        (out["loss"] / 3).backward()
        res[fused] = (out["loss"].item(), out["logits"].detach().clone(), {k: p.grad.clone() for k, p in model.named_parameters()})
    (l0, z0, g0), (l1, z1, g1) = res[False], res[True]
    assert abs(l0 - l1) < 1e-5 * abs(l0)
    assert torch.equal(z0, z1)
    for k in g0:
        # both round dlogits to bf16 once (half a step each, 2^-8); the bound leaves what the later bf16 products make of it
        assert rel(g1[k], g0[k]) < 2e-2 or float(g0[k].norm()) < 1e-4 * max(float(x.norm()) for x in g0.values()), (k, rel(g1[k], g0[k]))
    with torch.no_grad():
        model.eval()
        model.fused_head_loss = False
        e0 = model(ids.to(dev), attn.to(dev), t.to(dev))
        model.fused_head_loss = True
        e1 = model(ids.to(dev), attn.to(dev), t.to(dev))
        assert abs(e0["loss"].item() - e1["loss"].item()) < 1e-4 * abs(e0["loss"].item())
        assert float((e0["logits"] - e1["logits"]).abs().max()) < 2e-2 * float(e0["logits"].abs().max())


def test_optimizer_steps_with_flat_gradients(gpu_device):
    """FlatAdamW (gradients accumulate straight into one buffer) over a differential model with the fused loss: every
    parameter, the map weights among them, gets the gradient autograd's own buffers would hold, and moves."""
    dev = gpu_device
    _, model, _, ids, attn, t = build(dev, 4, "differential", 10000.0)
    model.fused_head_loss = True
    u = torch.rand(ids.shape, generator=torch.Generator().manual_seed(9)).to(dev)
    process = model.forward_process
    model.forward_process = lambda i, tt, am=None: process(i, tt, am, uniforms=u)
    model.train()
    model(ids.to(dev), attn.to(dev), t.to(dev))["loss"].backward()
    own = {k: p.grad.clone() for k, p in model.named_parameters()}
    for p in model.parameters():
        p.grad = None
    opt = FlatAdamW(model.parameters(), lr=1e-3)
    before = {k: p.detach().clone() for k, p in model.named_parameters()}
    opt.zero_grad()
    model(ids.to(dev), attn.to(dev), t.to(dev))["loss"].backward()
    for k, p in model.named_parameters():
        assert rel(p.grad, own[k]) < 1e-4 or float(own[k].abs().max()) < 1e-12, k
    opt.step()
    for k, p in model.named_parameters():
        if float(own[k].abs().max()) > 0:
            assert not torch.equal(p.detach(), before[k]), k


@pytest.mark.parametrize("B,L,H,Hkv,D,V", [(3, 21, 2, 1, 32, 39), (2, 130, 2, 2, 64, 803)])
def test_the_operators_run_together(gpu_device, B, L, H, Hkv, D, V):
    """Projection -> rotary -> differential attention -> head loss, forward and backward, against the 64-bit statements
    chained on the operators' own (bf16) intermediate values, each link within its own bounds."""
    dev = gpu_device
    g = torch.Generator(device=dev).manual_seed(B + L)
    x = torch.randn(B, L, 2 * H * D + 4 * Hkv * D, generator=g, device=dev).to(BF).requires_grad_(True)
    lam = torch.rand(B, L, H, generator=g, device=dev).to(BF).requires_grad_(True)
    d = H * 2 * D
    w = (torch.randn(V, d, generator=g, device=dev) / d ** 0.5).requires_grad_(True)
    tg = torch.randint(0, V, (B, L), generator=g, device=dev)
    ind = torch.rand(B, L, generator=g, device=dev) < 0.5
    n = torch.randint(1, L + 1, (B,), generator=g, device=dev)
    m = torch.arange(L, device=dev)[None] < n[:, None]
    table = ops.rotary_table(D, L, device=dev)
    q, k, v = x.split([2 * H * D, 2 * Hkv * D, 2 * Hkv * D], -1)
    q, k, v = q.unflatten(-1, (2 * H, D)), k.unflatten(-1, (2 * Hkv, D)), v.unflatten(-1, (Hkv, 2 * D))
    q2, k2 = ops.rotary(q, k, table)
    o = ops.differential_attention(q2, k2, v, lam, key_mask=m)
    loss = ops.linear_cross_entropy(o.flatten(-2), w, tg, ind, m.long())
    dq2, dk2, do = torch.autograd.grad(loss, (q2, k2, o), retain_graph=True)
    dx, dlam, dw = torch.autograd.grad(loss, (x, lam, w))
    at = torch.arange(L, device=dev).expand(B, L)
    for a, b in ((q, q2), (k, k2)):
        want = R.rotary(a.detach(), table, at, False)
        assert float(((b.double() - want).abs() - 1.02 * R.U * want.abs() - 8 * R.F * a.double().abs().amax()).max()) <= 0
    ce = R.linear_cross_entropy(o.detach().reshape(B * L, d), w.detach().to(BF), tg.reshape(-1), (ind & m).reshape(-1).float(), tol=True)
    assert float((loss.double() - ce["loss"]).abs() - ce["loss_tol"]) <= 0
    assert float(((dw.double() - ce["dw"]).abs() - ce["dw_tol"]).max()) <= 0
    assert float(((do.double().reshape(B * L, d) - ce["dh"]).abs() - ce["dh_tol"]).max()) <= 0
    spans = [(slice(b * L, (b + 1) * L),) * 2 for b in range(B)]
    flat = lambda z: z.detach().reshape(B * L, *z.shape[2:])  # noqa: E731
    r = R.differential_attention(flat(q2), flat(k2), flat(v), flat(lam), spans, m.reshape(-1), B * L, B * L, flat(do), tol=True)
    assert float(((flat(o).double() - r["out"]).abs() - r["out_tol"]).max()) <= 0
    for got, name in ((dq2, "dq"), (dk2, "dk")):
        assert float(((flat(got).double() - r[name]).abs() - r[name + "_tol"]).max()) <= 0
    assert float(((flat(dlam).double() - r["dlam"]).abs() - r["dlam_tol"] - 1.01 * R.U * r["dlam"].abs()).max()) <= 0
    gq, gk, gv = dx.split([2 * H * D, 2 * Hkv * D, 2 * Hkv * D], -1)
    for got, up in ((gq.unflatten(-1, (2 * H, D)), dq2), (gk.unflatten(-1, (2 * Hkv, D)), dk2)):
        want = R.rotary(up, table, at, False, inverse=True)
        assert float(((got.double() - want).abs() - 1.02 * R.U * want.abs() - 8 * R.F * up.double().abs().amax()).max()) <= 0
    assert float(((flat(gv.unflatten(-1, (Hkv, 2 * D))).double() - r["dv"]).abs() - r["dv_tol"]).max()) <= 0
