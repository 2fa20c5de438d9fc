"""Forward of the block-level modules on their own (``MultiHeadAttention``, ``FeedForward``, ``TransformerBlock``).

The reference's modules are callable (src/model/backbone.py:32-78, :95-101, :120-129); ``DiffusionBackbone`` here
never calls them (it runs the whole stack in fused launches), but a caller that applies a single block or projection
gets the same arithmetic from the same kernels: bf16 operands on the matrix cores with fp32 accumulation, fp32
LayerNorm / residual / softmax, exactly the unfused path of the backbone. Inference only: under autograd with
trainable parameters these raise (training runs through ``DiffusionBackbone`` / ``DiscreteMaskingDiffusion``), and
dropout is not applied (``eval()`` semantics)."""
import torch

from .. import _lib, ops


def _pad_rows(w: torch.Tensor, mult: int = 128) -> torch.Tensor:
    n = w.shape[0]
    n_pad = (n + mult - 1) // mult * mult
    if n_pad == n:
        return w.contiguous()
    out = torch.zeros(n_pad, w.shape[1], dtype=w.dtype, device=w.device)
    out[:n] = w
    return out


class _Bf16Copies:
    """bf16 (row-padded) copies of a module's matrices, rebuilt when a parameter changed."""

    def __init__(self):
        self.key, self.t = None, None

    def get(self, params, build):
        key = (_lib.weights_generation(),) + tuple((p.data_ptr(), p._version, p.device) for p in params)
        if key != self.key:
            with torch.no_grad():
                self.t = build()
            self.key = key
        return self.t


def _check(x: torch.Tensor, what: str, params):
    _lib.require_device(x, what)
    if torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in params)):
        raise NotImplementedError(f"{what}: the block-level forward is inference-only (call it under torch.no_grad(); "
                                  f"training runs through DiffusionBackbone)")
    if x.dim() != 3:
        raise ValueError(f"{what}: expected [batch, seq_len, hidden], got {tuple(x.shape)}")


def _gemm(a_bf16, w_bf16, bias, out, M, n_real, K, epilogue):
    n_pad = w_bf16.shape[0]
    if K % 64 != 0:
        raise NotImplementedError(f"bidiff GEMM needs an inner size that is a multiple of 64, got {K}")
    _lib.check(_lib.lib().bd_gemm_bf16(_lib.ptr(a_bf16), _lib.ptr(w_bf16), _lib.ptr(bias), _lib.ptr(out), M, n_pad, n_real, K,
                                       out.shape[-1], epilogue, _lib.stream_handle()), "bd_gemm_bf16")


def _cast(x_f32):
    y = torch.empty(x_f32.shape, dtype=torch.bfloat16, device=x_f32.device)
    _lib.check(_lib.lib().bd_cast_f32_to_bf16(_lib.ptr(x_f32), _lib.ptr(y), x_f32.numel(), _lib.stream_handle()), "bd_cast_f32_to_bf16")
    return y


def _layernorm(x_f32, norm, M, d):
    y = torch.empty(M, d, dtype=torch.bfloat16, device=x_f32.device)
    _lib.check(_lib.lib().bd_layernorm(_lib.ptr(x_f32), _lib.ptr(norm.weight), _lib.ptr(norm.bias), _lib.ptr(y), None, None, M, d,
                                       float(norm.eps), _lib.stream_handle()), "bd_layernorm")
    return y


def _keymask(attention_mask, B, L, device):
    if attention_mask is None:
        return None
    if tuple(attention_mask.shape) != (B, L):
        raise ValueError(f"attention_mask must be [batch, seq_len] = {(B, L)}, got {tuple(attention_mask.shape)}")
    return (attention_mask.to(device) != 0).to(torch.uint8).contiguous()


def _attn_weights(mha):
    def build():
        wqkv = torch.cat([mha.q_proj.weight, mha.k_proj.weight, mha.v_proj.weight], 0).detach()
        bqkv = torch.cat([mha.q_proj.bias, mha.k_proj.bias, mha.v_proj.bias], 0).detach().float().contiguous()
        return (_pad_rows(wqkv.to(torch.bfloat16)), bqkv, _pad_rows(mha.out_proj.weight.detach().to(torch.bfloat16)),
                mha.out_proj.bias.detach().float().contiguous())
    if not hasattr(mha, "_bf16"):
        object.__setattr__(mha, "_bf16", _Bf16Copies())
    return mha._bf16.get(list(mha.parameters()), build)


def _ffn_weights(ffn):
    def build():
        return (_pad_rows(ffn.fc1.weight.detach().to(torch.bfloat16)), ffn.fc1.bias.detach().float().contiguous(),
                _pad_rows(ffn.fc2.weight.detach().to(torch.bfloat16)), ffn.fc2.bias.detach().float().contiguous())
    if not hasattr(ffn, "_bf16"):
        object.__setattr__(ffn, "_bf16", _Bf16Copies())
    return ffn._bf16.get(list(ffn.parameters()), build)


def _attention_core(mha, a_bf16, keymask, B, L, out_f32, epilogue):
    """out_f32 (epilogue 3: = / epilogue 2: +=) out_proj(attention(q, k, v of a_bf16))."""
    d, H, dh = mha.hidden_size, mha.num_heads, mha.head_dim
    if dh not in (32, 64, 128):
        raise NotImplementedError(f"the stand-alone attention forward supports head sizes 32, 64 and 128, got {dh} "
                                  f"(DiffusionBackbone runs other head sizes zero-padded)")
    M = B * L
    wqkv, bqkv, wo, bo = _attn_weights(mha)
    if 3 * d % 8 != 0:
        raise NotImplementedError("hidden size must be a multiple of 8")
    qkv = torch.empty(M, 3 * d, dtype=torch.bfloat16, device=a_bf16.device)
    _gemm(a_bf16, wqkv, bqkv, qkv, M, 3 * d, d, 0)
    att = torch.empty(M, d, dtype=torch.bfloat16, device=a_bf16.device)
    if mha.rotary_base is not None:
        turn_positions(mha, qkv.view(B, L, 3 * d), None, dh, L)
    if mha.differential:
        differential_heads(qkv.view(B, L, 3 * d), mha, keymask, None, None, dh, att.view(B, L, d), False)
    else:
        _lib.check(_lib.lib().bd_attention_fwd(_lib.ptr(qkv), _lib.ptr(keymask), _lib.ptr(att), None, B, L, H, dh,
                                               _lib.stream_handle()), "bd_attention_fwd")
    _gemm(att, wo, bo, out_f32, M, d, d, epilogue)


def split_qkv(qkv, n_maps, dh, differential):
    """Views of a projection's output [..., 3 * heads * dh]: q and k [..., heads, dh] and v [..., heads, dh], or, for
    differential attention, v [..., heads / 2, 2 dh] (both heads of a pair)."""
    q, k, v = qkv.split(n_maps * dh, -1)
    n_v, w_v = (n_maps // 2, 2 * dh) if differential else (n_maps, dh)
    return q.unflatten(-1, (n_maps, dh)), k.unflatten(-1, (n_maps, dh)), v.unflatten(-1, (n_v, w_v))


def turn_positions(mha, qkv, positions, dh_padded, n_positions, inverse=False):
    """Rotary positions on the q and k parts of ``qkv`` [B, L, 3 * width] (or packed rows), in place. The head's own
    values turn (a padded head's zeros behind them stay). The tables are kept on the module by the base that they were made
    with, shorter ones too: a captured graph may still read one that a longer call replaced. Each holds twice the positions
    of the one before or more, so that a call that grows token by token makes few of them."""
    tables = mha.__dict__.setdefault("_rotary_by_base", {}).setdefault(mha.rotary_base, [])
    table = next((x for x in tables if x.device == qkv.device and x.shape[0] >= n_positions), None)
    if table is None:
        longest = max((x.shape[0] for x in tables if x.device == qkv.device), default=0)
        table = ops.rotary_table(mha.head_dim, max(n_positions, 2 * longest), base=mha.rotary_base, device=qkv.device)
        tables.append(table)
    q, k, _ = split_qkv(qkv, mha.num_heads, dh_padded, False)
    ops._rotary_launch([(q, q), (k, k)], table, positions, False, inverse)


def differential_heads(qkv, mha, keymask, cu, longest, dh_padded, out, training):
    """Differential attention of ``qkv`` [B, L, 3 * width] (or packed rows) into ``out`` [..., width]; returns what the
    backward reads. The query projection carries sqrt(padded / own head size), as for the softmax kernels."""
    q, k, v = split_qkv(qkv, mha.num_heads, dh_padded, True)
    lam = mha.lambda_weight.detach()
    o = out.unflatten(-1, (mha.num_heads // 2, 2 * dh_padded))
    return ops._attention_forward(q, k, v, lam, [0, 0, 1], keymask, cu, longest, dh_padded ** -0.5, training, o)[1]


def differential_heads_backward(qkv, mha, keymask, cu, longest, dh_padded, saved, dout, dqkv):
    """Writes ``dqkv``; returns the gradient of ``mha.lambda_weight``."""
    q, k, v = split_qkv(qkv, mha.num_heads, dh_padded, True)
    dq, dk, dv = split_qkv(dqkv, mha.num_heads, dh_padded, True)
    lam = mha.lambda_weight.detach()
    dl = torch.empty_like(lam)
    ops._attention_backward(q, k, v, lam, [0, 0, 1], keymask, cu, longest, dh_padded ** -0.5, saved,
                            dout.unflatten(-1, (mha.num_heads // 2, 2 * dh_padded)), dq, dk, dv, dl)
    return dl


def backbone_forward_blocks(model, ids, timesteps, keymask, want_hidden=True, want_logits=False, hidden_out=None, logits_out=None,
                            upto=None):
    """Inference forward of a backbone whose attention the fused launches do not have (differential maps, rotary
    positions): the per-layer kernels in the training forward's order, nothing kept. Returns (hidden bf16 [B, L, d] or
    None, logits fp32 or None), or the fp32 residual stream after ``upto`` blocks."""
    from ..training import autograd as ag
    ag._enter()
    B, L = ids.shape
    M, d, F, V, H = B * L, model.hidden_size, model.ffn_hidden_size, model.vocab_size, model.num_heads
    if d % 128 or F % 128:
        raise ValueError("bidiff per-layer forward needs hidden and ffn sizes that are multiples of 128")
    dev, bf, eps = ids.device, torch.bfloat16, float(model.final_norm.eps)
    tw = ag._train_weights(model)
    aw, st = tw.aw, ag._s()
    x = torch.empty(M, d, device=dev)
    _lib.check(_lib.lib().bd_embed(_lib.ptr(ids), _lib.ptr(timesteps), _lib.ptr(model.token_embedding.weight),
                                   _lib.ptr(model.position_embedding.weight), _lib.ptr(model.timestep_embedding.weight), _lib.ptr(x),
                                   B, L, d, V, model.max_position_embeddings, model.num_diffusion_steps + 1, st), "bd_embed")
    h = torch.empty(M, d, dtype=bf, device=dev)
    qkv = torch.empty(M, 3 * aw, dtype=bf, device=dev)
    att = torch.empty(M, aw, dtype=bf, device=dev)
    u = torch.empty(M, F, dtype=bf, device=dev)
    n = len(model.layers) if upto is None else upto
    for blk, w in list(zip(model.layers, tw.layers))[:n]:
        ag._ln(x, blk.norm1.weight, blk.norm1.bias, h, None, M, d, eps)
        ag._gemm(h, w["wqkv"], w["bqkv"], qkv, M, 3 * aw, 3 * aw, d, 3 * aw, 0)
        if model.rotary_base is not None:
            turn_positions(blk.attn, qkv.view(B, L, 3 * aw), None, tw.dhp, model.max_position_embeddings)
        if blk.attn.differential:
            differential_heads(qkv.view(B, L, 3 * aw), blk.attn, keymask, None, None, tw.dhp, att.view(B, L, aw), False)
        else:
            _lib.check(_lib.lib().bd_attention_fwd(_lib.ptr(qkv), _lib.ptr(keymask), _lib.ptr(att), None, B, L, H, tw.dhp, st),
                       "bd_attention_fwd")
        ag._gemm(att, w["wo"], blk.attn.out_proj.bias, x, M, d, d, aw, d, 2)
        ag._ln(x, blk.norm2.weight, blk.norm2.bias, h, None, M, d, eps)
        ag._gemm(h, w["w1"], blk.ffn.fc1.bias, u, M, F, F, d, F, 1)
        ag._gemm(u, w["w2"], blk.ffn.fc2.bias, x, M, d, d, F, d, 2)
    if upto is not None:
        return x.view(B, L, d)
    hidden = hidden_out if hidden_out is not None else torch.empty(B, L, d, dtype=bf, device=dev)
    ag._ln(x, model.final_norm.weight, model.final_norm.bias, hidden, None, M, d, eps)
    logits = None
    if want_logits:
        logits = logits_out if logits_out is not None else torch.empty(B, L, V, device=dev)
        ag._gemm(hidden, tw.wout, None, logits, M, tw.vpad, V, d, V, 3)
    return (hidden if want_hidden else None), logits


def _ffn_core(ffn, a_bf16, M, out_f32, epilogue):
    w1, b1, w2, b2 = _ffn_weights(ffn)
    d, F = ffn.fc1.in_features, ffn.fc1.out_features
    h = torch.empty(M, F, dtype=torch.bfloat16, device=a_bf16.device)
    _gemm(a_bf16, w1, b1, h, M, F, d, 1)
    _gemm(h, w2, b2, out_f32, M, d, F, epilogue)


def attention_forward(mha, x, attention_mask=None):
    params = list(mha.parameters())
    _check(x, "MultiHeadAttention.forward", params)
    B, L, d = x.shape
    xf = x.detach().to(torch.float32).contiguous()
    out = torch.empty(B * L, d, dtype=torch.float32, device=x.device)
    _attention_core(mha, _cast(xf.view(B * L, d)), _keymask(attention_mask, B, L, x.device), B, L, out, 3)
    return out.view(B, L, d)


def ffn_forward(ffn, x):
    params = list(ffn.parameters())
    _check(x, "FeedForward.forward", params)
    B, L, d = x.shape
    xf = x.detach().to(torch.float32).contiguous()
    out = torch.empty(B * L, d, dtype=torch.float32, device=x.device)
    _ffn_core(ffn, _cast(xf.view(B * L, d)), B * L, out, 3)
    return out.view(B, L, d)


def block_forward(block, x, attention_mask=None):
    params = list(block.parameters())
    _check(x, "TransformerBlock.forward", params)
    B, L, d = x.shape
    M = B * L
    out = x.detach().to(torch.float32).contiguous().clone().view(M, d)      # the residual stream, updated in place
    _attention_core(block.attn, _layernorm(out, block.norm1, M, d), _keymask(attention_mask, B, L, x.device), B, L, out, 2)
    _ffn_core(block.ffn, _layernorm(out, block.norm2, M, d), M, out, 2)
    return out.view(B, L, d)
