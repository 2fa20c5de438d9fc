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


def up(x, m):
    return (x + m - 1) // m * m


@pytest.mark.parametrize("M,d,V", [(32768, 384, 803), (131072, 4096, 1000), (131072, 4096, 256), (8192, 384, 803), (1 << 20, 384, 5000)])
def test_scratch_of_the_head_loss(M, d, V):
    """The backward asks for the score gradients of a piece (256 MB, or 256 columns where the rows are more than that), the slabs
    of dh where sums over pieces or splits need them (512 MB, or one fp32 [M, d]) and at most 64 MB of slabs of dW; none of
    the former where the product writes dh itself, or where dh is not asked for."""
    size = ops._lib.lib().bd_linear_ce_workspace_bytes
    rows = up(M, 256)
    scores, dh, dw = max(256 << 20, 512 * rows), max(512 << 20, 4 * rows * d), 64 << 20
    both, only_dw, only_dh = size(M, d, V, 1), size(M, d, V, 3), size(M, d, V, 4)
    assert 0 < only_dw <= scores + dw and 0 < only_dh <= scores + dh and max(only_dw, only_dh) <= both <= scores + dh + dw
    one_piece = 2 * rows * up(V, 256) <= 256 << 20
    if one_piece and (-(-rows // 128) + 3) // 4 * -(-d // 128) > 128:      # (a quarter of the rows keeps half of the CUs busy: no splits)
        assert only_dh <= scores and both <= scores + dw


def turned_with(monkeypatch, mha, lengths):
    """The tables that calls of these lengths turn with, and all that the module keeps."""
    from bidiff.model import _blocks
    handed = []
    monkeypatch.setattr(_blocks.ops, "_rotary_launch", lambda pairs, table, *a: handed.append(table))
    for n in lengths:
        _blocks.turn_positions(mha, torch.zeros(1, n, 3 * mha.hidden_size, dtype=BF), None, mha.head_dim, n)
    return handed, [t for tables in mha.__dict__["_rotary_by_base"].values() for t in tables]


def test_rotary_tables_follow_the_base(monkeypatch):
    """A module whose base was changed (a longer context) turns by the new one, and by the old one again when it is put back."""
    from bidiff.model.backbone import MultiHeadAttention
    mha = MultiHeadAttention(64, 2, 0.0, rotary_base=10000.0)
    for base in (10000.0, 500000.0, 10000.0):
        mha.rotary_base = base
        (table, again), _ = turned_with(monkeypatch, mha, (9, 5))
        assert torch.equal(table[:9], ops.rotary_table(32, 9, base=base)) and again is table


def test_rotary_tables_of_growing_lengths(monkeypatch):
    """A module that is called with one more token each time keeps a handful of tables, and those it has handed out stay."""
    from bidiff.model.backbone import MultiHeadAttention
    mha = MultiHeadAttention(64, 2, 0.0, rotary_base=10000.0)
    handed, kept = turned_with(monkeypatch, mha, range(1, 1500))
    assert all(t.shape[0] >= n for n, t in enumerate(handed, 1))
    assert all(any(t is x for x in kept) for t in handed)          # a captured graph may still read any of them
    assert sum(t.shape[0] for t in kept) <= 4 * 1500 and len(kept) <= 12
    assert torch.equal(handed[-1][:1499], ops.rotary_table(32, 1499))


def test_models_pickled_before_the_options_existed():
    """A module that was saved whole without the newer attributes (attention, rotary_base, fused_head_loss) works as what it was."""
    from bidiff.model.backbone import DiffusionBackbone
    from bidiff.model.diffusion import DiscreteMaskingDiffusion
    bb = DiffusionBackbone(39, hidden_size=128, num_layers=1, num_heads=2, ffn_hidden_size=256, max_position_embeddings=16, num_diffusion_steps=5)
    model = DiscreteMaskingDiffusion(bb, num_steps=5, mask_token_id=1, pad_token_id=0, bos_token_id=2, eos_token_id=3)
    want = bb.config_dict()
    for m in (bb, *(b.attn for b in bb.layers)):
        for name in ("attention", "rotary_base", "differential"):
            m.__dict__.pop(name, None)
    model.__dict__.pop("fused_head_loss", None)
    assert bb.plain_attention and not model.fused_head_loss
    assert bb.layers[0].attn.rotary_base is None and not bb.layers[0].attn.differential
    assert bb.config_dict() == want


@pytest.mark.parametrize("scale", [1e-39, 9e-31, 2e30, 1e39, float("inf"), -0.1])
def test_scales_out_of_range_are_refused(scale):
    """Near the ends of fp32 the maximum's slack or the scaled scores are no numbers any more: refused in Python and at the C ABI."""
    with pytest.raises(ValueError, match="scale"):
        ops.differential_attention(z(2, 3, 4, 32), z(2, 5, 4, 32), z(2, 5, 2, 64), z(2), scale=scale)
    import ctypes as C
    from bidiff import _lib
    a = _lib.DiffAttnArgs()
    for n in ("q", "k", "v", "lam", "out", "workspace"):
        setattr(a, n, 1 << 20)                # an aligned, made-up address that is never followed
    a.B, a.Lq, a.Lk, a.H, a.Hkv, a.head_dim, a.scale, a.workspace_bytes = 2, 3, 5, 4, 2, 64, scale, 1 << 40
    assert _lib.lib().bd_diff_attention_fwd(C.byref(a), None) == -1 and b"scale" in _lib.lib().bd_last_error()
