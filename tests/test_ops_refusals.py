"""What the stand-alone operators refuse, in Python and at the C ABI, before anything reaches a GPU: every call here
fails its checks on the host (null or made-up addresses are never followed)."""
import ctypes as C

import pytest
import torch

from bidiff import _lib, ops

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def attn(q=(2, 3, 4, 32), k=(2, 5, 4, 32), v=(2, 5, 2, 64), lam=(2,), **kw):
    t = [x if isinstance(x, torch.Tensor) else z(*x) for x in (q, k, v, lam)]
    return ops.differential_attention(*t, **kw)


@pytest.mark.parametrize("err,call", [
    (ValueError, lambda: attn(q=(3, 4, 32))),
    (TypeError, lambda: attn(q=z(2, 3, 4, 32, dtype=torch.float16))),
    (TypeError, lambda: attn(lam=z(2, dtype=torch.float64))),
    (NotImplementedError, lambda: attn(q=(2, 3, 4, 48), k=(2, 5, 4, 48), v=(2, 5, 2, 96))),
    (ValueError, lambda: attn(v=(2, 5, 2, 32))),                       # values not twice as wide
    (ValueError, lambda: attn(q=(2, 3, 3, 32))),                       # an odd number of maps
    (ValueError, lambda: attn(k=(2, 5, 2, 32))),                       # keys of another head count than values
    (ValueError, lambda: attn(q=(2, 3, 6, 32), lam=(3,))),             # 3 heads on 2 key heads
    (ValueError, lambda: attn(k=(2, 6, 4, 32))),
    (ValueError, lambda: attn(q=(1, 3, 4, 32))),
    (ValueError, lambda: attn(lam=(3,))),
    (ValueError, lambda: attn(lam=(5, 2, 3, 2))),
    (ValueError, lambda: attn(scale=0.0)),
    (ValueError, lambda: attn(scale=float("nan"))),
    (ValueError, lambda: attn(max_seqlen=4)),
    (ValueError, lambda: attn(key_mask=torch.ones(2, 4, dtype=torch.bool))),
    (ValueError, lambda: attn(q=(4, 4, 32), k=(4, 4, 32), v=(4, 2, 64), cu_seqlens=torch.tensor([0.0, 4.0]), max_seqlen=4)),
    (ValueError, lambda: attn(q=(4, 4, 32), k=(4, 4, 32), v=(4, 2, 64), cu_seqlens=torch.tensor([0]), max_seqlen=4)),
    (ValueError, lambda: attn(q=(4, 4, 32), k=(4, 4, 32), v=(4, 2, 64), cu_seqlens=torch.tensor([0, 4]), max_seqlen=0)),
    (ValueError, lambda: attn(q=(3, 4, 32), k=(4, 4, 32), v=(4, 2, 64), cu_seqlens=torch.tensor([0, 4]), max_seqlen=4)),
    (ValueError, lambda: attn(k=torch.zeros(2, 5, 4, 32, dtype=BF, device="meta"))),
    (RuntimeError, lambda: attn()),                                    # CPU tensors: no execution path
    (RuntimeError, lambda: attn(q=(4, 4, 32), k=(4, 4, 32), v=(4, 2, 64), cu_seqlens=torch.tensor([0, 4]))),
])
def test_differential_attention_refuses(err, call):
    with pytest.raises(err):
        call()


TABLE = torch.zeros(8, 4, 2)


@pytest.mark.parametrize("err,call", [
    (ValueError, lambda: ops.rotary(z(3, 8), None, TABLE)),
    (TypeError, lambda: ops.rotary(z(1, 3, 2, 8, dtype=torch.float16), None, TABLE)),
    (ValueError, lambda: ops.rotary(z(1, 3, 2, 8), z(1, 4, 2, 8), TABLE)),
    (ValueError, lambda: ops.rotary(z(1, 3, 2, 8), z(1, 3, 2, 8, dtype=torch.float32), TABLE)),
    (ValueError, lambda: ops.rotary(z(1, 3, 2, 6), None, TABLE)),                     # turns more than a head has
    (ValueError, lambda: ops.rotary(z(1, 3, 2, 8), None, TABLE.double())),
    (ValueError, lambda: ops.rotary(z(1, 3, 2, 8), None, TABLE[:, ::2])),
    (ValueError, lambda: ops.rotary(z(1, 3, 2, 8), None, TABLE[:0])),
    (TypeError, lambda: ops.rotary(z(1, 3, 2, 8), None, TABLE, torch.zeros(3, dtype=torch.int32))),
    (ValueError, lambda: ops.rotary(z(1, 3, 2, 8), None, TABLE, torch.zeros(4, dtype=torch.long))),
    (NotImplementedError, lambda: ops.rotary(z(1, 3, 2, 8), None, TABLE.clone().requires_grad_(True))),
    (RuntimeError, lambda: ops.rotary_(z(1, 3, 2, 8).requires_grad_(True), None, TABLE)),
    (ValueError, lambda: ops.rotary_(z(1, 1, 2, 8).expand(1, 3, 2, 8), None, TABLE)),
    (ValueError, lambda: ops.rotary_(z(1, 3, 8, 2).transpose(2, 3), None, TABLE[:, :1].contiguous())),
    (RuntimeError, lambda: ops.rotary(z(1, 3, 2, 8), None, TABLE)),
    (RuntimeError, lambda: ops.rotary_(z(1, 3, 2, 8), None, TABLE)),
    (ValueError, lambda: ops.rotary_table(7, 4)),
    (ValueError, lambda: ops.rotary_table(8, 0)),
    (ValueError, lambda: ops.rotary_table(8, 4, scaling="cubic")),
    (ValueError, lambda: ops.rotary_table(2, 4, scaling="ntk", factor=2.0)),
    (ValueError, lambda: ops.rotary_table(8, 4, scaling="yarn", factor=2.0)),
    (ValueError, lambda: ops.rotary_table(8, 4, factor=0.0)),
])
def test_rotary_refuses(err, call):
    with pytest.raises(err):
        call()


def ce(hidden=(3, 64), weight=(7, 64), targets=None, *rest):
    t = [x if isinstance(x, torch.Tensor) else z(*x) for x in (hidden, weight)]
    return ops.linear_cross_entropy(*t, torch.zeros(3, dtype=torch.long) if targets is None else targets, *rest)


@pytest.mark.parametrize("err,call", [
    (TypeError, lambda: ce(hidden=z(3, 64, dtype=torch.float16))),
    (TypeError, lambda: ce(weight=z(7, 64, dtype=torch.float64))),
    (ValueError, lambda: ce(weight=(7, 128))),
    (ValueError, lambda: ce(weight=(0, 64))),
    (ValueError, lambda: ce(weight=(64,))),
    (NotImplementedError, lambda: ce(hidden=(3, 96), weight=(7, 96))),
    (TypeError, lambda: ce(targets=torch.zeros(3, dtype=torch.int32))),
    (ValueError, lambda: ce(targets=torch.zeros(4, dtype=torch.long))),
    (ValueError, lambda: ops.linear_cross_entropy(z(3, 64), z(7, 64), torch.zeros(3, dtype=torch.long), torch.ones(2))),
    (ValueError, lambda: ops.linear_cross_entropy(z(3, 64), z(7, 64), torch.zeros(3, dtype=torch.long), None, torch.ones(3, 1))),
    (RuntimeError, lambda: ce()),
    (RuntimeError, lambda: ce(hidden=(0, 64), targets=torch.zeros(0, dtype=torch.long))),
])
def test_linear_cross_entropy_refuses(err, call):
    with pytest.raises(err):
        call()


# ---------------------------------------------------------------- the C ABI's own checks
FAKE = 1 << 20      # an aligned, made-up address: the calls below return before anything is launched


def diff_args(**kw):
    a = _lib.DiffAttnArgs()
    for n in ("q", "k", "v", "lam", "out", "dout", "dq", "dk", "dv", "dlam", "lse", "workspace"):
        setattr(a, n, FAKE)
    a.B, a.Lq, a.Lk, a.H, a.Hkv, a.head_dim, a.scale, a.workspace_bytes = 2, 3, 5, 4, 2, 64, 0.1, 1 << 40
    for n, x in kw.items():
        if n.endswith("_stride"):
            getattr(a, n)[:] = x
        else:
            setattr(a, n, x)
    return a


@pytest.mark.parametrize("kw", [{"q": None}, {"lam": None}, {"out": None}, {"B": 0}, {"Lk": 0}, {"Hkv": 3}, {"head_dim": 48}, {"scale": 0.0},
                                {"lam_dtype": 2}, {"q": FAKE + 2}, {"out": FAKE + 8}, {"k_stride": (8, 8, 4)}, {"out_stride": (8, 4, 8)},
                                {"cu_seqlens": FAKE}, {"cu_seqlens": FAKE, "Lk": 3}, {"maps": FAKE, "lse": None}, {"B": 1 << 25},
                                {"Lk": 65536, "B": 1, "workspace": None}, {"Lk": 65536, "B": 1, "workspace_bytes": 16}])
def test_diff_attention_forward_refuses_at_the_c_abi(kw):
    assert _lib.lib().bd_diff_attention_fwd(C.byref(diff_args(**kw)), None) == -1
    assert b"bd_diff_attention_fwd" in _lib.lib().bd_last_error()


@pytest.mark.parametrize("kw", [{"dout": None}, {"dk": None}, {"lse": None}, {"dlam": None}, {"dv": FAKE + 2}, {"dq_stride": (8, 2, 8)},
                                {"workspace_bytes": 16}, {"workspace": None}])
def test_diff_attention_backward_refuses_at_the_c_abi(kw):
    assert _lib.lib().bd_diff_attention_bwd(C.byref(diff_args(**kw)), None) == -1
    assert b"bd_diff_attention_bwd" in _lib.lib().bd_last_error()


def test_null_arguments_and_sizes_at_the_c_abi():
    L = _lib.lib()
    assert L.bd_diff_attention_fwd(None, None) == -1 and L.bd_diff_attention_bwd(None, None) == -1
    assert L.bd_diff_attention_workspace_bytes(C.byref(diff_args(Hkv=3)), 0) == -1
    assert L.bd_diff_attention_dlam(None, FAKE, 0, 1, 1, 1, 1, 1, 1, None) == -1
    assert L.bd_diff_attention_dlam(FAKE, FAKE, 7, 1, 1, 1, 1, 1, 1, None) == -1
    assert L.bd_linear_ce_state_bytes(0, 64) == -1 and L.bd_linear_ce_workspace_bytes(1, 64, 0, 0) == -1


@pytest.mark.parametrize("change", [{"M": 0}, {"d": 96}, {"V": 0}, {"loss": None}, {"hidden": FAKE + 2}, {"state_bytes": 16}, {"ws_bytes": 16},
                                    {"M": 1 << 24}])
def test_linear_ce_forward_refuses_at_the_c_abi(change):
    a = dict(hidden=FAKE, weight=FAKE, targets=FAKE, ind=None, attn=None, loss=FAKE, M=4, d=64, V=9, state=FAKE, state_bytes=1 << 40, ws=FAKE,
             ws_bytes=1 << 40)
    a.update(change)
    assert _lib.lib().bd_linear_ce_fwd(*a.values(), None) == -1
    assert b"bd_linear_ce_fwd" in _lib.lib().bd_last_error()


@pytest.mark.parametrize("change", [{"M": 0}, {"d": 96}, {"g": None}, {"dh": None, "dw": None}, {"dt": 3}, {"state_bytes": 16}, {"ws_bytes": 16}])
def test_linear_ce_backward_refuses_at_the_c_abi(change):
    a = dict(weight=FAKE, g=FAKE, dh=FAKE, dw=FAKE, dt=0, M=4, d=64, V=9, state=FAKE, state_bytes=1 << 40, ws=FAKE, ws_bytes=1 << 40)
    a.update(change)
    assert _lib.lib().bd_linear_ce_bwd(*a.values(), None) == -1
    assert b"bd_linear_ce_bwd" in _lib.lib().bd_last_error()


@pytest.mark.parametrize("change", [{"n": 3}, {"table": None}, {"rows": 0}, {"B": 0}, {"rd": 5}, {"rd": 66}, {"dtype": 2}, {"heads": 0}, {"src": None},
                                    {"dst": FAKE, "dst_stride": (8, 8, 16)}, {"B": 1 << 20, "L": 1 << 20}])
def test_rotary_refuses_at_the_c_abi(change):
    a = dict(n=1, table=FAKE, rows=4, B=1, L=2, D=64, rd=64, dtype=0, heads=2, src=FAKE, dst=2 * FAKE, dst_stride=(8, 8, 8))
    a.update(change)
    t = (_lib.RotaryTensor * 3)()
    for x in t:
        x.src, x.dst, x.n_heads = a["src"], a["dst"], a["heads"]
        x.src_stride[:], x.dst_stride[:] = (8, 8, 8), a["dst_stride"]
    assert _lib.lib().bd_rotary(t, a["n"], a["table"], a["rows"], None, 0, a["B"], a["L"], a["D"], a["rd"], 0, 0, a["dtype"], None) == -1
    assert b"bd_rotary" in _lib.lib().bd_last_error()


def test_rotary_in_place_refuses_the_same_memory_twice():
    x = z(1, 3, 4, 8)
    with pytest.raises(ValueError, match="same memory"):
        ops.rotary_(x, x, TABLE)
    with pytest.raises(ValueError, match="same memory"):
        ops.rotary_(x, x[:, :, :2], TABLE)


def test_linear_cross_entropy_refuses_more_rows_than_it_counts():
    h, w = z(1, 64, dtype=torch.bfloat16).expand(1 << 24, 64), z(5, 64, dtype=torch.bfloat16)
    t = torch.zeros(1, dtype=torch.long).expand(1 << 24)
    with pytest.raises(NotImplementedError, match="rows"):
        ops.linear_cross_entropy(h, w, t)
    with pytest.raises(RuntimeError):                    # one row fewer is only refused for where it lies
        ops.linear_cross_entropy(h[1:], w, t[1:])
