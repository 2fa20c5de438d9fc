"""Stand-alone operators for denoisers built from this package's parts, each with its gradient.

``rotary`` turns query and key heads by their positions (beside the learned position table of ``DiffusionBackbone``),
``differential_attention`` is the difference of two softmax maps over one set of values (beside the attention of
``MultiHeadAttention``), and ``linear_cross_entropy`` is the masked cross entropy of the vocabulary head without its
logits (beside ``training.autograd.masked_cross_entropy``). All run on the current stream of their operands' device, take
their scratch memory from torch's allocator, repeat bit for bit, and may be captured into a HIP graph (packed rows:
with ``max_seqlen`` given). Operands on a CPU raise ``RuntimeError`` (there is no other execution path), operands with a
forward-mode tangent ``NotImplementedError``.
"""
import ctypes as C
import functools
import math
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float32: 1}

# The argument blocks are packed by ``struct`` (a ctypes structure costs a call per field; a small call is host-bound)
_ROTARY_TENSOR = struct.Struct("PP6qi4x")
_ATTENTION = struct.Struct("4P15qi4xPqP7if4Pq5Pi4x12q")
assert _ROTARY_TENSOR.size == C.sizeof(_lib.RotaryTensor) and _ATTENTION.size == C.sizeof(_lib.DiffAttnArgs)


class _Elsewhere:
    """Makes the operands' device current for the launches inside."""

    def __init__(self, device):
        self.ctx = torch.cuda.device(device)

    def __enter__(self):
        self.ctx.__enter__()
        return _lib.stream_handle()

    def __exit__(self, *exc):
        return self.ctx.__exit__(*exc)


class _Here:
    def __enter__(self):
        return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _on(device):
    """Context for launches on ``device``: its current stream's handle, the device made current if it is not."""
    return _HERE if torch.cuda.current_device() == device.index else _Elsewhere(device)


def _same_device(what, first, *others):
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise ValueError(f"bidiff {what}: operands on {dev} and {t.device}; all must be on one device")


def _no_tangents(what, *operands):
    """The kernels have no forward-mode derivative: a dual operand is refused (its tangent would be lost)."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in operands):
        raise NotImplementedError(f"bidiff {what}: no forward-mode derivative; an operand carries a tangent")


def _like(t):
    """A contiguous tensor of ``t``'s shape, dtype and device, not filled."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _keeps_maps(Lk, D):
    """Beyond 8 keys for each value of a head the forward of a training step leaves each map's output in fp32 for the backward
    (16 * head_dim bytes a row and head); up to there the backward walks the keys once more instead. Measured, all kernels of
    a step, maps kept / keys walked twice: 3 heads of 64, 256 x 128 tokens 140 / 122 us, 64 x 512 211 / 203, 42 x 768 262 / 272,
    16 x 2048 440 / 479; heads of 128, 32 x 512 263 / 243, 16 x 1024 447 / 458, 8 x 2048 736 / 813; heads of 32, 256 x 128
    73 / 69, 128 x 256 92 / 90, 96 packed sequences of up to 509 267 / 282. (At heads of 128 and 1024 keys, on the border, the
    rule is 2 % on the wrong side.)"""
    return Lk > 8 * D


def _rows_of_16_bytes(t):
    """``t`` or a copy of it whose rows the kernels can read in 16-byte pieces."""
    *st, last = t.stride()
    if last == 1 and t.data_ptr() % 16 == 0 and not any(s % 8 for s in st):
        return t
    return t.clone(memory_format=torch.contiguous_format)


# ------------------------------------------------------------------------------------------------ rotary positions
def rotary_table(dim: int, max_positions: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original_positions: Optional[int] = None, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device=None) -> torch.Tensor:
    """Table of (cos, sin) for ``rotary``: fp32 [max_positions, dim / 2, 2], from angles evaluated in 64 bits.

    ``scaling`` stretches the positions for contexts longer than those trained on by ``factor``: None; ``"linear"``
    (positions divided by it; Chen et al. 2023, "Extending Context Window of Large Language Models via Positional
    Interpolation"); ``"ntk"`` (the base raised so that the slowest pair is stretched by the factor and the fastest not at
    all); ``"yarn"`` (Peng et al. 2023, "YaRN: Efficient Context Window Extension of Large Language Models": pairs that turn at
    least ``beta_fast`` times within ``original_positions`` are kept, those below ``beta_slow`` turns are stretched, a linear
    ramp over the pair's index between; cos and sin times 0.1 ln(factor) + 1)."""
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary_table: dim must be positive and even, got {dim}")
    if max_positions <= 0 or not base > 0.0 or not factor > 0.0:
        raise ValueError("rotary_table: max_positions, base and factor must be positive")
    i = torch.arange(dim // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / dim)
    scale = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ntk":
        if dim == 2:
            raise ValueError("rotary_table: ntk scaling needs more than one pair")
        freq = (base * factor ** (dim / (dim - 2))) ** (-2.0 * i / dim)
    elif scaling == "yarn":
        if not original_positions or original_positions <= 0 or not beta_fast > beta_slow > 0.0:
            raise ValueError("rotary_table: yarn scaling needs original_positions > 0 and beta_fast > beta_slow > 0")
        if not base > 1.0:
            raise ValueError("rotary_table: yarn scaling needs a base above 1")

        def pair_of(turns):      # the (fractional) pair that turns this often within the original positions
            return dim * math.log(original_positions / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), dim - 1)
        stretched = ((i - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        freq = freq / factor * stretched + freq * (1.0 - stretched)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif scaling is not None:
        raise ValueError(f"rotary_table: unknown scaling {scaling!r}")
    angle = torch.arange(max_positions, dtype=torch.float64)[:, None] * freq
    return (torch.stack([angle.cos(), angle.sin()], -1) * scale).float().to(device if device is not None else "cpu")


def _rotary_launch(pairs, table, positions, interleaved, inverse):
    """pairs: one or two (source, destination) of [B, L, heads, D] (or [rows, heads, D])."""
    src = pairs[0][0]
    shape = src.shape
    packed = len(shape) == 3
    B, L = (1, shape[0]) if packed else shape[:2]
    args = b""
    for s, d in pairs:
        st, dt = s.stride()[:-1], d.stride()[:-1]
        if packed:
            st, dt = (0,) + st, (0,) + dt
        args += _ROTARY_TENSOR.pack(s.data_ptr(), d.data_ptr(), *st, *dt, s.shape[-2])
    pos, pos_stride = (None, 0) if positions is None else (positions.data_ptr(), positions.stride(0) if positions.dim() == 2 else 0)
    with _on(src.device) as stream:
        _lib.check(_lib.lib().bd_rotary(args, len(pairs), table.data_ptr(), table.shape[0], pos, pos_stride, B, L, shape[-1],
                                        2 * table.shape[1], interleaved, inverse, _DTYPES[src.dtype], stream), "bd_rotary")


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, positions, interleaved, *xs):
        ctx.save_for_backward(table, positions)
        ctx.interleaved = interleaved
        out = [_like(x) for x in xs]
        _rotary_launch(list(zip(xs, out)), table, positions, interleaved, False)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        table, positions = ctx.saved_tensors
        dx, pairs = [None] * len(grads), []
        for i, g in enumerate(grads):
            if ctx.needs_input_grad[3 + i]:
                if g.stride(-1) != 1:
                    g = g.contiguous()
                dx[i] = _like(g)
                pairs.append((g, dx[i]))
        if pairs:
            _rotary_launch(pairs, table, positions, ctx.interleaved, True)
        return (None, None, None, *dx)


def _rotary_check(xs, table, positions):
    q = xs[0]
    _same_device("rotary", q, *xs[1:], table, positions)
    _no_tangents("rotary", *xs, table)
    shape = q.shape
    if len(shape) not in (3, 4):
        raise ValueError(f"rotary: expected [batch, tokens, heads, head_dim] or [rows, heads, head_dim], got {tuple(shape)}")
    if q.dtype not in _DTYPES:
        raise TypeError(f"rotary: bf16 or fp32 heads expected, got {q.dtype}")
    lead = shape[:-2]
    if len(xs) == 2 and (xs[1].dtype != q.dtype or xs[1].shape[:-2] != lead or xs[1].shape[-1] != shape[-1]):
        raise ValueError("rotary: q and k must agree in dtype, tokens and head size")
    if table.dtype != torch.float32 or table.dim() != 3 or table.shape[2] != 2 or not table.is_contiguous() or not table.numel():
        raise ValueError("rotary: table must be a contiguous fp32 [positions, rotary_dim / 2, 2] tensor (rotary_table makes one)")
    if 2 * table.shape[1] > shape[-1]:
        raise ValueError(f"rotary: the table turns {2 * table.shape[1]} values, a head has {shape[-1]}")
    if table.requires_grad:
        raise NotImplementedError("rotary: the table has no gradient")
    if positions is not None:
        if positions.dtype != torch.long:
            raise TypeError(f"rotary: positions must be int64, got {positions.dtype}")
        if positions.shape != lead and positions.shape != lead[-1:]:
            raise ValueError(f"rotary: positions must be {list(lead)} or {list(lead[-1:])}, got {tuple(positions.shape)}")
        if positions.stride(-1) != 1 and positions.shape[-1] > 1:
            positions = positions.contiguous()
    return positions


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: Optional[torch.Tensor] = None,
           interleaved: bool = False):
    """(q, k) with their heads turned by the tokens' positions; differentiable. q [B, L, heads, D] and k [B, L, key heads, D]
    (or packed rows [rows, heads, D]; k may be None, and None comes back), bf16 or fp32, any strides with a contiguous last
    axis. The first ``2 * table.shape[1]`` values of a head turn, the others are copied. ``positions`` int64 [B, L] or [L]
    (default: 0, 1, ...); a token whose position the table does not hold comes out NaN. ``interleaved``: pairs (2 i, 2 i + 1)
    instead of (i, i + half)."""
    xs = [q] if k is None else [q, k]
    positions = _rotary_check(xs, table, positions)
    _lib.require_device(q, "rotary")
    xs = [x if x.stride(-1) == 1 else x.contiguous() for x in xs]
    if q.numel() == 0 or (k is not None and k.numel() == 0):
        if q.shape[:-2].numel() == 0:
            return q.clone(), None if k is None else k.clone()
        raise ValueError("rotary: q and k need at least one head")
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        out = _Rotary.apply(table, positions, bool(interleaved), *xs)
    else:
        out = [_like(x) for x in xs]
        _rotary_launch(list(zip(xs, out)), table, positions, interleaved, False)
    return out[0], out[1] if k is not None else None


def rotary_(q: torch.Tensor, k: Optional[torch.Tensor], table: torch.Tensor, positions: Optional[torch.Tensor] = None,
            interleaved: bool = False, inverse: bool = False):
    """``rotary`` in place, for inference and for kernels' own buffers (no gradient is recorded; q and k must not share values;
    a graph that saved the old values raises in its backward pass, as after torch's in-place operations). ``inverse`` turns
    back."""
    xs = [q] if k is None else [q, k]
    positions = _rotary_check(xs, table, positions)
    if torch.is_grad_enabled() and any(x.requires_grad for x in xs):
        raise RuntimeError("rotary_: in place on a tensor that requires grad; use rotary")
    if k is not None and q.numel() and q.data_ptr() == k.data_ptr():
        raise ValueError("rotary_: q and k are the same memory; it would turn twice")
    for x in xs:
        if x.numel() and x.stride(-1) != 1:
            raise ValueError("rotary_: the last axis must be contiguous")
        if any(s == 0 and n > 1 for s, n in zip(x.stride(), x.shape)):
            raise ValueError("rotary_: in place on an expanded tensor")
    _lib.require_device(q, "rotary_")
    if all(x.numel() for x in xs):
        _rotary_launch([(x, x) for x in xs], table, positions, interleaved, inverse)
        for x in xs:                     # a graph that saved the old values has to notice, as with torch's in-place operations
            if not x.is_inference():
                torch.autograd.graph.increment_version(x)
    elif q.shape[:-2].numel():
        raise ValueError("rotary_: q and k need at least one head")
    return q, k


# ------------------------------------------------------------------------------------------------ differential attention
def _three(t):
    """The strides of the leading axes as (batch, row, head); packed rows have no batch axis."""
    st = t.stride()[:-1]
    return st if len(st) == 3 else (0,) + st


@functools.lru_cache(maxsize=256)
def _attention_workspace(B, Lq, Lk, H, Hkv, D, packed, rows, backward):
    a = _lib.DiffAttnArgs()
    a.B, a.Lq, a.Lk, a.H, a.Hkv, a.head_dim, a.total_rows, a.cu_seqlens = B, Lq, Lk, H, Hkv, D, rows, 16 if packed else None
    need = _lib.lib().bd_diff_attention_workspace_bytes(C.byref(a), int(backward))
    if need < 0:
        _lib.check(-1, "bd_diff_attention_workspace_bytes")
    return need


def _attention_sizes(q, k, v, cu, longest):
    """(B, Lq, Lk, H, Hkv, D, packed, rows)"""
    qs = q.shape
    if cu is not None:
        return cu.shape[0] - 1, longest, longest, qs[-2] // 2, v.shape[-2], qs[-1], True, qs[0]
    return qs[0], qs[1], k.shape[1], qs[-2] // 2, v.shape[-2], qs[-1], False, qs[0] * qs[1]


def _attention_call(entry, sizes, q, k, v, lam, lam_strides, key_mask, cu, scale, out=None, lse=0, maps=0, ws=0, ws_bytes=0, grads=None,
                    stream=None):
    B, Lq, Lk, H, Hkv, D, packed, rows = sizes
    none3 = (0, 0, 0)
    ptr = [0] * 5
    gst = none3 * 4
    dlam_dtype = 0
    if grads is not None:
        *tensors, dlam, dlam_dtype = grads
        ptr = [0 if t is None else t.data_ptr() for t in tensors] + [dlam]
        gst = sum((none3 if t is None else tuple(_three(t)) for t in tensors), ())
    args = _ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), *_three(q), *_three(k), *_three(v), *lam_strides,
        *(none3 if out is None else _three(out)), _DTYPES[lam.dtype],
        0 if key_mask is None else key_mask.data_ptr(), 0 if key_mask is None else key_mask.stride(0),
        cu.data_ptr() if packed else 0, rows if packed else 0, B, Lq, Lk, H, Hkv, D, scale,
        0 if out is None else out.data_ptr(), lse, maps, ws, ws_bytes, *ptr, dlam_dtype, *gst)
    _lib.check(getattr(_lib.lib(), entry)(args, stream), entry)


def _lam_strides(lam, lead, H):
    """(batch, row, head) strides of lam broadcast to lead + (H,) (0 along a broadcast axis), or None if it does not fit."""
    want = (*lead, H) if len(lead) == 2 else (1, *lead, H)
    off = 3 - lam.dim()
    if off < 0 or (off == 0 and len(lead) == 1):
        return None
    st = [0, 0, 0]
    for i, (n, s) in enumerate(zip(lam.shape, lam.stride())):
        if n != want[off + i] and n != 1:
            return None
        st[off + i] = s if n != 1 else 0
    return st


def _attention_forward(q, k, v, lam, lam_strides, key_mask, cu, longest, scale, training, out=None):
    sizes = _attention_sizes(q, k, v, cu, longest)
    _, _, Lk, H, _, D, _, rows = sizes
    dev = q.device
    if out is None:
        out = torch.empty(*q.shape[:-2], H, 2 * D, dtype=torch.bfloat16, device=dev)
    ws_bytes = _attention_workspace(*sizes, False)
    # one allocation for what the backward reads (log-sum-exps, then the maps), one for scratch
    saved = ws = None
    lse = maps = 0
    if training:
        n_lse = (rows * H * 2 + 3) // 4 * 4
        saved = torch.empty(n_lse + (rows * H * 4 * D if _keeps_maps(Lk, D) else 0), dtype=torch.float32, device=dev)
        lse = saved.data_ptr()
        maps = lse + 4 * n_lse if _keeps_maps(Lk, D) else 0
    if ws_bytes:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with _on(dev) as stream:
        _attention_call("bd_diff_attention_fwd", sizes, q, k, v, lam, lam_strides, key_mask, cu, scale, out, lse, maps,
                        ws.data_ptr() if ws_bytes else 0, ws_bytes, stream=stream)
    return out, saved


def _attention_backward(q, k, v, lam, lam_strides, key_mask, cu, longest, scale, saved, dout, dq, dk, dv, dlam):
    """Writes dq, dk, dv (any strides the kernels take) and dlam (lam's shape and dtype, contiguous). None: not asked for (dk
    and dv together)."""
    sizes = _attention_sizes(q, k, v, cu, longest)
    _, _, Lk, H, _, D, packed, rows = sizes
    # a weight for every (row, head): its gradient is written as it comes; one that was broadcast: summed from fp32
    whole = dlam is not None and lam.numel() == rows * H
    need = (_attention_workspace(*sizes, True) + 15) // 16 * 16
    ws = torch.empty(need + (0 if whole else 4 * rows * H), dtype=torch.uint8, device=q.device)
    wp, lse = ws.data_ptr(), saved.data_ptr()
    maps = lse + 4 * ((rows * H * 2 + 3) // 4 * 4) if _keeps_maps(Lk, D) else 0
    with _on(q.device) as stream:
        _attention_call("bd_diff_attention_bwd", sizes, q, k, v, lam, lam_strides, key_mask, cu, scale, None, lse, maps, wp, need,
                        (dout, dq, dk, dv, dlam.data_ptr() if whole else wp + need, _DTYPES[lam.dtype] if whole else 1), stream)
        if dlam is not None and not whole:
            lead = (1, rows) if packed else q.shape[:2]
            shape = (1,) * (3 - lam.dim()) + tuple(lam.shape)
            _lib.check(_lib.lib().bd_diff_attention_dlam(wp + need, dlam.data_ptr(), _DTYPES[lam.dtype], lead[0], lead[1], H,
                                                         shape[0] == lead[0], shape[1] == lead[1], shape[2] == H, stream),
                       "bd_diff_attention_dlam")


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, lam_strides, key_mask, cu, longest, scale):
        out, saved = _attention_forward(q, k, v, lam, lam_strides, key_mask, cu, longest, scale, True)
        ctx.save_for_backward(q, k, v, lam, key_mask, cu, saved)
        ctx.longest, ctx.scale, ctx.lam_strides = longest, scale, lam_strides
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, lam, key_mask, cu, saved = ctx.saved_tensors
        for_q, for_k, for_v, for_lam = ctx.needs_input_grad[:4]
        dq, dl = _like(q) if for_q else None, _like(lam) if for_lam else None
        dk, dv = (_like(k), _like(v)) if for_k or for_v else (None, None)      # (one kernel makes both)
        _attention_backward(q, k, v, lam, ctx.lam_strides, key_mask, cu, ctx.longest, ctx.scale, saved, _rows_of_16_bytes(dout),
                            dq, dk, dv, dl)
        return dq, dk if for_k else None, dv if for_v else None, dl, None, None, None, None, None


def differential_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lam: torch.Tensor,
                           key_mask: Optional[torch.Tensor] = None, cu_seqlens: Optional[torch.Tensor] = None,
                           max_seqlen: Optional[int] = None, scale: Optional[float] = None) -> torch.Tensor:
    """sum_j (softmax(q1 k1) - lam softmax(q2 k2))_ij v_j, every query against every visible key of its sequence.

    bf16: q [B, Lq, 2 H, D] (heads 2 h and 2 h + 1 are the two maps of head h), k [B, Lk, 2 Hkv, D], v [B, Lk, Hkv, 2 D],
    D = 32, 64 or 128, H a multiple of Hkv; returns [B, Lq, H, 2 D]. ``lam`` (bf16 or fp32) broadcasts to [B, Lq, H]: a
    weight per head, or one for each row. ``key_mask`` [B, Lk]: non-zero = visible; a query without a visible key gives
    zeros, and what masked keys and values hold reaches nothing (their gradients are zeros). Packed rows: the same tensors
    without the batch axis, ``cu_seqlens`` int [sequences + 1] (rows cu[b] .. cu[b + 1] - 1 belong to sequence b; offsets
    that do not fall; rows before the first and behind the last sequence come out zero), ``max_seqlen`` the longest (None: read
    back from the device; a longer sequence's rows from there on come out NaN, in the gradients too), ``key_mask``
    [sequences, max_seqlen]. ``scale`` (1e-30 to 1e30) defaults to 1 / sqrt(D). The backward pass leaves out what no operand needs: dq where q
    is frozen, the keys' side where k and v are."""
    _same_device("differential_attention", q, k, v, lam, key_mask, cu_seqlens)
    _no_tangents("differential_attention", q, k, v, lam)
    packed = cu_seqlens is not None
    dims = 3 if packed else 4
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != dims or len(ks) != dims or len(vs) != dims:
        raise ValueError(f"differential_attention: q, k and v need {dims} axes"
                         f"{' (packed rows have no batch axis)' if packed else ''}, got {len(qs)}, {len(ks)} and {len(vs)}")
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise TypeError(f"differential_attention: q, k and v must be bf16, got {q.dtype}, {k.dtype} and {v.dtype}")
    if lam.dtype not in _DTYPES:
        raise TypeError(f"differential_attention: lam must be bf16 or fp32, got {lam.dtype}")
    D, Hkv = qs[-1], vs[-2]
    if D not in (32, 64, 128):
        raise NotImplementedError(f"differential_attention: head sizes 32, 64 and 128 are supported, got {D}")
    if ks[-1] != D or vs[-1] != 2 * D or ks[-2] != 2 * Hkv or qs[-2] % 2 or Hkv == 0 or qs[-2] == 0:
        raise ValueError(f"differential_attention: heads do not fit: q {tuple(qs[-2:])}, k {tuple(ks[-2:])}, "
                         f"v {tuple(vs[-2:])} (two maps a head, values twice as wide)")
    H = qs[-2] // 2
    if H % Hkv:
        raise ValueError(f"differential_attention: {H} heads cannot share {Hkv} key heads evenly")
    if ks[:-2] != vs[:-2] or qs[0] != ks[0]:
        raise ValueError("differential_attention: q, k and v disagree in batch or rows")
    lead = qs[:-2]
    if lam.dim() == 0:
        lam = lam.reshape(1)
    lam_strides = _lam_strides(lam, lead, H)
    if lam_strides is None:
        raise ValueError(f"differential_attention: lam {tuple(lam.shape)} does not broadcast to {(*lead, H)}")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 1e-30 <= scale <= 1e30:
        raise ValueError(f"differential_attention: scale must lie within 1e-30 and 1e30, got {scale}")
    longest = None
    if packed and max_seqlen is None:
        _lib.require_device(q, "differential_attention")
    if packed:
        if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.dtype not in (torch.int32, torch.int64):
            raise ValueError("differential_attention: cu_seqlens must be an int32 or int64 vector of sequences + 1 offsets")
        if cu_seqlens.dtype != torch.int32 or not cu_seqlens.is_contiguous():
            cu_seqlens = cu_seqlens.to(torch.int32).contiguous()
        longest = int((cu_seqlens[1:] - cu_seqlens[:-1]).max()) if max_seqlen is None else int(max_seqlen)
        if longest < 0 or (max_seqlen is not None and longest == 0 and q.shape[0]):
            raise ValueError(f"differential_attention: max_seqlen must be positive, got {longest}")
        longest = max(longest, 1)
    elif max_seqlen is not None:
        raise ValueError("differential_attention: max_seqlen goes with cu_seqlens")
    if key_mask is not None:
        want = (cu_seqlens.numel() - 1, longest) if packed else tuple(k.shape[:2])
        if tuple(key_mask.shape) != want:
            raise ValueError(f"differential_attention: key_mask must be {want}, got {tuple(key_mask.shape)}")
        if key_mask.dtype not in (torch.bool, torch.uint8):
            key_mask = key_mask != 0
        if key_mask.stride(1) != 1 and key_mask.shape[1] > 1:
            key_mask = key_mask.contiguous()
        if key_mask.dtype == torch.bool:
            key_mask = key_mask.view(torch.uint8)
    _lib.require_device(q, "differential_attention")
    if q.numel() == 0 or k.numel() == 0:         # nothing to attend with or to: zeros that stay attached to the graph
        return q.new_zeros(*lead, H, 2 * D) + sum(t.reshape(-1)[:0].sum() for t in (q, k, v, lam)).to(q.dtype)
    q, k, v = _rows_of_16_bytes(q), _rows_of_16_bytes(k), _rows_of_16_bytes(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or lam.requires_grad):
        return _DiffAttention.apply(q, k, v, lam, lam_strides, key_mask, cu_seqlens, longest, scale)
    return _attention_forward(q, k, v, lam, lam_strides, key_mask, cu_seqlens, longest, scale, False)[0]


# ------------------------------------------------------------------------------------------------ vocabulary head
def _to_bf16(x, stream):
    x = x.contiguous()
    if x.dtype == torch.bfloat16:
        return x
    y = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    _lib.check(_lib.lib().bd_cast_f32_to_bf16(x.data_ptr(), y.data_ptr(), x.numel(), stream), "bd_cast_f32_to_bf16")
    return y


@functools.lru_cache(maxsize=256)
def _head_sizes(M, d, V):
    """Bytes of the state and of the workspaces: forward, backward, forward without state, backward for the head's gradient
    alone, for the rows' alone."""
    L_ = _lib.lib()
    sizes = (L_.bd_linear_ce_state_bytes(M, d), *(L_.bd_linear_ce_workspace_bytes(M, d, V, kind) for kind in range(5)))
    if min(sizes) < 0:
        _lib.check(-1, "bd_linear_ce_workspace_bytes")
    return sizes


def _head_loss(hidden, weight, targets, indicator, attention_mask, training):
    """(loss, the head in bf16, what the backward needs or None)"""
    dev = hidden.device
    V, d = weight.shape
    M = targets.numel()
    sizes = _head_sizes(M, d, V)
    state_bytes, ws_bytes = sizes[0], sizes[1 if training else 3]
    with _on(dev) as stream:
        h, w = _to_bf16(hidden, stream), _to_bf16(weight, stream)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        state = torch.empty(state_bytes, dtype=torch.uint8, device=dev) if training else None
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        _lib.check(_lib.lib().bd_linear_ce_fwd(
            h.data_ptr(), w.data_ptr(), targets.data_ptr(), None if indicator is None else indicator.data_ptr(),
            None if attention_mask is None else attention_mask.data_ptr(), loss.data_ptr(), M, d, V,
            state.data_ptr() if training else None, state_bytes, ws.data_ptr(), ws_bytes, stream), "bd_linear_ce_fwd")
    return loss, w, state


class _LinearCE(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, targets, indicator, attention_mask):
        loss, w, state = _head_loss(hidden, weight, targets, indicator, attention_mask, True)
        # (the weighted rows are in the state; of an fp32 head its bf16 copy is kept)
        ctx.save_for_backward(w, state)
        ctx.like = (hidden.shape, hidden.dtype, weight.dtype)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, gout):
        w, state = ctx.saved_tensors
        shape, hidden_dtype, weight_dtype = ctx.like
        V, d = w.shape
        M = shape[:-1].numel()
        dev = w.device
        sizes = _head_sizes(M, d, V)
        for_rows, for_head = ctx.needs_input_grad[:2]
        state_bytes, ws_bytes = sizes[0], sizes[2 if for_rows and for_head else 5 if for_rows else 4]
        dh = torch.empty(shape, dtype=torch.bfloat16, device=dev) if for_rows else None
        dw = None
        if for_head:                     # fp32 gradients are accumulated into, bf16 ones written
            dw = (torch.zeros if weight_dtype == torch.float32 else torch.empty)(V, d, dtype=weight_dtype, device=dev)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        if gout.dtype != torch.float32:
            gout = gout.float()
        with _on(dev) as stream:
            _lib.check(_lib.lib().bd_linear_ce_bwd(
                w.data_ptr(), gout.data_ptr(), None if dh is None else dh.data_ptr(), None if dw is None else dw.data_ptr(),
                _DTYPES[weight_dtype], M, d, V, state.data_ptr(), state_bytes, ws.data_ptr(), ws_bytes, stream), "bd_linear_ce_bwd")
        if dh is not None and hidden_dtype != torch.bfloat16:
            dh = dh.to(hidden_dtype)
        return dh, dw, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                         mask_indicator: Optional[torch.Tensor] = None,
                         attention_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``masked_cross_entropy(hidden @ weight.T, targets, mask_indicator, attention_mask)`` without the logits: the mean
    cross entropy (fp32) over the rows that are marked and attended, an exact zero when there is none.

    hidden [..., d] (the rows behind the final norm) and weight [V, d] in bf16 or fp32 (fp32 operands are rounded to bf16
    once, as the head's product does), d a multiple of 64, any V; targets int64 [...]; ``mask_indicator`` [...] (non-zero =
    counts) and ``attention_mask`` [...] (the row's weight, a whole number: bool or an integer type) may be None. Rows that
    do not count are never read and get zero gradients; a counted row whose target lies outside the vocabulary makes the
    loss NaN. Gradients come in their operand's dtype, that of an fp32 weight accumulated in fp32."""
    _same_device("linear_cross_entropy", hidden, weight, targets, mask_indicator, attention_mask)
    _no_tangents("linear_cross_entropy", hidden, weight)
    for t, name in ((hidden, "hidden"), (weight, "weight")):
        if t.dtype not in _DTYPES:
            raise TypeError(f"linear_cross_entropy: {name} must be bf16 or fp32, got {t.dtype}")
    if weight.dim() != 2 or hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1] or weight.shape[0] == 0:
        raise ValueError(f"linear_cross_entropy: hidden {tuple(hidden.shape)} does not meet weight {tuple(weight.shape)}")
    lead = hidden.shape[:-1]
    if weight.shape[1] == 0 or weight.shape[1] % 64:
        raise NotImplementedError(f"linear_cross_entropy: the hidden size must be a multiple of 64, got {weight.shape[1]}")
    if lead.numel() >= 1 << 24 or weight.shape[0] >= 1 << 28 or weight.shape[1] > 65536:
        raise NotImplementedError(f"linear_cross_entropy: at most 2^24 - 1 rows, 2^28 - 1 classes and a hidden size of 65536, got "
                                  f"{lead.numel()}, {weight.shape[0]} and {weight.shape[1]}")
    if targets.dtype != torch.long:
        raise TypeError(f"linear_cross_entropy: targets must be int64, got {targets.dtype}")
    for t, name in ((targets, "targets"), (mask_indicator, "mask_indicator"), (attention_mask, "attention_mask")):
        if t is not None and t.shape != lead:
            raise ValueError(f"linear_cross_entropy: {name} must be {list(lead)}, got {tuple(t.shape)}")
    if attention_mask is not None and (attention_mask.is_floating_point() or attention_mask.is_complex()):
        raise TypeError(f"linear_cross_entropy: attention_mask holds whole numbers (bool or integers), got {attention_mask.dtype}")
    _lib.require_device(hidden, "linear_cross_entropy")
    if targets.numel() == 0:                     # no row at all: a zero that stays attached to the graph
        return (hidden.reshape(-1)[:0].sum() + weight.reshape(-1)[:0].sum()).float()
    if mask_indicator is not None:
        if mask_indicator.dtype not in (torch.bool, torch.uint8):
            mask_indicator = mask_indicator != 0
        mask_indicator = mask_indicator.contiguous()
        if mask_indicator.dtype == torch.bool:
            mask_indicator = mask_indicator.view(torch.uint8)
    if attention_mask is not None:
        attention_mask = attention_mask.to(torch.long).contiguous()
    if hidden.data_ptr() % 16:
        hidden = hidden.clone(memory_format=torch.contiguous_format)
    if weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)
    targets = targets.contiguous()
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad):
        return _LinearCE.apply(hidden, weight, targets, mask_indicator, attention_mask)
    return _head_loss(hidden, weight, targets, mask_indicator, attention_mask, False)[0]
